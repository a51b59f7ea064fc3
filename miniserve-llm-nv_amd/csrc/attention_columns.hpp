// Attention with one row of queries to a column of the 32x32x16 matrix instruction: keys
// and values of a pair of tiles (32 keys) go through LDS once for all columns of a
// workgroup's part; a column's scores, softmax state and outputs live in two lanes.  What
// the kernels for runs of tokens and for shared keys have in common.
#pragma once

#include "attention_tiles.hpp"

namespace ms {

// Softmax arithmetic runs in base 2: the scale and log2(e) enter the exponent's
// argument by one fused multiply-add and exp2 is one instruction.  The running
// maximum of a column moves only when a step exceeds it by more than kMaxSlack (in
// base-2 units): weights may then be as large as 2^kMaxSlack instead of 1, which
// 32-bit sums and bfloat16 weights hold without loss, and the rescaling of the
// output - the most expensive vector work of a step - is skipped for the steps in
// which no column's maximum moved.
constexpr float kMaxSlack = 6.0f;

// Keys and values of one pair of tiles in LDS.  Rows are padded so that lanes that
// read different rows spread over the banks (16 lanes that read 16 bytes each of
// consecutive rows touch every bank once, for keys and for values).
//
// A row of values holds the 16 keys of its tile in the order in which the product
// P.V wants them: the scores' product leaves lane half h with the keys 4h..4h+3 and
// 8+4h..8+4h+3 of a tile, so the groups of four keys lie in the order 0, 2, 1, 3 and a
// lane reads its eight values as one 16-byte word.
//
// Key rows of 128 elements are not padded (eight buffers of them must fit the LDS):
// the 16-byte chunk c of row r lies at chunk c ^ (r & 15) instead.
template <int D>
struct alignas(16) PairBuffer {
  static constexpr bool kSwizzled = D == 128;
  static constexpr int kKeyRow = kSwizzled ? D : D + 8;      // elements; 16-byte aligned rows
  static constexpr int kValueRow = 24;                       // 16 keys of one value column + padding
  bf16 k[2 * kTileKeys][kKeyRow];
  bf16 v[2][D][kValueRow];
  // where the 8 elements from d = 8 * chunk of key row `row` lie
  __device__ __forceinline__ bf16* key_chunk(int row, int chunk) {
    return &k[row][8 * (kSwizzled ? (chunk ^ (row & 15)) : chunk)];
  }
  __device__ __forceinline__ const bf16* key_chunk(int row, int chunk) const {
    return &k[row][8 * (kSwizzled ? (chunk ^ (row & 15)) : chunk)];
  }
};

// The share of one thread in the cooperative load of a pair: 16-byte chunks, the
// same number for keys and for values, tile by tile, so that every load has a base
// that is the same in all lanes (a scalar register pair) and a 32-bit lane offset
// that never changes.
template <int D, int THREADS>
struct StagedPair {
  static constexpr int kTileChunks = 2 * D;                    // of one tile's keys; as many of its values
  static constexpr int kPerTile = (kTileChunks + THREADS - 1) / THREADS;
  bf16x8 k[2][kPerTile], v[2][kPerTile];
};

// chunk of a tile -> element offsets in the cache (from the tile's first key, and from
// the same offset of the page's value rows) and in the LDS buffer
template <int D, int THREADS>
struct ChunkPlace {
  int key, part;     // keys: (key 0..15, 8 consecutive d)
  int d, half;       // values: (column d, keys 8 half .. 8 half + 7)
  __device__ __forceinline__ ChunkPlace(int thread, int j) {
    // small heads have fewer chunks than threads: the surplus threads repeat the last chunk
    const int chunk = min(thread + j * THREADS, StagedPair<D, THREADS>::kTileChunks - 1);
    key = chunk / (D / 8);
    part = chunk - key * (D / 8);
    d = chunk >> 1;
    half = chunk & 1;
  }
};

// Where the two tiles of a pair lie in the cache: the page of each and the offset of its
// first key in the page.  The same in every lane (scalar registers); looked up from the
// block table two rounds before the pair's loads are issued, so that nothing waits for
// the table.
struct PairPages {
  int32_t page[2];
  int offset[2];
};

__device__ __forceinline__ PairPages find_pair_pages(int tile, int end_tile, const int32_t* __restrict__ table,
                                               int block_size) {
  // A pair past the end repeats the last one and a missing second tile repeats the
  // first; what they hold lies beyond the last key and is masked.
  tile = min(tile, end_tile - 1);
  PairPages pages;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int this_tile = side == 1 && tile + 1 < end_tile ? tile + 1 : tile;
    if (block_size == kTileKeys) {      // a page is a tile: no division
      pages.page[side] = uniform(table[this_tile]);
      pages.offset[side] = 0;
    } else {
      const int first_key = this_tile * kTileKeys;
      pages.page[side] = uniform(table[first_key / block_size]);
      pages.offset[side] = first_key % block_size;
    }
  }
  return pages;
}

// page_stride: elements of one page of a pool (all its kv heads); head_base: where the
// workgroup's kv head begins in a page.  Both are the same for keys and values.
template <int D, int THREADS>
__device__ __forceinline__ void stage_load(StagedPair<D, THREADS>& staged, int thread, const PairPages& pages,
                                           const bf16* __restrict__ key_pool, const bf16* __restrict__ value_pool,
                                           int64_t page_stride, int head_base, int block_size) {
  // No branch stands around a load: the counters that order the loads stay exact.
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int64_t slab = pages.page[side] * page_stride + head_base;
    const bf16* keys = key_pool + slab + pages.offset[side] * D;
    const bf16* values = value_pool + slab + pages.offset[side];
#pragma unroll
    for (int j = 0; j < StagedPair<D, THREADS>::kPerTile; ++j) {
      const ChunkPlace<D, THREADS> place(thread, j);
      staged.k[side][j] = load_bf16x8(keys + static_cast<uint32_t>(place.key * D + 8 * place.part));
      staged.v[side][j] = load_bf16x8(values + static_cast<uint32_t>(place.d * block_size + 8 * place.half));
    }
  }
}

template <int D, int THREADS>
__device__ __forceinline__ void stage_store(const StagedPair<D, THREADS>& staged, int thread, PairBuffer<D>& buffer) {
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int j = 0; j < StagedPair<D, THREADS>::kPerTile; ++j) {
      const ChunkPlace<D, THREADS> place(thread, j);
      *reinterpret_cast<bf16x8*>(buffer.key_chunk(side * kTileKeys + place.key, place.part)) = staged.k[side][j];
      // keys 8 half .. 8 half + 7: the groups 2 half and 2 half + 1, which lie at 4 half and 8 + 4 half
      const bf16x8 values = staged.v[side][j];
      *reinterpret_cast<bf16x4*>(&buffer.v[side][place.d][4 * place.half]) = bf16x4{values[0], values[1], values[2], values[3]};
      *reinterpret_cast<bf16x4*>(&buffer.v[side][place.d][8 + 4 * place.half]) =
          bf16x4{values[4], values[5], values[6], values[7]};
    }
}

// What a wave keeps of its 32 columns: this lane holds column `lane & 31`; of the
// 32 x 32 outputs of a product it holds rows 8 (v / 4) + 4 h + v % 4, h = lane / 32.
template <int D>
struct PrefillState {
  static constexpr int CS = (D + 31) / 32;   // blocks of 32 rows of O^T
  floatx16 o[CS];
  float run_max;    // scaled by log2(e) * scale; the same in both lanes of a column
  float run_sum;    // of this lane's keys only; the two lanes are added at the end
};

// One pair of key tiles (32 keys from `key0`) against the wave's 32 columns.  `masked`
// (the same in all lanes): some key of the pair is hidden from some column, or lies
// beyond what the sequence has written.  One body serves both cases, so that the
// outputs stay in the same registers whichever way a step goes.
template <int D>
__device__ __forceinline__ void consume_pair(PrefillState<D>& st, const PairBuffer<D>& buffer,
                                             const bf16x8 (&q_reg)[D / 16], int key0, int lo, int pos, int last_key,
                                             float scale_log2, int h, int column, bool masked) {
  constexpr int KS = D / 16, CS = PrefillState<D>::CS;
  floatx16 s;
#pragma unroll
  for (int v = 0; v < 16; ++v) s[v] = 0.f;
#pragma unroll
  for (int step = 0; step < KS; ++step) {
    const bf16x8 keys = *reinterpret_cast<const bf16x8*>(buffer.key_chunk(column, 2 * step + h));
    s = mfma_32x32x16(keys, q_reg[step], s);
  }
  // The values of the step are asked for now; they arrive while the weights are made.
  // slot x of the contraction index of half j: key0 + 16 j + 8 (x / 4) + 4 h + x % 4,
  // for P (registers 8 j + x below) and for V alike.
  bf16x8 values[CS][2];
#pragma unroll
  for (int c = 0; c < CS; ++c) {
    const int d = (D % 32 == 0) ? 32 * c + column : min(32 * c + column, D - 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) values[c][j] = *reinterpret_cast<const bf16x8*>(&buffer.v[j][d][8 * h]);
  }
  // register v: key0 + 8 (v / 4) + 4 h + v % 4
  if (masked) {
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int key = key0 + 8 * (v / 4) + 4 * h + (v % 4);
      s[v] = (key >= lo && key <= pos) ? s[v] : -INFINITY;
    }
    // A stale value (a slot beyond what the sequence has written) times a zero weight
    // must not become NaN: such slots exist only in steps that are masked.
#pragma unroll
    for (int c = 0; c < CS; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (key0 + 16 * j + 8 * (x / 4) + 4 * h + (x % 4) > last_key) values[c][j][x] = static_cast<__bf16>(0.0f);
  }
  float tile_max = -INFINITY;
#pragma unroll
  for (int v = 0; v < 16; ++v) tile_max = fmaxf(tile_max, s[v]);
  tile_max = max_xor32(tile_max) * scale_log2;
  // the maximum moves only when it is exceeded by more than the slack (or is still unset)
  const bool move = tile_max > st.run_max + kMaxSlack;
  const float new_max = move ? tile_max : st.run_max;
  // a column may have seen no key yet: keep everything at zero
  const float safe_max = new_max == -INFINITY ? 0.f : new_max;
  float tile_sum = 0.f;
  bf16x8 p[2];
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const float weight = fast_exp2(fmaf(s[v], scale_log2, -safe_max));
    tile_sum += weight;
    p[v / 8][v % 8] = static_cast<__bf16>(weight);
  }
  if (__any(move)) {
    const float alpha = move ? fast_exp2(st.run_max - safe_max) : 1.0f;
    st.run_sum *= alpha;
#pragma unroll
    for (int c = 0; c < CS; ++c)
#pragma unroll
      for (int v = 0; v < 16; ++v) st.o[c][v] *= alpha;
  }
  st.run_sum += tile_sum;
  st.run_max = new_max;
#pragma unroll
  for (int c = 0; c < CS; ++c)
#pragma unroll
    for (int j = 0; j < 2; ++j) st.o[c] = mfma_32x32x16(values[c][j], p[j], st.o[c]);
}

// At the end the parts of a workgroup share the finishing: of the blocks of 32 rows of
// O^T, block c is finished (joined over the parts, divided by the sum, stored) by part
// c % PARTS.  What a wave publishes for that: its maximum, its sum, and the blocks that
// another part finishes, lane by lane.
template <int D, int PARTS>
struct MergeSlot {
  static constexpr int CS = PrefillState<D>::CS;
  static constexpr int kBlocks = CS - CS / PARTS;      // most blocks that a part does not finish itself
  float value[kBlocks * 16 + 2][kWave];
  // where part `part` keeps block c (which it does not finish): behind its other such blocks
  __device__ static __forceinline__ int place(int part, int c) {
    const int own_below = c > part ? (c - part - 1) / PARTS + 1 : 0;
    return c - own_below;
  }
};

}  // namespace ms
