// Paged attention for a batch whose sequences share the front of their cache: the
// sequences of a group name the same pages for the group's first keys, and those keys
// are read once for all rows of the group instead of once a sequence.
//
// A row is one query token under one query head.  With M = max, and every sum over the
// keys that the row sees, attention splits over any partition of the keys into parts:
//
//   m_c = max_j s_j,  l_c = sum_j e^{s_j - m_c},  O_c = sum_j e^{s_j - m_c} v_j      (j in part c)
//   out = sum_c e^{m_c - M} O_c / sum_c e^{m_c - M} l_c,   M = max_c m_c
//
// The parts here are splits of the group's shared keys and splits of the sequence's own
// keys behind them.  One kernel makes the (m, l, O) of all parts, a second joins them; sequences
// that are short enough are walked whole, by a kernel of their own that leaves no parts.
//
// A workgroup takes a tile of rows of one kv head (rows of the whole group for
// shared keys, of one sequence for its own) and a range of keys, dealt out to the waves in
// pairs of 16-key tiles.  Two walks:
//
//   direct   tiles of 16 or 32 rows, 16x16x32 products, every wave against pairs of its own,
//            operands from the cache straight into registers (few rows: the keys' bytes
//            are what it costs).  32-bit storage runs it on the 32-bit matrix instruction.
//   columns  tiles of 64 or 128 rows, 32x32x16 products, 32 rows to a wave: the waves of a
//            part share every pair through LDS (many rows: each key read from the L2 has
//            to serve as many of them as possible).
//
// The waves' (m, l, O) are joined through LDS, so a workgroup leaves one part a row.
//
// Measured on MI355X (bf16, head size 128, 8 kv heads, both kernels, recorded in a graph):
//
//   2 rows of 16 heads over 512 shared keys,     11 us   one kernel, a sequence whole: a unit's
//     40 of their own                                     loads (283 KB at some 40 KB a us); in
//                                                        parts 9, but 15 an eager call, not 11
//   8 rows of 32 heads over 2,048                11 us   start of two kernels and the chain
//                                                        table -> keys -> products of each
//   45 rows of 32 heads, 7 groups of up to       39 us   161 MB in 33 us at a copy's rate; the
//     5,000 and up to 700 keys of their own               sequences' own keys are most of it
//   64 rows of 64 heads over 30,000             102 us   63 GFLOP: 0.62 PFLOP/s.  The products alone
//                                                        take 52 us at a large product's rate, the
//                                                        exponentials and conversions between them
//                                                        as much again, and the waves of a unit
//                                                        overlap only some of it
//
// With every sequence reading its keys for itself the last three take 89 us (45 rows), 138 us
// (16 rows with 5 tokens each over 4,096, here 19) and 632 us.
#include <algorithm>

#include "attention_columns.hpp"

namespace {

using ms::bf16;
using ms::bf16x4;
using ms::bf16x8;
using ms::floatx4;

typedef float floatx8 __attribute__((ext_vector_type(8)));

using ms::kTileKeys;

constexpr int kXcds = 8;            // dies of the chip, each with an L2 of its own (a wrong number costs speed only)
// Waves of a workgroup by the rows of its tile.  A compute unit holds eight of these waves
// (registers), and draws some 50 GB/s from memory whatever they have under way.  Few rows
// are bound by that and by the chain of loads at a workgroup's start: two workgroups of
// four waves, so that one's start runs beside the other's walk, and the keys on as many
// units as there are.  Many rows want one workgroup whose waves share every key.
constexpr int waves_of(int rows) { return rows <= 32 ? 4 : 8; }
constexpr int kMaxSplits = 64;      // of the shared keys, and of a sequence's own
// Fewest keys of a split (but for the last): a pair of tiles for every wave.  A shorter one
// leaves waves idle and gives the join more parts.
constexpr int split_keys(int rows) { return 2 * kTileKeys * waves_of(rows); }

// ---- operands by storage type -------------------------------------------------------

template <typename T>
struct Operand;

template <>
struct Operand<bf16> {
  using V8 = bf16x8;
  using V4 = bf16x4;
  static __device__ __forceinline__ V8 zero8() { return ms::zero_bf16x8(); }
  static __device__ __forceinline__ V4 zero4() { return ms::zero_bf16x4(); }
  // scores: s[key, row] += sum over 32 d
  static __device__ __forceinline__ floatx4 scores(V8 k, V8 q, floatx4 s) { return ms::mfma_16x16x32(k, q, s); }
  // The weights are rounded to the storage type for the second product, as the reference does and
  // as the 16-bit product asks.  A weight is off by at most half a step, 2^-8 of itself, and the
  // steps of many keys partly cancel: the norm of the outputs' error is 1.7e-3 to 1.95e-3 of the
  // outputs', of which 1.67e-3 are the outputs' own rounding.  The sums take the unrounded weights.
  static __device__ __forceinline__ floatx4 outputs(floatx4 pa, floatx4 pb, V4 va, V4 vb, floatx4 o) {
    bf16x8 p;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      p[e] = static_cast<__bf16>(pa[e]);
      p[e + 4] = static_cast<__bf16>(pb[e]);
    }
    return ms::mfma_16x16x32(p, ms::concat(va, vb), o);
  }
  static __device__ __forceinline__ void clear(V4& v, int e) { v[e] = static_cast<__bf16>(0.0f); }
  // scores are kept times log2(e), so that a weight is one exponential instruction; what that
  // leaves of a weight's 24 bits is far more than the 8 it is rounded to
  static constexpr float kScale = 1.4426950408889634f;
  static __device__ __forceinline__ float weight(float x) { return ms::fast_exp2(x); }
};

template <>
struct Operand<float> {
  using V8 = floatx8;
  using V4 = floatx4;
  static __device__ __forceinline__ V8 zero8() { return V8{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}; }
  static __device__ __forceinline__ V4 zero4() { return V4{0.f, 0.f, 0.f, 0.f}; }
  static __device__ __forceinline__ floatx4 scores(V8 k, V8 q, floatx4 s) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j], q[j], s, 0, 0, 0);
    return s;
  }
  static __device__ __forceinline__ floatx4 outputs(floatx4 pa, floatx4 pb, V4 va, V4 vb, floatx4 o) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o = __builtin_amdgcn_mfma_f32_16x16x4f32(pa[e], va[e], o, 0, 0, 0);
      o = __builtin_amdgcn_mfma_f32_16x16x4f32(pb[e], vb[e], o, 0, 0, 0);
    }
    return o;
  }
  static __device__ __forceinline__ void clear(V4& v, int e) { v[e] = 0.f; }
  static constexpr float kScale = 1.0f;
  static __device__ __forceinline__ float weight(float x) { return expf(x); }
};

// ---- where work lies ----------------------------------------------------------------

struct Sizes {
  int num_tokens, num_seqs, num_groups, num_q_heads, num_kv_heads, block_size, max_blocks;
  int most_keys;          // that a table names pages for; lengths beyond count as this
  float scale;
  int tile_rows, shared_tiles, shared_splits, own_tiles, own_splits;
};

// What a kernel is called with, as its functions see it.  (The pointers are arguments of their
// own, and not part of a struct that is passed: only so does the compiler know that no store
// changes the tables, and reads them with scalar loads.  A vector load of a page number waits
// for all loads of keys that are under way.)
struct Batch : Sizes {
  const int32_t* block_table;
  const int32_t* query_start;
  const int32_t* context_lens;
  const int32_t* group_start;
  const int32_t* shared_lens;
};

// Rows and keys of one workgroup, the same in all its lanes.
struct Work {
  int first_token;        // of the rows' segment (a group's or a sequence's tokens, which are contiguous)
  int rows, row0;         // rows of the segment, first row of this tile
  int kv_head;
  int first_key, end_key;         // keys [first_key, end_key) of this split
  int pos_of_first;       // row of token i sees keys <= pos_of_first + i; for shared keys every row sees all
  bool causal;
  const int32_t* table;
  int slot;
};

// The group's part of a flat list of tiles: every group has ceil(rows / tile_rows) of them.
__device__ __forceinline__ bool find_group_tile(const Batch& b, int tile, int rows_per_token, int tile_rows, int& group,
                                                int& local) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int g0 = 0; g0 < b.num_groups; g0 += ms::kWave) {
    const int g = g0 + lane;
    int tiles = 0;
    if (g < b.num_groups) {
      const int tokens = b.query_start[b.group_start[g + 1]] - b.query_start[b.group_start[g]];
      tiles = (tokens * rows_per_token + tile_rows - 1) / tile_rows;
    }
    int upto = tiles;
#pragma unroll
    for (int offset = 1; offset < ms::kWave; offset <<= 1) {
      const int other = __shfl_up(upto, offset, ms::kWave);
      if (lane >= offset) upto += other;
    }
    const uint64_t past = __ballot(base + upto > tile);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      group = ms::uniform(g0 + at);
      local = ms::uniform(tile - (base + __shfl(upto - tiles, at, ms::kWave)));
      return true;
    }
    base += __shfl(upto, ms::kWave - 1, ms::kWave);
  }
  return false;
}

// The most keys that a group shares.  Splits are cut by it, so that those of all groups
// have the same number of keys (a short group has fewer of them).
__device__ __forceinline__ int longest_shared(const Batch& b) {
  const int lane = threadIdx.x & 63;
  int longest = 0;
  for (int g = lane; g < b.num_groups; g += ms::kWave) longest = max(longest, b.shared_lens[g]);
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) longest = max(longest, __shfl_xor(longest, offset, ms::kWave));
  return ms::uniform(min(longest, b.most_keys));
}

// The group of a sequence, -1 for one that is in none.
__device__ __forceinline__ int group_of_sequence(const Batch& b, int seq) {
  const int lane = threadIdx.x & 63;
  int at_or_before = 0;
  for (int g0 = 0; g0 < b.num_groups; g0 += ms::kWave) {
    const int g = g0 + lane;
    at_or_before += __popcll(__ballot(g < b.num_groups && b.group_start[g] <= seq));
  }
  const int group = at_or_before - 1;
  return group >= 0 && seq < b.group_start[group + 1] ? group : -1;
}

// ---- the walk along the keys ---------------------------------------------------------

template <typename T, int D>
struct Pair {
  static constexpr int KS = (D + 31) / 32;
  static constexpr int CS = D / 16;
  typename Operand<T>::V8 k_a[KS], k_b[KS];
  typename Operand<T>::V4 v_a[CS], v_b[CS];
};

// ``pages``: of the pair's two tiles, looked up a round earlier.
template <typename T, int D>
__device__ __forceinline__ void load_pair(Pair<T, D>& pair, const Batch& b, const ms::PairPages& pages,
                                          const T* __restrict__ key_pool, const T* __restrict__ value_pool, int kv_head,
                                          int g, int r) {
  // bases that are the same in all lanes, and 32-bit lane offsets that never change
  using Op = Operand<T>;
  const int64_t page_stride = static_cast<int64_t>(b.num_kv_heads) * b.block_size * D;
  const int head_base = kv_head * b.block_size * D;
  const T* k_a = key_pool + (pages.page[0] * page_stride + head_base + pages.offset[0] * D);
  const T* k_b = key_pool + (pages.page[1] * page_stride + head_base + pages.offset[1] * D);
  const T* v_a = value_pool + (pages.page[0] * page_stride + head_base + pages.offset[0]);
  const T* v_b = value_pool + (pages.page[1] * page_stride + head_base + pages.offset[1]);
  const uint32_t k_lane = r * D + 8 * g, v_lane = r * b.block_size + 4 * g;
#pragma unroll
  for (int s = 0; s < Pair<T, D>::KS; ++s) {
    // (a head size off the grid of 32: the last slice's upper half lies in no row)
    const bool inside = D % 32 == 0 || s + 1 < Pair<T, D>::KS || g < 2;
    pair.k_a[s] = inside ? *reinterpret_cast<const typename Op::V8*>(k_a + 32 * s + k_lane) : Op::zero8();
    pair.k_b[s] = inside ? *reinterpret_cast<const typename Op::V8*>(k_b + 32 * s + k_lane) : Op::zero8();
  }
#pragma unroll
  for (int c = 0; c < Pair<T, D>::CS; ++c) {
    pair.v_a[c] = *reinterpret_cast<const typename Op::V4*>(v_a + 16 * c * b.block_size + v_lane);
    pair.v_b[c] = *reinterpret_cast<const typename Op::V4*>(v_b + 16 * c * b.block_size + v_lane);
  }
}

// One wave's state of 16 rows: row r's maximum and sum (the same in the four lane groups),
// and the unnormalised outputs of the rows 4 g + e.
template <int D>
struct RowState {
  floatx4 o[D / 16];
  float run_max, run_sum;
};

// ``last``: the last key that this lane's row sees.
template <typename T, int D>
__device__ __forceinline__ void consume(RowState<D>& st, const Pair<T, D>& pair, const typename Operand<T>::V8* q,
                                        int tile, int first_key, int last, float scale, int g) {
  using Op = Operand<T>;
  const int key_a = tile * kTileKeys + 4 * g, key_b = key_a + kTileKeys;
  floatx4 s_a = {0.f, 0.f, 0.f, 0.f}, s_b = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < Pair<T, D>::KS; ++s) {
    s_a = Op::scores(pair.k_a[s], q[s], s_a);
    s_b = Op::scores(pair.k_b[s], q[s], s_b);
  }
  float tile_max = -INFINITY;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    s_a[e] = key_a + e >= first_key && key_a + e <= last ? s_a[e] * scale : -INFINITY;
    s_b[e] = key_b + e >= first_key && key_b + e <= last ? s_b[e] * scale : -INFINITY;
    tile_max = fmaxf(tile_max, fmaxf(s_a[e], s_b[e]));
  }
  tile_max = fmaxf(tile_max, __shfl_xor(tile_max, 16, ms::kWave));
  tile_max = fmaxf(tile_max, __shfl_xor(tile_max, 32, ms::kWave));
  const float new_max = fmaxf(st.run_max, tile_max);
  const float shift = new_max == -INFINITY ? 0.f : new_max;       // a row that has seen no key yet: all its weights are 0
  const float alpha = Op::weight(st.run_max - shift);
  float tile_sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    s_a[e] = Op::weight(s_a[e] - shift);
    s_b[e] = Op::weight(s_b[e] - shift);
    tile_sum += s_a[e] + s_b[e];
  }
  tile_sum += __shfl_xor(tile_sum, 16, ms::kWave);
  tile_sum += __shfl_xor(tile_sum, 32, ms::kWave);
  st.run_sum = st.run_sum * alpha + tile_sum;
  st.run_max = new_max;
  float alpha_row[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) alpha_row[e] = __shfl(alpha, 4 * g + e, ms::kWave);
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) st.o[c][e] *= alpha_row[e];
    st.o[c] = Op::outputs(s_a, s_b, pair.v_a[c], pair.v_b[c], st.o[c]);
  }
}

// Values of keys outside the range may never have been written: they must not meet a zero weight.
template <typename T, int D>
__device__ __forceinline__ void clear_outside(Pair<T, D>& pair, int tile, int first_key, int end_key, int g) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int ka = tile * kTileKeys + 4 * g + e, kb = ka + kTileKeys;
#pragma unroll
    for (int c = 0; c < Pair<T, D>::CS; ++c) {
      if (ka < first_key || ka >= end_key) Operand<T>::clear(pair.v_a[c], e);
      if (kb < first_key || kb >= end_key) Operand<T>::clear(pair.v_b[c], e);
    }
  }
}

__device__ __forceinline__ int64_t slot_of(const Batch& b, const Work& w, int row) {
  const int per_token = b.num_q_heads / b.num_kv_heads;
  const int token = row / per_token, head = w.kv_head * per_token + row - token * per_token;
  return (static_cast<int64_t>(w.first_token + token) * b.num_q_heads + head) * (b.shared_splits + b.own_splits) + w.slot;
}

// Rows of outputs in LDS are padded by four values, so that the four rows that a wave stores
// at once lie in different banks.
template <int D, int WAVES>
constexpr size_t direct_lds_bytes() {
  return (2 * WAVES * 16 + WAVES * 16 * (D + 4)) * sizeof(float);
}

// 16 R rows against the keys of ``w`` (at least one), by the wave's pairs: every WAVES-th.
template <typename T, int D, int R, int WAVES>
__device__ __forceinline__ void walk_rows(RowState<D> (&st)[R], const Batch& b, const Work& w, const T* __restrict__ q,
                                          const T* __restrict__ key_pool, const T* __restrict__ value_pool, int wave) {
  using Op = Operand<T>;
  constexpr int KS = Pair<T, D>::KS, CS = D / 16;
  const int lane = threadIdx.x & 63;
  const int g = lane >> 4, r = lane & 15;
  const int per_token = b.num_q_heads / b.num_kv_heads;
  const int end_tile = (w.end_key - 1) / kTileKeys + 1;
  constexpr int step = 2 * WAVES;
  int t = w.first_key / kTileKeys + 2 * wave;
  // (a pair behind the end is looked up as the last one, and not loaded)
  ms::PairPages pages = ms::find_pair_pages(t, end_tile, w.table, b.block_size);

  typename Op::V8 q_reg[R][KS];
  int last[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = w.row0 + 16 * i + r;
    const int token = row / per_token, head = w.kv_head * per_token + row - token * per_token;
    const bool live = row < w.rows;
    last[i] = !live ? -1 : w.causal ? min(w.end_key - 1, w.pos_of_first + token) : w.end_key - 1;
    const T* q_row = q + (static_cast<int64_t>(w.first_token + token) * b.num_q_heads + head) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d0 = 32 * s + 8 * g;
      q_reg[i][s] = live && d0 < D ? *reinterpret_cast<const typename Op::V8*>(q_row + d0) : Op::zero8();
    }
#pragma unroll
    for (int c = 0; c < CS; ++c) st[i].o[c] = floatx4{0.f, 0.f, 0.f, 0.f};
    st[i].run_max = -INFINITY;
    st[i].run_sum = 0.f;
  }

  const auto consume_all = [&](Pair<T, D>& pair, int tile) {
    if (tile * kTileKeys < w.first_key || (tile + 2) * kTileKeys > w.end_key)
      clear_outside<T, D>(pair, tile, w.first_key, w.end_key, g);
#pragma unroll
    for (int i = 0; i < R; ++i) consume<T, D>(st[i], pair, q_reg[i], tile, w.first_key, last[i], b.scale * Op::kScale, g);
  };
  // One pair on its way while another is consumed, where the registers hold two.
  constexpr bool kAhead = R == 1 && sizeof(T) == 2;
  if constexpr (kAhead) {
    if (t < end_tile) {
      Pair<T, D> ping, pong;
      load_pair<T, D>(ping, b, pages, key_pool, value_pool, w.kv_head, g, r);
      pages = ms::find_pair_pages(t + step, end_tile, w.table, b.block_size);
      while (true) {
        int next = t + step;
        if (next < end_tile) {
          load_pair<T, D>(pong, b, pages, key_pool, value_pool, w.kv_head, g, r);
          pages = ms::find_pair_pages(next + step, end_tile, w.table, b.block_size);
        }
        consume_all(ping, t);
        t = next;
        if (t >= end_tile) break;
        next = t + step;
        if (next < end_tile) {
          load_pair<T, D>(ping, b, pages, key_pool, value_pool, w.kv_head, g, r);
          pages = ms::find_pair_pages(next + step, end_tile, w.table, b.block_size);
        }
        consume_all(pong, t);
        t = next;
        if (t >= end_tile) break;
      }
    }
  } else {
    for (; t < end_tile; t += step) {
      Pair<T, D> pair;
      load_pair<T, D>(pair, b, pages, key_pool, value_pool, w.kv_head, g, r);
      pages = ms::find_pair_pages(t + step, end_tile, w.table, b.block_size);
      consume_all(pair, t);
    }
  }
}

// 16 R rows by the whole workgroup: the pairs dealt out to the waves, their states joined
// through LDS, 16 rows at a time, four values of a row to a thread.
template <typename T, int D, int R, int WAVES>
__device__ __forceinline__ void walk_direct(const Batch& b, const Work& w, const T* __restrict__ q,
                                            const T* __restrict__ key_pool, const T* __restrict__ value_pool,
                                            float* __restrict__ partial_o, float* __restrict__ partial_ml,
                                            float* __restrict__ lds) {
  using Op = Operand<T>;
  constexpr int CS = D / 16, ROW = D + 4;
  const int lane = threadIdx.x & 63;
  const int wave = ms::uniform(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  RowState<D> st[R];
  walk_rows<T, D, R, WAVES>(st, b, w, q, key_pool, value_pool, wave);
  float* m_s = lds;                                  // [WAVES][16]
  float* l_s = m_s + WAVES * 16;                    // [WAVES][16]
  float* o_s = l_s + WAVES * 16;                    // [WAVES][16][ROW]
  constexpr int kAtOnce = WAVES * ms::kWave / (D / 4);      // rows that the threads finish at once
  const int first_row = threadIdx.x / (D / 4), d = 4 * (threadIdx.x % (D / 4));
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i > 0) __syncthreads();
    if (g == 0) {
      m_s[wave * 16 + r] = st[i].run_max;
      l_s[wave * 16 + r] = st[i].run_sum;
    }
#pragma unroll
    for (int c = 0; c < CS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o_s[(wave * 16 + 4 * g + e) * ROW + 16 * c + r] = st[i].o[c][e];
    __syncthreads();
    if (first_row >= kAtOnce) continue;                     // threads that are left over
#pragma unroll 1
    for (int in_tile = first_row; in_tile < 16 && w.row0 + 16 * i + in_tile < w.rows; in_tile += kAtOnce) {
      float mx = -INFINITY;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) mx = fmaxf(mx, m_s[v * 16 + in_tile]);
      const float shift = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f;
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < WAVES; ++v) {
        // 0 for a wave without keys; a NaN among its scores stays one in its sum
        const float factor = Op::weight(m_s[v * 16 + in_tile] - shift);
        const floatx4 o = *reinterpret_cast<const floatx4*>(&o_s[(v * 16 + in_tile) * ROW + d]);
        sum += factor * l_s[v * 16 + in_tile];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(o[e], factor, acc[e]);
      }
      const int64_t slot = slot_of(b, w, w.row0 + 16 * i + in_tile);
      if (d == 0) {
        partial_ml[2 * slot] = mx;
        partial_ml[2 * slot + 1] = sum;
      }
      *reinterpret_cast<floatx4*>(partial_o + slot * D + d) = acc;
    }
  }
}

constexpr int kColumnWaves = waves_of(128);

// 32 CW rows against the shared keys of ``w`` (at least one): CW waves of 32 columns make a
// part, and the 8 / CW parts take the pairs in turn, each through LDS buffers of its own.
template <int D, int CW>
__device__ __forceinline__ void walk_columns(const Batch& b, const Work& w, const bf16* __restrict__ q,
                                             const bf16* __restrict__ key_pool, const bf16* __restrict__ value_pool,
                                             float* __restrict__ partial_o, float* __restrict__ partial_ml,
                                             void* __restrict__ lds) {
  constexpr int PARTS = kColumnWaves / CW;
  constexpr int PART_THREADS = CW * ms::kWave;
  constexpr int KS = D / 16, CS = ms::PrefillState<D>::CS;
  using Slot = ms::MergeSlot<D, PARTS>;
  ms::PairBuffer<D>* buffers = static_cast<ms::PairBuffer<D>*>(lds);       // [parity][part]
  Slot* slots = static_cast<Slot*>(lds);                                   // [part][wave]
  const int lane = threadIdx.x & 63;
  const int wave_of_group = ms::uniform(threadIdx.x >> 6);
  const int part = wave_of_group / CW, wave = wave_of_group - part * CW;
  const int thread = threadIdx.x - part * PART_THREADS;
  const int h = lane >> 5, column = lane & 31;
  const int per_token = b.num_q_heads / b.num_kv_heads;
  const int64_t page_stride = static_cast<int64_t>(b.num_kv_heads) * b.block_size * D;
  const int head_base = w.kv_head * b.block_size * D;
  const int row = w.row0 + 32 * wave + column;
  const bool live = row < w.rows;
  const int token = live ? row / per_token : 0, head = w.kv_head * per_token + (live ? row - token * per_token : 0);
  const float scale_log2 = b.scale * Operand<bf16>::kScale;
  // Whole pairs of tiles in the loop, which need no masks; a rest of fewer than 32 keys behind it.
  const int t0 = w.first_key / kTileKeys, t1 = t0 + (w.end_key - w.first_key) / (2 * kTileKeys) * 2;
  const int end_tile = (w.end_key - 1) / kTileKeys + 1;

  ms::PrefillState<D> st;
#pragma unroll
  for (int c = 0; c < CS; ++c)
#pragma unroll
    for (int v = 0; v < 16; ++v) st.o[c][v] = 0.f;
  st.run_max = -INFINITY;
  st.run_sum = 0.f;

  // The queries are asked for before the first keys: loads come back in their order, and a wait
  // for later ones, which the compiler repeats in every round, would be one for the keys ahead.
  bf16x8 q_reg[KS];
#pragma unroll
  for (int step = 0; step < KS; ++step)
    q_reg[step] = ms::load_bf16x8(q + (static_cast<int64_t>(w.first_token + token) * b.num_q_heads + head) * D + 16 * step + 8 * h);
  // Loads are issued kDepth rounds before their pair is consumed (two where a thread stages
  // little enough), no branch stands around a load, and each buffer is named at compile time.
  constexpr int kRound = 2 * PARTS;
  constexpr int kDepth = ms::StagedPair<D, PART_THREADS>::kPerTile > 1 ? 1 : 2;
  ms::StagedPair<D, PART_THREADS> ahead[kDepth];
  ms::PairPages pages[kDepth];
#pragma unroll
  for (int i = 0; i < kDepth; ++i) {
    const int first = t0 + 2 * part + kRound * i;
    ms::stage_load<D, PART_THREADS>(ahead[i], thread, ms::find_pair_pages(first, end_tile, w.table, b.block_size), key_pool,
                                    value_pool, page_stride, head_base, b.block_size);
    pages[i] = ms::find_pair_pages(first + kDepth * kRound, end_tile, w.table, b.block_size);
  }
  for (int round_tile = t0; round_tile < t1; round_tile += 2 * kRound) {
#pragma unroll
    for (int parity = 0; parity < 2; ++parity) {
      const int i = kDepth == 2 ? parity : 0;
      const int t = round_tile + kRound * parity + 2 * part;
      ms::PairBuffer<D>& buffer = buffers[PARTS * parity + part];
      ms::stage_store<D, PART_THREADS>(ahead[i], thread, buffer);
      ms::stage_load<D, PART_THREADS>(ahead[i], thread, pages[i], key_pool, value_pool, page_stride, head_base, b.block_size);
      pages[i] = ms::find_pair_pages(t + 2 * kDepth * kRound, end_tile, w.table, b.block_size);
      __syncthreads();    // the pair is in LDS; every wave is done with the other buffers' previous content
      if (t < t1) ms::consume_pair<D>(st, buffer, q_reg, t * kTileKeys, 0, 0, 0, scale_log2, h, column, false);
    }
  }

  if (t1 * kTileKeys < w.end_key) {
    // the rest, through the first buffer of the first part
    __syncthreads();
    if (part == 0) {
      ms::stage_load<D, PART_THREADS>(ahead[0], thread, ms::find_pair_pages(t1, end_tile, w.table, b.block_size), key_pool,
                                       value_pool, page_stride, head_base, b.block_size);
      ms::stage_store<D, PART_THREADS>(ahead[0], thread, buffers[0]);
    }
    __syncthreads();
    if (part == 0)
      ms::consume_pair<D>(st, buffers[0], q_reg, t1 * kTileKeys, w.first_key, w.end_key - 1, w.end_key - 1, scale_log2, h,
                          column, true);
  }

  __syncthreads();    // everybody is done with what the memory held before
  {
    Slot& mine = slots[part * CW + wave];
#pragma unroll
    for (int c = 0; c < CS; ++c) {
      if (c % PARTS == part) continue;
      const int at = 16 * Slot::place(part, c);
#pragma unroll
      for (int v = 0; v < 16; ++v) mine.value[at + v][lane] = st.o[c][v];
    }
    mine.value[16 * Slot::kBlocks][lane] = st.run_max;
    mine.value[16 * Slot::kBlocks + 1][lane] = st.run_sum;
  }
  __syncthreads();
  if (part >= CS) return;      // no block of outputs is this part's to finish
  float joint = -INFINITY, total = 0.f, factor[PARTS];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) joint = fmaxf(joint, slots[p * CW + wave].value[16 * Slot::kBlocks][lane]);
  const float shift = joint == -INFINITY ? 0.f : joint;
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    const Slot& theirs = slots[p * CW + wave];
    factor[p] = ms::fast_exp2(theirs.value[16 * Slot::kBlocks][lane] - shift);       // 0 for a part without keys
    total += theirs.value[16 * Slot::kBlocks + 1][lane] * factor[p];
  }
  total += __shfl_xor(total, 32, ms::kWave);      // the column's other lane has the other keys
  if (!live) return;
  const int64_t slot = slot_of(b, w, row);
  if (part == 0 && h == 0) {
    partial_ml[2 * slot] = joint;
    partial_ml[2 * slot + 1] = total;
  }
#pragma unroll
  for (int c = 0; c < CS; ++c) {
    if (c % PARTS != part) continue;
    float sums[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) sums[v] = 0.f;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      if (p == part) {
#pragma unroll
        for (int v = 0; v < 16; ++v) sums[v] = fmaf(st.o[c][v], factor[p], sums[v]);
      } else {
        const Slot& theirs = slots[p * CW + wave];
        const int at = 16 * Slot::place(p, c);
#pragma unroll
        for (int v = 0; v < 16; ++v) sums[v] = fmaf(theirs.value[at + v][lane], factor[p], sums[v]);
      }
    }
#pragma unroll
    for (int quad = 0; quad < 4; ++quad) {
      const int d = 32 * c + 8 * quad + 4 * h;
      if (D % 32 != 0 && d >= D) continue;
      *reinterpret_cast<floatx4*>(partial_o + slot * D + d) =
          floatx4{sums[4 * quad], sums[4 * quad + 1], sums[4 * quad + 2], sums[4 * quad + 3]};
    }
  }
}

template <typename T, int D, int ROWS>
constexpr size_t lds_bytes() {
  constexpr size_t direct = direct_lds_bytes<D, waves_of(ROWS)>();
  if constexpr (ROWS <= 32) {
    return direct;
  } else {
    constexpr int PARTS = kColumnWaves * 32 / ROWS;
    constexpr size_t buffers = 2 * PARTS * sizeof(ms::PairBuffer<D>);
    constexpr size_t slots = kColumnWaves * sizeof(ms::MergeSlot<D, PARTS>);
    constexpr size_t columns = buffers > slots ? buffers : slots;
    return columns > direct ? columns : direct;
  }
}

// Rows of a tile whose part got no keys.
__device__ __forceinline__ void leave_empty(const Batch& b, const Work& w, int tile_rows, float* __restrict__ partial_ml) {
  for (int i = threadIdx.x; i < tile_rows && w.row0 + i < w.rows; i += blockDim.x) {
    const int64_t slot = slot_of(b, w, w.row0 + i);
    partial_ml[2 * slot] = -INFINITY;
    partial_ml[2 * slot + 1] = 0.f;
  }
}

// Workgroups: first the shared keys, (kv head, split, tile of ROWS rows) each; then the
// sequences' own keys, (kv head, split, tile of 16 rows, sequence) each.
template <typename T, int D, int ROWS>
__global__ __launch_bounds__(waves_of(ROWS) * ms::kWave) MS_WAVES_PER_EU(2, 2) void attention_shared_kernel(
    Sizes sizes, const int32_t* __restrict__ block_table, const int32_t* __restrict__ query_start,
    const int32_t* __restrict__ context_lens, const int32_t* __restrict__ group_start,
    const int32_t* __restrict__ shared_lens, const T* __restrict__ q, const T* __restrict__ key_pool,
    const T* __restrict__ value_pool, float* __restrict__ partial_o, float* __restrict__ partial_ml) {
  const Batch b{sizes, block_table, query_start, context_lens, group_start, shared_lens};
  constexpr int WAVES = waves_of(ROWS);
  __shared__ __align__(16) unsigned char lds[lds_bytes<T, D, ROWS>()];
  const int per_token = b.num_q_heads / b.num_kv_heads;
  int item = blockIdx.x;
  Work w;
  // The tiles of one kv head and split read the same keys: they are handed to one die, where
  // all but the first find them in the L2 (consecutive workgroups go to the dies in turn).
  const int units = b.num_kv_heads * b.shared_splits;
  const int shared_items = (units + kXcds - 1) / kXcds * kXcds * b.shared_tiles;
  if (item < shared_items) {
    const int turn = item / kXcds;
    const int unit = turn / b.shared_tiles * kXcds + item % kXcds;
    if (unit >= units) return;
    const int tile = turn % b.shared_tiles, split = unit / b.num_kv_heads;
    w.kv_head = unit - split * b.num_kv_heads;
    int group = 0, local = tile, longest = min(b.shared_lens[0], b.most_keys);
    if (b.num_groups > 1) {
      longest = longest_shared(b);
      if (!find_group_tile(b, tile, per_token, ROWS, group, local)) return;
    }
    const int first_seq = b.group_start[group];
    w.first_token = b.query_start[first_seq];
    w.rows = (b.query_start[b.group_start[group + 1]] - w.first_token) * per_token;
    w.row0 = local * ROWS;
    if (w.row0 >= w.rows) return;
    const int keys = min(max(b.shared_lens[group], 0), b.most_keys);
    const int per_split = max((longest + b.shared_splits - 1) / b.shared_splits, split_keys(ROWS));
    const int whole_pairs = (per_split + 2 * kTileKeys - 1) / (2 * kTileKeys) * 2 * kTileKeys;
    w.first_key = min(split * whole_pairs, keys);
    w.end_key = min(w.first_key + whole_pairs, keys);
    w.causal = false;
    w.pos_of_first = 0;
    w.table = b.block_table + static_cast<int64_t>(first_seq) * b.max_blocks;
    w.slot = split;
    if (w.first_key >= w.end_key) {
      leave_empty(b, w, ROWS, partial_ml);
    } else if constexpr (ROWS <= 32) {
      walk_direct<T, D, ROWS / 16, WAVES>(b, w, q, key_pool, value_pool, partial_o, partial_ml,
                                          reinterpret_cast<float*>(lds));
    } else {
      walk_columns<D, ROWS / 32>(b, w, q, key_pool, value_pool, partial_o, partial_ml, lds);
    }
    return;
  }
  item -= shared_items;
  w.kv_head = item % b.num_kv_heads;
  item /= b.num_kv_heads;
  const int split = item % b.own_splits;
  item /= b.own_splits;
  const int first_tile = item % b.own_tiles;
  const int seq = item / b.own_tiles;
  const int group = b.num_groups > 1 ? group_of_sequence(b, seq) : seq >= b.group_start[0] && seq < b.group_start[1] ? 0 : -1;
  const int context = min(max(b.context_lens[seq], 0), b.most_keys);
  w.first_token = b.query_start[seq];
  const int tokens = b.query_start[seq + 1] - w.first_token;
  w.rows = tokens * per_token;
  w.pos_of_first = b.context_lens[seq] - tokens;
  const int from = min(group < 0 ? 0 : max(b.shared_lens[group], 0), context);
  // splits begin at whole tiles, counted from the first own key's
  const int start = from / kTileKeys * kTileKeys;
  const int per_split = max((context - start + b.own_splits - 1) / b.own_splits, split_keys(ROWS));
  const int whole_pairs = (per_split + 2 * kTileKeys - 1) / (2 * kTileKeys) * 2 * kTileKeys;
  w.first_key = min(max(start + split * whole_pairs, from), context);
  w.end_key = min(start + (split + 1) * whole_pairs, context);
  w.causal = true;
  w.table = b.block_table + static_cast<int64_t>(seq) * b.max_blocks;
  for (int tile = first_tile; tile * 16 < w.rows; tile += b.own_tiles) {
    w.row0 = tile * 16;
    w.slot = b.shared_splits + split;
    if (w.first_key >= w.end_key) {
      leave_empty(b, w, 16, partial_ml);
    } else {
      if (tile != first_tile) __syncthreads();      // what the tile before left in LDS is read
      walk_direct<T, D, 1, WAVES>(b, w, q, key_pool, value_pool, partial_o, partial_ml, reinterpret_cast<float*>(lds));
    }
    if (group < 0 && split == 0) {
      // no workgroup makes shared parts for a sequence without a group: they are empty
      for (w.slot = 0; w.slot < b.shared_splits; ++w.slot) leave_empty(b, w, 16, partial_ml);
    }
  }
}

// Short sequences: a workgroup walks all keys of a sequence, the shared ones through the table of
// the group's first and then its own, so that no parts are left and nothing is joined: one launch
// instead of two, which is what an eager call of this size costs (times at ops.WHOLE_BYTES).
// Workgroups: (kv head, tile of 16 rows, sequence).
constexpr int kWholeWaves = 8;

template <typename T, int D>
__global__ __launch_bounds__(kWholeWaves * ms::kWave) MS_WAVES_PER_EU(2, 2) void attention_shared_whole_kernel(
    Sizes sizes, const int32_t* __restrict__ block_table, const int32_t* __restrict__ query_start,
    const int32_t* __restrict__ context_lens, const int32_t* __restrict__ group_start,
    const int32_t* __restrict__ shared_lens, const T* __restrict__ q, const T* __restrict__ key_pool,
    const T* __restrict__ value_pool, T* __restrict__ out) {
  using Op = Operand<T>;
  constexpr int KS = Pair<T, D>::KS, CS = D / 16;
  const Batch b{sizes, block_table, query_start, context_lens, group_start, shared_lens};
  __shared__ __align__(16) float lds[direct_lds_bytes<D, kWholeWaves>() / sizeof(float)];
  const int lane = threadIdx.x & 63, wave = ms::uniform(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int per_token = b.num_q_heads / b.num_kv_heads;
  const int kv_head = blockIdx.x % b.num_kv_heads;
  const int first_tile = blockIdx.x / b.num_kv_heads % b.own_tiles;
  const int seq = blockIdx.x / b.num_kv_heads / b.own_tiles;
  const int group = b.num_groups > 1 ? group_of_sequence(b, seq) : seq >= b.group_start[0] && seq < b.group_start[1] ? 0 : -1;
  const int context = min(max(b.context_lens[seq], 0), b.most_keys);
  const int first_token = b.query_start[seq], tokens = b.query_start[seq + 1] - first_token;
  const int rows = tokens * per_token, pos_of_first = b.context_lens[seq] - tokens;
  const int shared = group < 0 ? 0 : min(max(b.shared_lens[group], 0), b.most_keys);
  const int from = min(shared, context), start = from / kTileKeys;
  const int32_t* own_table = b.block_table + static_cast<int64_t>(seq) * b.max_blocks;
  const int32_t* shared_table = group < 0 ? own_table : b.block_table + static_cast<int64_t>(b.group_start[group]) * b.max_blocks;
  // pairs of tiles: those of the shared keys, then those of its own
  const int shared_tiles = (shared + kTileKeys - 1) / kTileKeys, own_end = (context + kTileKeys - 1) / kTileKeys;
  const int shared_pairs = (shared_tiles + 1) / 2;
  const int pairs = shared_pairs + (context > from ? (own_end - start + 1) / 2 : 0);
  const auto tile_of = [&](int pair) { return pair < shared_pairs ? 2 * pair : start + 2 * (pair - shared_pairs); };
  const auto pages_of = [&](int pair) {
    const bool of_group = pair < shared_pairs || context <= from;
    return ms::find_pair_pages(min(tile_of(pair), (of_group ? shared_tiles : own_end) - 1), of_group ? shared_tiles : own_end,
                               of_group ? shared_table : own_table, b.block_size);
  };
  const auto head_of = [&](int row, int& token) {
    token = row / per_token;
    return kv_head * per_token + row - token * per_token;
  };
  float* m_s = lds;                                      // [waves][16]
  float* l_s = m_s + kWholeWaves * 16;                   // [waves][16]
  float* o_s = l_s + kWholeWaves * 16;                   // [waves][16][D + 4]
  constexpr int ROW = D + 4;

  for (int tile = first_tile; tile * 16 < rows; tile += b.own_tiles) {
    const int row = tile * 16 + r;
    int token;
    const int head = head_of(row, token);
    const bool live = row < rows;
    typename Op::V8 q_reg[KS];
    const T* q_row = q + (static_cast<int64_t>(first_token + token) * b.num_q_heads + head) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d0 = 32 * s + 8 * g;
      q_reg[s] = live && d0 < D ? *reinterpret_cast<const typename Op::V8*>(q_row + d0) : Op::zero8();
    }
    RowState<D> st;
#pragma unroll
    for (int c = 0; c < CS; ++c) st.o[c] = floatx4{0.f, 0.f, 0.f, 0.f};
    st.run_max = -INFINITY;
    st.run_sum = 0.f;
    const int own_last = live ? min(context - 1, pos_of_first + token) : -1, shared_last = live ? shared - 1 : -1;
    const auto use = [&](Pair<T, D>& pair, int p) {
      const bool of_group = p < shared_pairs;
      const int at = tile_of(p), first = of_group ? 0 : from, end = of_group ? shared : context;
      if (at * kTileKeys < first || (at + 2) * kTileKeys > end) clear_outside<T, D>(pair, at, first, end, g);
      consume<T, D>(st, pair, q_reg, at, first, of_group ? shared_last : own_last, b.scale * Op::kScale, g);
    };
    int p = wave;
    if (p < pairs) {
      // (a pair behind the end is looked up as the last one, and not loaded)
      ms::PairPages pages = pages_of(p);
      const auto load = [&](Pair<T, D>& pair, int of) {
        load_pair<T, D>(pair, b, pages, key_pool, value_pool, kv_head, g, r);
        pages = pages_of(of + kWholeWaves);
      };
      if constexpr (sizeof(T) == 2) {
        Pair<T, D> ping, pong;
        load(ping, p);
        while (true) {
          int next = p + kWholeWaves;
          if (next < pairs) load(pong, next);
          use(ping, p);
          p = next;
          if (p >= pairs) break;
          next = p + kWholeWaves;
          if (next < pairs) load(ping, next);
          use(pong, p);
          p = next;
          if (p >= pairs) break;
        }
      } else {
        for (; p < pairs; p += kWholeWaves) {
          Pair<T, D> pair;
          load(pair, p);
          use(pair, p);
        }
      }
    }
    if (tile != first_tile) __syncthreads();      // what the tile before left in LDS is read
    if (g == 0) {
      m_s[wave * 16 + r] = st.run_max;
      l_s[wave * 16 + r] = st.run_sum;
    }
#pragma unroll
    for (int c = 0; c < CS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o_s[(wave * 16 + 4 * g + e) * ROW + 16 * c + r] = st.o[c][e];
    __syncthreads();
    constexpr int kAtOnce = kWholeWaves * ms::kWave / (D / 4);      // rows that the threads finish at once
    const int d = 4 * (threadIdx.x % (D / 4));
    for (int in_tile = threadIdx.x / (D / 4); in_tile < 16 && tile * 16 + in_tile < rows; in_tile += kAtOnce) {
      if (threadIdx.x >= kAtOnce * (D / 4)) break;                  // threads that are left over
      float mx = -INFINITY;
#pragma unroll
      for (int v = 0; v < kWholeWaves; ++v) mx = fmaxf(mx, m_s[v * 16 + in_tile]);
      const float shift = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f;
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < kWholeWaves; ++v) {
        const float factor = Op::weight(m_s[v * 16 + in_tile] - shift);      // 0 for a wave without keys
        const floatx4 o = *reinterpret_cast<const floatx4*>(&o_s[(v * 16 + in_tile) * ROW + d]);
        sum += factor * l_s[v * 16 + in_tile];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(o[e], factor, acc[e]);
      }
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      int token_of_row;
      const int head_of_row = head_of(tile * 16 + in_tile, token_of_row);
      T* to = out + (static_cast<int64_t>(first_token + token_of_row) * b.num_q_heads + head_of_row) * D + d;
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e] = ms::from_float<T>(acc[e] * inv);
    }
  }
  // tokens before the first sequence and behind the last
  if (first_tile == 0 && (seq == 0 || seq == b.num_seqs - 1)) {
    const auto clear = [&](int token0, int token1) {
      const int values = per_token * D;
      for (int64_t i = threadIdx.x; i < static_cast<int64_t>(max(token1 - token0, 0)) * values; i += kWholeWaves * ms::kWave) {
        const int64_t token = token0 + i / values;
        out[(token * b.num_q_heads + kv_head * per_token) * D + i % values] = ms::from_float<T>(0.f);
      }
    };
    if (seq == 0) clear(0, min(b.query_start[0], b.num_tokens));
    if (seq == b.num_seqs - 1) clear(max(b.query_start[b.num_seqs], 0), b.num_tokens);
  }
}

// Joins the parts of a row, a wave each.  A row that saw no key gives zeros, and so do the
// rows of tokens before the first sequence and behind the last.
constexpr int kJoinWaves = 4;

template <typename T, int D>
__global__ __launch_bounds__(kJoinWaves * ms::kWave) void attention_shared_join_kernel(const float* __restrict__ partial_o,
                                                                                 const float* __restrict__ partial_ml,
                                                                                 const int32_t* __restrict__ query_start,
                                                                                 T* __restrict__ out, int64_t rows,
                                                                                 int num_seqs, int num_q_heads, int slots) {
  constexpr int kLanes = D / 4;                       // a part's output, four values a lane
  constexpr int kAtOnce = ms::kWave / kLanes;         // parts that the wave reads with one instruction
  constexpr int kDeep = 8;                            // of those instructions in flight
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kJoinWaves + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int group = min(lane / kLanes, kAtOnce), d = 4 * (lane % kLanes);
  const bool reads = group < kAtOnce;
  const float* from = partial_o + row * slots * D + d;
  // the first parts are on their way while the weights are made; what an empty part holds is not used
  floatx4 ahead[kDeep];
#pragma unroll
  for (int u = 0; u < kDeep; ++u)
    ahead[u] = *reinterpret_cast<const floatx4*>(from + static_cast<int64_t>(min(group + u * kAtOnce, slots - 1)) * D);
  const int64_t token = row / num_q_heads;
  const bool live = token >= query_start[0] && token < query_start[num_seqs];
  float m[2], mx = -INFINITY, l[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int s = lane + 64 * h;
    const bool here = live && s < slots;
    m[h] = here ? partial_ml[2 * (row * slots + s)] : -INFINITY;
    l[h] = here ? partial_ml[2 * (row * slots + s) + 1] : 0.f;
    mx = fmaxf(mx, m[h]);
  }
  mx = ms::wave_max(mx);
  const float shift = mx == -INFINITY ? 0.f : mx;
  float total = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    m[h] = Operand<T>::weight(m[h] - shift);      // 0 for a part without keys
    total += m[h] * l[h];
  }
  total = ms::wave_sum(total);
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  floatx4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int first = 0; first < slots; first += kDeep * kAtOnce) {
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int s = first + group + u * kAtOnce;
      const float near = __shfl(m[0], s & 63, ms::kWave), far = __shfl(m[1], s & 63, ms::kWave);
      const float factor = s >= slots || !reads ? 0.f : s < 64 ? near : far;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = factor > 0.f ? fmaf(factor, ahead[u][e], acc[e]) : acc[e];
    }
    if (first + kDeep * kAtOnce < slots) {
#pragma unroll
      for (int u = 0; u < kDeep; ++u)
        ahead[u] = *reinterpret_cast<const floatx4*>(
            from + static_cast<int64_t>(min(first + (kDeep + u) * kAtOnce + group, slots - 1)) * D);
    }
  }
  // the lanes' shares of a value, added up in the order of the groups
  floatx4 sum = acc;
#pragma unroll
  for (int other = 1; other < kAtOnce; ++other)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += __shfl(acc[e], (lane + other * kLanes) & 63, ms::kWave);
  if (lane >= kLanes) return;
  T* to = out + row * D + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) to[e] = ms::from_float<T>(sum[e] * inv);
}

template <typename T, int D>
int launch(const Batch& b, const void* q, const void* key_pool, const void* value_pool, void* out, void* partial_o,
           void* partial_ml, hipStream_t stream) {
  if (b.shared_splits == 0) {
    hipLaunchKernelGGL((attention_shared_whole_kernel<T, D>),
                       dim3(static_cast<unsigned>(b.num_seqs) * b.own_tiles * b.num_kv_heads), dim3(kWholeWaves * ms::kWave), 0,
                       stream, static_cast<const Sizes&>(b), b.block_table, b.query_start, b.context_lens, b.group_start,
                       b.shared_lens, static_cast<const T*>(q), static_cast<const T*>(key_pool),
                       static_cast<const T*>(value_pool), static_cast<T*>(out));
    MS_CHECK_LAUNCH("attention_shared_prefix (whole)");
    return 0;
  }
  const int units = b.num_kv_heads * b.shared_splits;
  const int64_t items = static_cast<int64_t>((units + kXcds - 1) / kXcds * kXcds) * b.shared_tiles +
                        static_cast<int64_t>(b.num_seqs) * b.own_tiles * b.own_splits * b.num_kv_heads;
  MS_REQUIRE(items < (1LL << 31) / (8 * ms::kWave), "attention_shared_prefix: the batch is too large");
#define MS_SHARED_ROWS(ROWS)                                                                                   \
  hipLaunchKernelGGL((attention_shared_kernel<T, D, ROWS>), dim3(static_cast<unsigned>(items)),                \
                     dim3(waves_of(ROWS) * ms::kWave), 0, stream, static_cast<const Sizes&>(b), b.block_table, \
                     b.query_start, b.context_lens, b.group_start, b.shared_lens, static_cast<const T*>(q),    \
                     static_cast<const T*>(key_pool), static_cast<const T*>(value_pool),                       \
                     static_cast<float*>(partial_o), static_cast<float*>(partial_ml))
  if constexpr (sizeof(T) == 2) {
    if (b.tile_rows == 128) MS_SHARED_ROWS(128);
    else if (b.tile_rows == 64) MS_SHARED_ROWS(64);
    else if (b.tile_rows == 32) MS_SHARED_ROWS(32);
    else MS_SHARED_ROWS(16);
  } else {
    MS_SHARED_ROWS(16);
  }
#undef MS_SHARED_ROWS
  MS_CHECK_LAUNCH("attention_shared_prefix");
  const int64_t rows = static_cast<int64_t>(b.num_tokens) * b.num_q_heads;
  hipLaunchKernelGGL((attention_shared_join_kernel<T, D>), dim3(static_cast<unsigned>((rows + kJoinWaves - 1) / kJoinWaves)),
                     dim3(kJoinWaves * ms::kWave), 0, stream, static_cast<const float*>(partial_o),
                     static_cast<const float*>(partial_ml), b.query_start, static_cast<T*>(out), rows, b.num_seqs,
                     b.num_q_heads, b.shared_splits + b.own_splits);
  MS_CHECK_LAUNCH("attention_shared_prefix (join)");
  return 0;
}

template <typename T>
int run_shared(const Batch& b, int head_dim, const void* q, const void* key_pool, const void* value_pool, void* out,
               void* partial_o, void* partial_ml, hipStream_t stream) {
#define MS_SHARED_CASE(DIM) \
  case DIM:                 \
    return launch<T, DIM>(b, q, key_pool, value_pool, out, partial_o, partial_ml, stream);
  switch (head_dim) {
    MS_SHARED_CASE(16) MS_SHARED_CASE(32) MS_SHARED_CASE(48) MS_SHARED_CASE(64) MS_SHARED_CASE(80)
    MS_SHARED_CASE(96) MS_SHARED_CASE(112) MS_SHARED_CASE(128)
    default:
      return ms_fail("attention_shared_prefix: head_dim %d", head_dim);
  }
#undef MS_SHARED_CASE
}

}  // namespace

// Whether ms_attention_shared_prefix takes this geometry: head sizes in steps of 16 up to
// 128, pages of a multiple of 16 keys.
extern "C" int ms_attention_shared_prefix_supported(int head_dim, int block_size) {
  return head_dim >= 16 && head_dim <= 128 && head_dim % 16 == 0 && block_size > 0 && block_size % kTileKeys == 0;
}

// q, out: [num_tokens, num_q_heads, head_dim]; pools as for ms_attention_decode; query_start
// [num_seqs + 1], context_lens [num_seqs], group_start [num_groups + 1], shared_lens
// [num_groups]; partial_o: float [num_tokens, num_q_heads, shared_splits + own_splits,
// head_dim]; partial_ml: the same with 2 in head_dim's place.  rows_per_tile: 16, 32, 64
// or 128 rows of a group a workgroup (32-bit storage: 16); own_tiles: workgroups that share
// a sequence's tiles of 16 rows.  With 0 shared and 0 own splits every such workgroup walks all
// keys of its sequence, and the workspaces are not used.
extern "C" int ms_attention_shared_prefix(const void* q, const void* key_pool, const void* value_pool,
                                          const void* block_table, const void* query_start, const void* context_lens,
                                          const void* group_start, const void* shared_lens, void* out, void* partial_o,
                                          void* partial_ml, int num_tokens, int num_seqs, int num_groups,
                                          int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                                          int max_blocks, float scale, int rows_per_tile, int shared_splits,
                                          int own_tiles, int own_splits, int dtype, hipStream_t stream) {
  MS_REQUIRE(num_tokens > 0 && num_seqs > 0 && num_groups > 0 && max_blocks > 0,
             "attention_shared_prefix: nothing to do (%d tokens, %d sequences, %d groups)", num_tokens, num_seqs, num_groups);
  MS_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
             "attention_shared_prefix: %d query heads are not a multiple of %d kv heads", num_q_heads, num_kv_heads);
  MS_REQUIRE(ms_attention_shared_prefix_supported(head_dim, block_size),
             "attention_shared_prefix: head_dim %d (multiples of 16 up to 128) or block_size %d (multiples of 16) is not supported",
             head_dim, block_size);
  MS_REQUIRE(rows_per_tile == 16 || (dtype == MS_BF16 && (rows_per_tile == 32 || rows_per_tile == 64 || rows_per_tile == 128)),
             "attention_shared_prefix: tiles of %d rows", rows_per_tile);
  MS_REQUIRE(static_cast<int64_t>(num_kv_heads) * block_size * head_dim < (int64_t{1} << 31),
             "attention_shared_prefix: a page of %d kv heads x %d keys x %d is too large", num_kv_heads, block_size, head_dim);
  MS_REQUIRE(own_tiles >= 1 && ((shared_splits == 0 && own_splits == 0) ||
                                (shared_splits >= 1 && shared_splits <= kMaxSplits && own_splits >= 1 && own_splits <= kMaxSplits)),
             "attention_shared_prefix: %d and %d splits are outside 1..%d", shared_splits, own_splits, kMaxSplits);
  MS_REQUIRE(dtype == MS_F32 || dtype == MS_BF16, "attention_shared_prefix: unknown dtype %d", dtype);
  const int64_t rows = static_cast<int64_t>(num_tokens) * (num_q_heads / num_kv_heads);
  MS_REQUIRE(rows < (1LL << 31) - 4096 && rows / rows_per_tile + num_groups < (1LL << 24) / std::max(shared_splits, 1) &&
                 static_cast<int64_t>(num_seqs) * own_tiles * std::max(own_splits, 1) < (1LL << 22) / num_kv_heads,
             "attention_shared_prefix: the batch is too large");
  Batch b;
  b.block_table = static_cast<const int32_t*>(block_table);
  b.query_start = static_cast<const int32_t*>(query_start);
  b.context_lens = static_cast<const int32_t*>(context_lens);
  b.group_start = static_cast<const int32_t*>(group_start);
  b.shared_lens = static_cast<const int32_t*>(shared_lens);
  b.num_tokens = num_tokens;
  b.num_seqs = num_seqs;
  b.num_groups = num_groups;
  b.num_q_heads = num_q_heads;
  b.num_kv_heads = num_kv_heads;
  b.block_size = block_size;
  b.max_blocks = max_blocks;
  const int64_t named = static_cast<int64_t>(max_blocks) * block_size;
  b.most_keys = named < (1LL << 30) ? static_cast<int>(named) : 1 << 30;
  b.scale = scale;
  // every group has at most one tile that is not full
  b.tile_rows = rows_per_tile;
  b.shared_tiles = num_groups == 1 ? static_cast<int>((rows + rows_per_tile - 1) / rows_per_tile)
                                   : static_cast<int>(rows / rows_per_tile) + num_groups;
  b.shared_splits = shared_splits;
  b.own_tiles = own_tiles;
  b.own_splits = own_splits;
  if (dtype == MS_F32)
    return run_shared<float>(b, head_dim, q, key_pool, value_pool, out, partial_o, partial_ml, stream);
  return run_shared<bf16>(b, head_dim, q, key_pool, value_pool, out, partial_o, partial_ml, stream);
}
