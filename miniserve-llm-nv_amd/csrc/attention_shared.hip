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
// keys behind them.  One kernel makes the (m, l, O) of all parts, a second joins them.
//
// A workgroup of 4 waves takes a tile of 16 R rows of one kv head (rows of the whole
// group for shared keys, of one sequence for its own) and a range of keys, which its waves
// walk in pairs of 16-key tiles, each wave pairs of its own, with its own running maximum,
// sum and output (32-bit); they are joined through LDS at the end.  Operands come from the
// cache as it lies (see attention_tiles.hpp); 32-bit storage runs the same walk on the
// 32-bit matrix instruction.
#include "mfma.hpp"

namespace {

using ms::bf16;
using ms::bf16x4;
using ms::bf16x8;
using ms::floatx4;

typedef float floatx8 __attribute__((ext_vector_type(8)));

constexpr int kTileKeys = 16;
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * ms::kWave;
constexpr int kMaxSplits = 64;      // of the shared keys, and of a sequence's own

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
  // the weights are rounded to the storage type for the second product, as the reference does
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

struct Batch {
  const int32_t* __restrict__ block_table;
  const int32_t* __restrict__ query_start;
  const int32_t* __restrict__ context_lens;
  const int32_t* __restrict__ group_start;
  const int32_t* __restrict__ shared_lens;
  int num_tokens, num_seqs, num_groups, num_q_heads, num_kv_heads, block_size, max_blocks;
  float scale;
  int shared_tiles, shared_splits, own_tiles, own_splits;
};

// Rows and keys of one workgroup, the same in all its lanes.
struct Work {
  int first_token;        // of the rows' segment (a group's or a sequence's tokens, which are contiguous)
  int rows, row0;         // rows of the segment, first row of this tile
  int first_key, end_key;         // keys [first_key, end_key) of this split
  int pos_of_first;       // row of token i sees keys <= pos_of_first + i; for shared keys every row sees all
  bool causal;
  const int32_t* table;
  int slot;
};

// The group's part of a flat list of tiles: every group has ceil(rows / tile_rows) of them.
__device__ __forceinline__ bool find_group_tile(const Batch& b, int tile, int group_rows_per_token, int tile_rows,
                                                int& group, int& local) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int g0 = 0; g0 < b.num_groups; g0 += ms::kWave) {
    const int g = g0 + lane;
    int tiles = 0;
    if (g < b.num_groups) {
      const int tokens = b.query_start[b.group_start[g + 1]] - b.query_start[b.group_start[g]];
      tiles = (tokens * group_rows_per_token + tile_rows - 1) / tile_rows;
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

template <typename T, int D>
__device__ __forceinline__ void load_pair(Pair<T, D>& pair, const Batch& b, const Work& w, int tile, int last_tile,
                                          const T* __restrict__ key_pool, const T* __restrict__ value_pool, int kv_head,
                                          int g, int r) {
  using Op = Operand<T>;
  const int key_a = tile * kTileKeys;
  const int key_b = min(tile + 1, last_tile) * kTileKeys;       // without a second tile the first is read twice
  const int page_a = key_a / b.block_size, page_b = key_b / b.block_size;
  const int off_a = key_a - page_a * b.block_size, off_b = key_b - page_b * b.block_size;
  const int64_t slab_a = static_cast<int64_t>(w.table[page_a]) * b.num_kv_heads + kv_head;
  const int64_t slab_b = static_cast<int64_t>(w.table[page_b]) * b.num_kv_heads + kv_head;
  const T* k_row_a = key_pool + (slab_a * b.block_size + off_a + r) * D;
  const T* k_row_b = key_pool + (slab_b * b.block_size + off_b + r) * D;
  const T* v_a = value_pool + slab_a * D * b.block_size + off_a + 4 * g;
  const T* v_b = value_pool + slab_b * D * b.block_size + off_b + 4 * g;
#pragma unroll
  for (int s = 0; s < Pair<T, D>::KS; ++s) {
    const int d0 = 32 * s + 8 * g;
    pair.k_a[s] = d0 < D ? *reinterpret_cast<const typename Op::V8*>(k_row_a + d0) : Op::zero8();
    pair.k_b[s] = d0 < D ? *reinterpret_cast<const typename Op::V8*>(k_row_b + d0) : Op::zero8();
  }
#pragma unroll
  for (int c = 0; c < Pair<T, D>::CS; ++c) {
    const int64_t d = 16 * c + r;
    pair.v_a[c] = *reinterpret_cast<const typename Op::V4*>(v_a + d * b.block_size);
    pair.v_b[c] = *reinterpret_cast<const typename Op::V4*>(v_b + d * b.block_size);
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

// 16 R rows against the keys of ``w``; leaves (m, l, O) of the part in the rows' slots.
template <typename T, int D, int R>
__device__ void walk(const Batch& b, const Work& w, const T* __restrict__ q, const T* __restrict__ key_pool,
                     const T* __restrict__ value_pool, float* __restrict__ partial_o, float* __restrict__ partial_ml,
                     float* __restrict__ lds) {
  using Op = Operand<T>;
  constexpr int KS = Pair<T, D>::KS, CS = D / 16;
  const int lane = threadIdx.x & 63;
  const int wave = ms::uniform(threadIdx.x >> 6);
  const int g = lane >> 4, r = lane & 15;
  const int kv_head = blockIdx.y;
  const int per_token = b.num_q_heads / b.num_kv_heads;
  const int slots = b.shared_splits + b.own_splits;

  typename Op::V8 q_reg[R][KS];
  int last[R];
  RowState<D> st[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = w.row0 + 16 * i + r;
    const int token = row / per_token, head = kv_head * per_token + row % per_token;
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

  if (w.first_key < w.end_key) {
    const int first_tile = w.first_key / kTileKeys, last_tile = (w.end_key - 1) / kTileKeys;
    for (int t = first_tile + 2 * wave; t <= last_tile; t += 2 * kWaves) {
      Pair<T, D> pair;
      load_pair<T, D>(pair, b, w, t, last_tile, key_pool, value_pool, kv_head, g, r);
      if (t * kTileKeys < w.first_key || (t + 2) * kTileKeys > w.end_key) {
        // keys outside the range may never have been written: their values must not meet a zero weight
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int ka = t * kTileKeys + 4 * g + e, kb = ka + kTileKeys;
#pragma unroll
          for (int c = 0; c < CS; ++c) {
            if (ka < w.first_key || ka >= w.end_key) Op::clear(pair.v_a[c], e);
            if (kb < w.first_key || kb >= w.end_key) Op::clear(pair.v_b[c], e);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i)
        consume<T, D>(st[i], pair, q_reg[i], t, w.first_key, last[i], b.scale * Op::kScale, g);
    }
  }

  // ---- the waves' states, joined 16 rows at a time -------------------------------------
  float* m_s = lds;                                  // [kWaves][16]
  float* l_s = m_s + kWaves * 16;                    // [kWaves][16]
  float* o_s = l_s + kWaves * 16;                    // [kWaves - 1][16][D]
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i > 0) __syncthreads();
    if (g == 0) {
      m_s[wave * 16 + r] = st[i].run_max;
      l_s[wave * 16 + r] = st[i].run_sum;
    }
    if (wave > 0) {
#pragma unroll
      for (int c = 0; c < CS; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o_s[((wave - 1) * 16 + 4 * g + e) * D + 16 * c + r] = st[i].o[c][e];
    }
    __syncthreads();
    if (wave != 0) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int in_tile = 4 * g + e;
      const int row = w.row0 + 16 * i + in_tile;
      if (row >= w.rows) continue;
      float mx = -INFINITY;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) mx = fmaxf(mx, m_s[v * 16 + in_tile]);
      const float shift = mx == -INFINITY ? 0.f : mx;
      float factor[kWaves], sum = 0.f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        // 0 for a wave without keys; a NaN among its scores stays one in its sum
        factor[v] = Op::weight(m_s[v * 16 + in_tile] - shift);
        sum += factor[v] * l_s[v * 16 + in_tile];
      }
      const int token = row / per_token, head = kv_head * per_token + row % per_token;
      const int64_t slot = (static_cast<int64_t>(w.first_token + token) * b.num_q_heads + head) * slots + w.slot;
      if (r == 0) {
        partial_ml[2 * slot] = mx;
        partial_ml[2 * slot + 1] = sum;
      }
#pragma unroll
      for (int c = 0; c < CS; ++c) {
        float acc = st[i].o[c][e] * factor[0];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) acc += o_s[((v - 1) * 16 + in_tile) * D + 16 * c + r] * factor[v];
        partial_o[slot * D + 16 * c + r] = acc;
      }
    }
  }
}

// Items: first the shared keys, (tile of rows, split) each; then the sequences' own keys,
// (sequence, tile of rows, split) each.
template <typename T, int D, int R>
__global__ __launch_bounds__(kThreads) void attention_shared_kernel(Batch b, const T* __restrict__ q,
                                                                    const T* __restrict__ key_pool,
                                                                    const T* __restrict__ value_pool,
                                                                    float* __restrict__ partial_o,
                                                                    float* __restrict__ partial_ml) {
  __shared__ float lds[2 * kWaves * 16 + (kWaves - 1) * 16 * D];
  const int per_token = b.num_q_heads / b.num_kv_heads;
  int item = blockIdx.x;
  Work w;
  const int shared_items = b.shared_tiles * b.shared_splits;
  if (item < shared_items) {
    const int tile = item / b.shared_splits, split = item - tile * b.shared_splits;
    int group, local;
    if (!find_group_tile(b, tile, per_token, 16 * R, group, local)) return;
    const int first_seq = b.group_start[group];
    w.first_token = b.query_start[first_seq];
    w.rows = (b.query_start[b.group_start[group + 1]] - w.first_token) * per_token;
    w.row0 = local * 16 * R;
    const int keys = max(b.shared_lens[group], 0);
    const int pairs = (keys + 2 * kTileKeys - 1) / (2 * kTileKeys);
    const int per_split = (pairs + b.shared_splits - 1) / b.shared_splits * 2 * kTileKeys;
    w.first_key = min(split * per_split, keys);
    w.end_key = min(w.first_key + per_split, keys);
    w.causal = false;
    w.pos_of_first = 0;
    w.table = b.block_table + static_cast<int64_t>(first_seq) * b.max_blocks;
    w.slot = split;
    walk<T, D, R>(b, w, q, key_pool, value_pool, partial_o, partial_ml, lds);
    return;
  }
  item -= shared_items;
  const int seq = item / (b.own_tiles * b.own_splits);
  item -= seq * b.own_tiles * b.own_splits;
  const int first_tile = item / b.own_splits, split = item - first_tile * b.own_splits;
  const int group = group_of_sequence(b, seq);
  const int context = b.context_lens[seq];
  w.first_token = b.query_start[seq];
  const int tokens = b.query_start[seq + 1] - w.first_token;
  w.rows = tokens * per_token;
  w.pos_of_first = context - tokens;
  const int from = min(group < 0 ? 0 : max(b.shared_lens[group], 0), max(context, 0));
  // splits begin at a pair of tiles counted from the first own key's tile
  const int start = from / kTileKeys * kTileKeys;
  const int pairs = (max(context, 0) - start + 2 * kTileKeys - 1) / (2 * kTileKeys);
  const int per_split = (pairs + b.own_splits - 1) / b.own_splits * 2 * kTileKeys;
  w.first_key = min(max(start + split * per_split, from), max(context, 0));
  w.end_key = min(start + (split + 1) * per_split, max(context, 0));
  w.causal = true;
  w.table = b.block_table + static_cast<int64_t>(seq) * b.max_blocks;
  w.slot = b.shared_splits + split;
  for (int tile = first_tile; tile * 16 < w.rows; tile += b.own_tiles) {
    if (tile != first_tile) __syncthreads();
    w.row0 = tile * 16;
    walk<T, D, 1>(b, w, q, key_pool, value_pool, partial_o, partial_ml, lds);
    if (group < 0 && split == 0) {
      // no workgroup makes shared parts for a sequence without a group: they are empty
      for (int i = threadIdx.x; i < 16 * b.shared_splits; i += kThreads) {
        const int row = w.row0 + i / b.shared_splits;
        if (row >= w.rows) break;
        const int64_t slot = (static_cast<int64_t>(w.first_token + row / per_token) * b.num_q_heads +
                              blockIdx.y * per_token + row % per_token) * (b.shared_splits + b.own_splits) +
                             i % b.shared_splits;
        partial_ml[2 * slot] = -INFINITY;
        partial_ml[2 * slot + 1] = 0.f;
      }
    }
  }
}

// Joins the parts of a row, a wave each.  A row that saw no key gives zeros, and so do the
// rows of tokens behind the last sequence.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_shared_join_kernel(const float* __restrict__ partial_o,
                                                                         const float* __restrict__ partial_ml,
                                                                         const int32_t* __restrict__ query_start,
                                                                         T* __restrict__ out, int64_t rows,
                                                                         int num_seqs, int num_q_heads, int head_dim,
                                                                         int slots) {
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  if (row >= rows) return;
  const bool live = row / num_q_heads < query_start[num_seqs];
  float m[2], l[2], mx = -INFINITY;
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
  for (int d = lane; d < head_dim; d += ms::kWave) {
    float acc = 0.f;
    if (live) {
#pragma unroll 4
      for (int s = 0; s < slots; ++s) {
        const float factor = __shfl(s < 64 ? m[0] : m[1], s & 63, ms::kWave);
        const float value = partial_o[(row * slots + s) * head_dim + d];
        acc = factor > 0.f ? fmaf(factor, value, acc) : acc;      // the output of an empty part was never written
      }
    }
    out[row * head_dim + d] = ms::from_float<T>(acc * inv);
  }
}

template <typename T, int D>
void launch(const Batch& b, int rows_per_tile, const void* q, const void* key_pool, const void* value_pool,
            void* partial_o, void* partial_ml, hipStream_t stream) {
  const int64_t items = static_cast<int64_t>(b.shared_tiles) * b.shared_splits +
                        static_cast<int64_t>(b.num_seqs) * b.own_tiles * b.own_splits;
  const dim3 grid(static_cast<unsigned>(items), b.num_kv_heads);
#define MS_SHARED_ROWS(R)                                                                                          \
  hipLaunchKernelGGL((attention_shared_kernel<T, D, R>), grid, dim3(kThreads), 0, stream, b, static_cast<const T*>(q), \
                     static_cast<const T*>(key_pool), static_cast<const T*>(value_pool),                           \
                     static_cast<float*>(partial_o), static_cast<float*>(partial_ml))
  if (rows_per_tile == 16) MS_SHARED_ROWS(1);
  else MS_SHARED_ROWS(2);
#undef MS_SHARED_ROWS
}

template <typename T>
int run_shared(const Batch& b, int head_dim, int rows_per_tile, const void* q, const void* key_pool,
               const void* value_pool, void* out, void* partial_o, void* partial_ml, hipStream_t stream) {
#define MS_SHARED_CASE(DIM)                                                                        \
  case DIM:                                                                                        \
    launch<T, DIM>(b, rows_per_tile, q, key_pool, value_pool, partial_o, partial_ml, stream);      \
    break;
  switch (head_dim) {
    MS_SHARED_CASE(16) MS_SHARED_CASE(32) MS_SHARED_CASE(48) MS_SHARED_CASE(64) MS_SHARED_CASE(80)
    MS_SHARED_CASE(96) MS_SHARED_CASE(112) MS_SHARED_CASE(128)
    default:
      return ms_fail("attention_shared_prefix: head_dim %d", head_dim);
  }
#undef MS_SHARED_CASE
  MS_CHECK_LAUNCH("attention_shared_prefix");
  const int64_t rows = static_cast<int64_t>(b.num_tokens) * b.num_q_heads;
  hipLaunchKernelGGL((attention_shared_join_kernel<T>), dim3(static_cast<unsigned>((rows + kWaves - 1) / kWaves)),
                     dim3(kThreads), 0, stream, static_cast<const float*>(partial_o),
                     static_cast<const float*>(partial_ml), b.query_start, static_cast<T*>(out), rows, b.num_seqs,
                     b.num_q_heads, head_dim, b.shared_splits + b.own_splits);
  MS_CHECK_LAUNCH("attention_shared_prefix (join)");
  return 0;
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
// head_dim]; partial_ml: the same with 2 in head_dim's place.  rows_per_tile: 16 or 32 rows
// of a group a workgroup; own_tiles: workgroups that share a sequence's tiles of 16 rows.
extern "C" int ms_attention_shared_prefix(const void* q, const void* key_pool, const void* value_pool,
                                          const void* block_table, const void* query_start, const void* context_lens,
                                          const void* group_start, const void* shared_lens, void* out, void* partial_o,
                                          void* partial_ml, int num_tokens, int num_seqs, int num_groups,
                                          int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                                          int max_blocks, float scale, int rows_per_tile, int shared_splits,
                                          int own_tiles, int own_splits, int dtype, hipStream_t stream) {
  MS_REQUIRE(num_tokens > 0 && num_seqs > 0 && num_groups > 0 && max_blocks > 0,
             "attention_shared_prefix: nothing to do (%d tokens, %d sequences, %d groups)", num_tokens, num_seqs, num_groups);
  MS_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_kv_heads <= 65535 && num_q_heads % num_kv_heads == 0,
             "attention_shared_prefix: %d query heads are not a multiple of %d kv heads", num_q_heads, num_kv_heads);
  MS_REQUIRE(ms_attention_shared_prefix_supported(head_dim, block_size),
             "attention_shared_prefix: head_dim %d (multiples of 16 up to 128) or block_size %d (multiples of 16) is not supported",
             head_dim, block_size);
  MS_REQUIRE(rows_per_tile == 16 || rows_per_tile == 32, "attention_shared_prefix: tiles of %d rows", rows_per_tile);
  MS_REQUIRE(shared_splits >= 1 && shared_splits <= kMaxSplits && own_splits >= 1 && own_splits <= kMaxSplits && own_tiles >= 1,
             "attention_shared_prefix: %d and %d splits are outside 1..%d", shared_splits, own_splits, kMaxSplits);
  MS_REQUIRE(dtype == MS_F32 || dtype == MS_BF16, "attention_shared_prefix: unknown dtype %d", dtype);
  const int64_t rows = static_cast<int64_t>(num_tokens) * (num_q_heads / num_kv_heads);
  MS_REQUIRE(rows < (1LL << 31) - 4096 && rows / rows_per_tile + num_groups < (1LL << 24) / shared_splits &&
                 static_cast<int64_t>(num_seqs) * own_tiles * own_splits < (1LL << 24),
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
  b.scale = scale;
  // every group has at most one tile that is not full
  b.shared_tiles = static_cast<int>(rows / rows_per_tile) + num_groups;
  b.shared_splits = shared_splits;
  b.own_tiles = own_tiles;
  b.own_splits = own_splits;
  if (dtype == MS_F32)
    return run_shared<float>(b, head_dim, rows_per_tile, q, key_pool, value_pool, out, partial_o, partial_ml, stream);
  return run_shared<bf16>(b, head_dim, rows_per_tile, q, key_pool, value_pool, out, partial_o, partial_ml, stream);
}
