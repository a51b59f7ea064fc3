// Drafted tokens against the target's probabilities.  A request brings rows of the target's
// 32-bit logits, one for each of its drafted tokens x_0 .. x_{k-1} and one more; with p_i the
// target's and q_i the draft's probabilities at row i:
//
//   p_i(t) = e^{(l_i(t) - M_i) / T} / Z_i,   M_i = max_t l_i(t),   Z_i = sum_t e^{(l_i(t) - M_i) / T}
//   x_i is taken while u_i q_i(x_i) < p_i(x_i)            (drafts without probabilities: q_i(x_i) = 1)
//   at the first one that is not taken, row j, the request's token is drawn from
//   w(t) = max(p_j(t) - q_j(t), 0)                         (without probabilities: p_j without x_j)
//   behind the last one from w = p_k; where no w is positive, from p_j.
//   The draw: the first t with w(0) + .. + w(t) > v (w(0) + .. + w(V-1)).
//
// Temperature 0: x_i is taken while it is the row's best token (the lowest of equals), and the
// best token of row j is the request's.  The numbers u and v are given.  A row with a NaN or an
// infinite logit ends the request there with -1, as a sampled row does.
//
// Which token comes out hangs on which side of a border a number lies, so that Z, w and their
// sums are held in 64 bits: with a vocabulary of 150,000 borders and sums that are off by a
// 32-bit rounding, about one draw in 10,000 would fall on the other side of one.
//
// Three kernels: (1) maximum, its place, and the sum of a chunk of a row; (2) how many drafts
// are taken, by every workgroup of the request for itself, and the masses of a chunk of w and
// p at the row where they end; (3) the draw: the chunk by the chunks' masses, then the token.
#include "common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / ms::kWave;
constexpr int kQuads = 4;                               // quads of elements a thread holds
constexpr int kChunk = kThreads * kQuads * 4;           // elements of a chunk

struct Batch {
  const float* __restrict__ logits;
  const int32_t* __restrict__ row_start;
  const int32_t* __restrict__ draft_tokens;
  const float* __restrict__ draft_probs;        // or null
  const float* __restrict__ accept_uniform;
  const float* __restrict__ draw_uniform;
  const float* __restrict__ temperature;        // or null: all 0
  int rows, vocab, requests, chunks;
};

struct RowPart {
  double sum;
  float max;
  int32_t place;        // -1: the chunk holds a number that is not finite
};

struct Masses {
  double residual, plain;
};

struct Decision {
  double inverse_sum;
  float max;
  int32_t row, accepted;
  int32_t token;        // chosen already (greedy, or -1), else -2
  int32_t draft;        // index of the draft that was not taken, -1: all were
};

// A request's rows and drafts.  Starts that are not what they should be (not ascending, or
// outside the rows) give a request fewer of them and wrong tokens, but no access outside.
struct Rows {
  int first, drafts, first_draft;
};

__device__ __forceinline__ Rows rows_of(const Batch& b, int request) {
  Rows r;
  r.first = min(max(b.row_start[request], 0), b.rows - 1);
  r.drafts = min(max(b.row_start[request + 1] - r.first - 1, 0), b.rows - 1 - r.first);
  // where request r's drafts begin: every request before it has one row more than drafts
  r.first_draft = min(max(r.first - request, 0), b.rows - b.requests);
  r.drafts = min(r.drafts, b.rows - b.requests - r.first_draft);
  return r;
}

__device__ __forceinline__ float temperature_of(const Batch& b, int request) {
  return b.temperature != nullptr ? b.temperature[request] : 0.f;
}

// The thread's elements of a chunk, four quads that lie on 16-byte borders of the row's
// memory: element(j, i) of quad j, values outside the row left at `outside`.
struct Quads {
  float value[kQuads][4];
  int first[kQuads];
};

__device__ __forceinline__ void load_quads(Quads& q, const float* __restrict__ row, int vocab, int chunk, int shift,
                                           float outside) {
  const bool aligned = ((reinterpret_cast<uintptr_t>(row) >> 2) & 3) == static_cast<uintptr_t>(shift);
#pragma unroll
  for (int j = 0; j < kQuads; ++j) {
    q.first[j] = chunk * kChunk + 4 * (threadIdx.x + j * kThreads) - shift;
    const int e = q.first[j];
    if (aligned && e >= 0 && e + 3 < vocab) {
      const float4 four = *reinterpret_cast<const float4*>(row + e);
      q.value[j][0] = four.x, q.value[j][1] = four.y, q.value[j][2] = four.z, q.value[j][3] = four.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) q.value[j][i] = e + i >= 0 && e + i < vocab ? row[e + i] : outside;
    }
  }
}

__device__ __forceinline__ int shift_of(const float* row) { return static_cast<int>((reinterpret_cast<uintptr_t>(row) >> 2) & 3); }

__device__ __forceinline__ double wave_sum_double(double v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, ms::kWave);
  return v;
}

__device__ __forceinline__ double block_sum_double(double v, double* scratch) {
  v = wave_sum_double(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total += scratch[w];
  return total;
}

// (1) grid (chunks, rows)
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(Batch b, RowPart* __restrict__ parts) {
  __shared__ float max_s[kWaves];
  __shared__ int place_s[kWaves];
  __shared__ double sum_s[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int chunk = blockIdx.x, row = blockIdx.y;
  const float* logits = b.logits + static_cast<int64_t>(row) * b.vocab;
  const float outside = -3.402823466e38f;
  Quads q;
  load_quads(q, logits, b.vocab, chunk, shift_of(logits), outside);
  float best = -INFINITY;
  int place = 0x7fffffff;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < kQuads; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = q.first[j] + i;
      const float v = q.value[j][i];
      if (!(fabsf(v) <= 3.402823466e38f)) bad = true;
      if (e >= 0 && e < b.vocab && (v > best || (v == best && e < place))) best = v, place = e;
    }
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) {
    const float other = __shfl_xor(best, offset, ms::kWave);
    const int other_place = __shfl_xor(place, offset, ms::kWave);
    if (other > best || (other == best && other_place < place)) best = other, place = other_place;
  }
  bad = __any(bad);
  if (lane == 0) {
    max_s[wave] = best;
    place_s[wave] = bad ? -1 : place;
  }
  __syncthreads();
  best = max_s[0], place = place_s[0];
  bad = place < 0;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    bad = bad || place_s[w] < 0;
    if (max_s[w] > best || (max_s[w] == best && place_s[w] < place)) best = max_s[w], place = place_s[w];
  }
  // the request of the row, for its temperature
  float temperature = 0.f;
  if (b.temperature != nullptr) {
    int at_or_before = 0;
    for (int r0 = 0; r0 < b.requests; r0 += ms::kWave) {
      const int r = r0 + lane;
      at_or_before += __popcll(__ballot(r < b.requests && b.row_start[r] <= row));
    }
    temperature = b.temperature[max(at_or_before - 1, 0)];
  }
  double sum = 0.0;
  if (temperature > 0.f && !bad) {
    const double factor = 1.0 / static_cast<double>(temperature);
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = q.first[j] + i;
        if (e >= 0 && e < b.vocab) sum += exp((static_cast<double>(q.value[j][i]) - static_cast<double>(best)) * factor);
      }
    sum = block_sum_double(sum, sum_s);
  }
  if (threadIdx.x == 0) {
    RowPart& part = parts[static_cast<int64_t>(row) * b.chunks + chunk];
    part.sum = sum;
    part.max = best;
    part.place = bad ? -1 : place;
  }
}

struct RowSums {
  double sum;
  float max;
  int place;      // -1: not finite
};

// A row's maximum, its place and its sum from the chunks'; by one wave, the same in all lanes.
__device__ __forceinline__ RowSums row_sums(const Batch& b, const RowPart* __restrict__ parts, int row, double factor) {
  const int lane = threadIdx.x & 63;
  RowSums r{0.0, -INFINITY, 0x7fffffff};
  bool bad = false;
  for (int c = lane; c < b.chunks; c += ms::kWave) {
    const RowPart part = parts[static_cast<int64_t>(row) * b.chunks + c];
    bad = bad || part.place < 0;
    if (part.max > r.max || (part.max == r.max && part.place < r.place)) r.max = part.max, r.place = part.place;
  }
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) {
    const float other = __shfl_xor(r.max, offset, ms::kWave);
    const int other_place = __shfl_xor(r.place, offset, ms::kWave);
    if (other > r.max || (other == r.max && other_place < r.place)) r.max = other, r.place = other_place;
  }
  if (__any(bad)) r.place = -1;
  if (factor > 0.0 && r.place >= 0) {
    double sum = 0.0;
    for (int c = lane; c < b.chunks; c += ms::kWave) {
      const RowPart part = parts[static_cast<int64_t>(row) * b.chunks + c];
      sum += part.sum * exp((static_cast<double>(part.max) - static_cast<double>(r.max)) * factor);
    }
    r.sum = wave_sum_double(sum);
  }
  return r;
}

// (2) grid (chunks, requests)
__global__ __launch_bounds__(kThreads) void verify_choose_kernel(Batch b, const RowPart* __restrict__ parts,
                                                                 Masses* __restrict__ masses,
                                                                 Decision* __restrict__ decisions) {
  __shared__ int end_s[kWaves];
  __shared__ double sum_s[kWaves];
  const int lane = threadIdx.x & 63, wave = ms::uniform(threadIdx.x >> 6);
  const int chunk = blockIdx.x, request = blockIdx.y;
  const Rows rows = rows_of(b, request);
  const float temperature = temperature_of(b, request);
  const bool greedy = !(temperature > 0.f);
  const double factor = greedy ? 0.0 : 1.0 / static_cast<double>(temperature);
  // each wave looks at drafts of its own; the first that is not taken ends them
  int end = rows.drafts;
  for (int i = wave; i < rows.drafts && i < end; i += kWaves) {
    const int row = rows.first + i;
    const int64_t draft = rows.first_draft + i;
    const RowSums sums = row_sums(b, parts, row, factor);
    const int token = b.draft_tokens[draft];
    bool taken = false;
    if (sums.place >= 0 && token >= 0 && token < b.vocab) {
      if (greedy) {
        taken = token == sums.place;
      } else {
        const double logit = b.logits[static_cast<int64_t>(row) * b.vocab + token];
        const double p = exp((logit - static_cast<double>(sums.max)) * factor) / sums.sum;
        const double q = b.draft_probs != nullptr ? b.draft_probs[draft * b.vocab + token] : 1.f;
        taken = static_cast<double>(b.accept_uniform[draft]) * q < p;
      }
    }
    if (!taken) end = i;
  }
  if (lane == 0) end_s[wave] = end;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) end = min(end, end_s[w]);
  const int row = rows.first + end;
  const RowSums sums = row_sums(b, parts, row, factor);
  const bool chosen = greedy || sums.place < 0;
  const int64_t draft = end < rows.drafts ? rows.first_draft + end : -1;
  if (chunk == 0 && threadIdx.x == 0) {
    Decision& d = decisions[request];
    d.inverse_sum = chosen ? 0.0 : 1.0 / sums.sum;
    d.max = sums.max;
    d.row = row;
    d.accepted = end;
    d.token = chosen ? sums.place : -2;
    d.draft = static_cast<int32_t>(draft);
  }
  if (chosen) return;
  const double inverse = 1.0 / sums.sum;
  const float* logits = b.logits + static_cast<int64_t>(row) * b.vocab;
  const int shift = shift_of(logits);
  Quads l, q;
  load_quads(l, logits, b.vocab, chunk, shift, 0.f);
  const bool subtract = draft >= 0 && b.draft_probs != nullptr;
  if (subtract) load_quads(q, b.draft_probs + draft * b.vocab, b.vocab, chunk, shift, 0.f);
  const int without = draft >= 0 && b.draft_probs == nullptr ? b.draft_tokens[draft] : -1;
  double residual = 0.0, plain = 0.0;
#pragma unroll
  for (int j = 0; j < kQuads; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = l.first[j] + i;
      if (e < 0 || e >= b.vocab) continue;
      const double p = exp((static_cast<double>(l.value[j][i]) - static_cast<double>(sums.max)) * factor) * inverse;
      plain += p;
      residual += subtract ? fmax(p - static_cast<double>(q.value[j][i]), 0.0) : (e == without ? 0.0 : p);
    }
  residual = block_sum_double(residual, sum_s);
  plain = block_sum_double(plain, sum_s);
  if (threadIdx.x == 0) masses[static_cast<int64_t>(request) * b.chunks + chunk] = Masses{residual, plain};
}

// (3) grid (requests)
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(Batch b, const Masses* __restrict__ masses,
                                                               const Decision* __restrict__ decisions,
                                                               int32_t* __restrict__ tokens,
                                                               int32_t* __restrict__ accepted) {
  __shared__ double wave_s[kWaves];
  __shared__ int chunk_s, token_s;
  __shared__ double before_s, target_s;
  __shared__ bool residual_s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int request = blockIdx.x;
  const Rows rows = rows_of(b, request);
  const Decision d = decisions[request];
  int token = d.token;
  if (token == -2) {
    if (threadIdx.x == 0) {
      const Masses* m = masses + static_cast<int64_t>(request) * b.chunks;
      double residual = 0.0, plain = 0.0;
      for (int c = 0; c < b.chunks; ++c) residual += m[c].residual, plain += m[c].plain;
      const bool use = residual > 0.0;
      const double target = static_cast<double>(b.draw_uniform[request]) * (use ? residual : plain);
      double before = 0.0, running = 0.0;
      int chunk = 0;
      for (int c = 0; c < b.chunks; ++c) {
        const double mass = use ? m[c].residual : m[c].plain;
        if (mass > 0.0) {
          chunk = c;
          before = running;
          running += mass;
          if (running > target) break;
        }
      }
      chunk_s = chunk, before_s = before, target_s = target, residual_s = use;
      token_s = -1;
    }
    __syncthreads();
    // the chunk's elements in their order, kQuads * 4 neighbours a thread
    const float* logits = b.logits + static_cast<int64_t>(d.row) * b.vocab;
    const double factor = 1.0 / static_cast<double>(temperature_of(b, request));
    const bool subtract = residual_s && d.draft >= 0 && b.draft_probs != nullptr;
    const int without = residual_s && d.draft >= 0 && b.draft_probs == nullptr ? b.draft_tokens[d.draft] : -1;
    const float* probs = subtract ? b.draft_probs + static_cast<int64_t>(d.draft) * b.vocab : nullptr;
    const int first = chunk_s * kChunk - shift_of(logits) + threadIdx.x * kQuads * 4;
    double mass[kQuads * 4], sum = 0.0;
#pragma unroll
    for (int i = 0; i < kQuads * 4; ++i) {
      const int e = first + i;
      mass[i] = 0.0;
      if (e >= 0 && e < b.vocab && e != without) {
        const double p = exp((static_cast<double>(logits[e]) - static_cast<double>(d.max)) * factor) * d.inverse_sum;
        mass[i] = subtract ? fmax(p - static_cast<double>(probs[e]), 0.0) : p;
      }
      sum += mass[i];
    }
    double upto = sum;
#pragma unroll
    for (int offset = 1; offset < ms::kWave; offset <<= 1) {
      const double other = __shfl_up(upto, offset, ms::kWave);
      if (lane >= offset) upto += other;
    }
    if (lane == ms::kWave - 1) wave_s[wave] = upto;
    __syncthreads();
    double running = before_s + upto - sum;
    for (int w = 0; w < wave; ++w) running += wave_s[w];
    // the first element at which the running sum passes the target; where rounding leaves
    // none (the target lies at the chunk's very end), the last one with a mass
    int passed = 0x7fffffff, last = -1;
#pragma unroll
    for (int i = 0; i < kQuads * 4; ++i) {
      running += mass[i];
      if (mass[i] > 0.0) {
        last = first + i;
        if (running > target_s && passed == 0x7fffffff) passed = first + i;
      }
    }
    __shared__ int passed_s[kWaves], last_s[kWaves];
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1) {
      passed = min(passed, __shfl_xor(passed, offset, ms::kWave));
      last = max(last, __shfl_xor(last, offset, ms::kWave));
    }
    if (lane == 0) passed_s[wave] = passed, last_s[wave] = last;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) passed = min(passed, passed_s[w]), last = max(last, last_s[w]);
    token = passed != 0x7fffffff ? passed : last;
  }
  for (int i = threadIdx.x; i <= rows.drafts; i += kThreads) {
    const int row = rows.first + i;
    tokens[row] = i < d.accepted ? b.draft_tokens[rows.first_draft + i] : i == d.accepted ? token : -1;
  }
  if (threadIdx.x == 0) accepted[request] = d.accepted;
}

int chunks_of(int vocab) { return (vocab + 3 + kChunk - 1) / kChunk; }      // a row may begin at any float of a quad

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

// Bytes of workspace that ms_verify_drafts takes for this many rows, requests and tokens of
// the vocabulary.
extern "C" size_t ms_verify_drafts_workspace_bytes(int rows, int requests, int vocab) {
  if (rows <= 0 || requests <= 0 || vocab <= 0) return 0;
  const size_t chunks = chunks_of(vocab);
  return aligned(rows * chunks * sizeof(RowPart)) + aligned(requests * chunks * sizeof(Masses)) +
         aligned(requests * sizeof(Decision));
}

// logits: float [rows, vocab]; row_start: int32 [requests + 1], request r's rows are
// row_start[r] .. row_start[r + 1] - 1, one more than it has drafts; draft_tokens: int32 [rows -
// requests]; draft_probs: float [rows - requests, vocab] or null; accept_uniform: float [rows -
// requests]; draw_uniform: float [requests]; temperature: float [requests] or null (all 0, and
// the uniform numbers may be null too); tokens: int32 [rows]; accepted: int32 [requests].
extern "C" int ms_verify_drafts(const void* logits, const void* row_start, const void* draft_tokens,
                                const void* draft_probs, const void* accept_uniform, const void* draw_uniform,
                                const void* temperature, void* tokens, void* accepted, void* workspace,
                                size_t workspace_bytes, int rows, int requests, int vocab, hipStream_t stream) {
  MS_REQUIRE(rows > 0 && rows <= 65535 && requests > 0 && requests <= rows && vocab > 0 && vocab < (1 << 30),
             "verify_drafts: %d rows (up to 65535) of %d tokens for %d requests", rows, vocab, requests);
  MS_REQUIRE(temperature == nullptr || (draw_uniform != nullptr && (accept_uniform != nullptr || rows == requests)),
             "verify_drafts: sampling needs uniform numbers");
  MS_REQUIRE(draft_tokens != nullptr || rows == requests, "verify_drafts: no drafted tokens");
  MS_REQUIRE(workspace_bytes >= ms_verify_drafts_workspace_bytes(rows, requests, vocab), "verify_drafts: workspace too small");
  Batch b;
  b.logits = static_cast<const float*>(logits);
  b.row_start = static_cast<const int32_t*>(row_start);
  b.draft_tokens = static_cast<const int32_t*>(draft_tokens);
  b.draft_probs = static_cast<const float*>(draft_probs);
  b.accept_uniform = static_cast<const float*>(accept_uniform);
  b.draw_uniform = static_cast<const float*>(draw_uniform);
  b.temperature = static_cast<const float*>(temperature);
  b.rows = rows;
  b.vocab = vocab;
  b.requests = requests;
  b.chunks = chunks_of(vocab);
  char* at = static_cast<char*>(workspace);
  RowPart* parts = reinterpret_cast<RowPart*>(at);
  at += aligned(static_cast<size_t>(rows) * b.chunks * sizeof(RowPart));
  Masses* masses = reinterpret_cast<Masses*>(at);
  at += aligned(static_cast<size_t>(requests) * b.chunks * sizeof(Masses));
  Decision* decisions = reinterpret_cast<Decision*>(at);
  hipLaunchKernelGGL(verify_rows_kernel, dim3(b.chunks, rows), dim3(kThreads), 0, stream, b, parts);
  MS_CHECK_LAUNCH("verify_drafts (rows)");
  hipLaunchKernelGGL(verify_choose_kernel, dim3(b.chunks, requests), dim3(kThreads), 0, stream, b,
                     static_cast<const RowPart*>(parts), masses, decisions);
  MS_CHECK_LAUNCH("verify_drafts (choose)");
  hipLaunchKernelGGL(verify_draw_kernel, dim3(requests), dim3(kThreads), 0, stream, b, static_cast<const Masses*>(masses),
                     static_cast<const Decision*>(decisions), static_cast<int32_t*>(tokens),
                     static_cast<int32_t*>(accepted));
  MS_CHECK_LAUNCH("verify_drafts (draw)");
  return 0;
}
