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
//
// (1) reads every logit once, and with 14 64-bit instructions an element those and the
// read take about as long: 576 rows of 151,936, 350 MB, 65 to 76 us = 4.6 to 5.4 TB/s on
// MI355X (a large copy: 4.9); with 64 requests of 8 drafts (2), (2a) and (3) take 33 us more.  One request of 4
// drafts takes 6 + 6 + 6 us, each the chain of its loads and sums over a workgroup.  (With the
// draw in (2), by the request's last workgroup, each has to make its masses visible to the
// other dies' caches: 110 us instead of 28 for (2) and (3) of 64 requests, 13 as before for one.)
#include "common.hpp"

namespace {

// Elements of a row that a wave takes in (1), 32 to a lane (the waves of a workgroup share
// nothing, so none waits for another), and that a workgroup takes in (2) and (3), where the row
// is one of the request's and many units share it.
constexpr int kRowChunk = 2048, kChunk = 4096;
constexpr int kRowThreads = 256, kChooseThreads = 512, kDrawThreads = kChunk / 4;

// 2^f on -1/2 .. 1/2, lowest power first: the polynomials of degree seven and nine whose largest
// relative error there is least (found by exchange of its extrema: 4.0e-11 and 1.3e-14).  They
// travel with a kernel's arguments, so that the coefficients lie in scalar registers: as literals
// the compiler copies each into vector registers before every use (39 instructions an element
// instead of 25).  The shorter one serves Z, the sum over all tokens of all rows (73 us for 576
// rows, with the longer one 89): it moves a border by 4e-11 of itself at most, past one uniform
// number in some 10^10.
constexpr int kDegree = 9, kSumDegree = 7;
constexpr double kPowerOfTwo[kDegree + 1] = {
    1.00000000000001266e+00,
    6.93147180559871012e-01,
    2.40226506956496527e-01,
    5.55041086686855825e-02,
    9.61812919206720199e-03,
    1.33335576176098788e-03,
    1.54034349480814238e-04,
    1.52529848355783673e-05,
    1.32594056112041923e-06,
    1.01503372609764174e-07,
};
constexpr double kSumPowerOfTwo[kSumDegree + 1] = {
    9.99999999961681983e-01,
    6.93147180728445564e-01,
    2.40226511981572074e-01,
    5.55041035345320847e-02,
    9.61802725371136973e-03,
    1.33339225590775260e-03,
    1.54692911308010617e-04,
    1.52019226419755618e-05,
};

struct Batch {
  double power[kDegree + 1], sum_power[kSumDegree + 1];
  const float* __restrict__ logits;
  const int32_t* __restrict__ row_start;
  const int32_t* __restrict__ draft_tokens;
  const float* __restrict__ draft_probs;        // or null
  const float* __restrict__ accept_uniform;
  const float* __restrict__ draw_uniform;
  const float* __restrict__ temperature;        // or null: all 0
  int rows, vocab, requests, row_chunks, chunks;
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

// e^{(l - max) / T} = 2^{d rate}, d = l - max, rate = log2(e) / T
__device__ __forceinline__ double rate_of(float temperature) { return 1.4426950408889634074 / static_cast<double>(temperature); }

// 2^{d rate} in 64 bits for d rate from -1001 to 0: 2^k 2^f with k the nearest whole number.  (1) is
// bound by these instructions, so that k is had by adding 3 * 2^51, which leaves it in the sum's low
// bits, and 2^k by adding k to the exponent's bits (conversions and scalings run at a quarter of an
// addition's rate).  The product is made inside the two multiply-adds and never rounded by itself.
// d has to be the logits' difference: with l and max multiplied each for itself, the rounding of
// max * rate, up to |max| rate 2^-53, is left over at the maximum, and at T = 10^-15 or logits
// of 10^16 that is more than the mass itself.
template <int DEGREE>
__device__ __forceinline__ double pow2_scaled(const double (&power)[DEGREE + 1], double d, double rate) {
  const double shifted = fma(d, rate, 6755399441055744.0);
  const double f = fma(d, rate, -(shifted - 6755399441055744.0));
  double r = power[DEGREE];
#pragma unroll
  for (int n = DEGREE - 1; n >= 0; --n) r = fma(r, f, power[n]);
  return __hiloint2double(__double2hiint(r) + (__double2loint(shifted) << 20), __double2loint(r));
}

// The least d of pow2_scaled: -1001 / rate.
__device__ __forceinline__ double floor_of(float temperature) { return -1001.0 * 0.69314718055994530942 * static_cast<double>(temperature); }

__device__ __forceinline__ double mass_of(const Batch& b, float logit, float max, double rate) {
  const double d = static_cast<double>(logit) - static_cast<double>(max);
  const double mass = pow2_scaled<kDegree>(b.power, d, rate);
  return d * rate < -1000.0 ? 0.0 : mass;
}

__device__ __forceinline__ bool not_finite(float v) { return __builtin_isfpclass(v, 0x3 | 0x4 | 0x200); }      // NaN, -inf, +inf

__device__ __forceinline__ int shift_of(const float* row) { return static_cast<int>((reinterpret_cast<uintptr_t>(row) >> 2) & 3); }

typedef float Four __attribute__((ext_vector_type(4)));

// A thread's elements of a chunk: quads that lie on 16-byte borders of the row's memory;
// quad j is value[j], its first element first[j].
template <int QUADS>
struct Quads {
  float value[QUADS][4];
  int first[QUADS];
  bool whole;       // no element of the chunk lies outside the row (the same in all threads)
};

// ``shift``: floats between the 16-byte border before the row and the row.  What lies outside
// the row is left at `outside`.
template <int QUADS, int THREADS>
__device__ __forceinline__ void load_quads(Quads<QUADS>& q, int thread, const float* __restrict__ row, int vocab, int begin,
                                           int shift, float outside) {
  // no branch around the loads of a chunk that lies inside the row: all are under way at once
  q.whole = shift_of(row) == shift && begin >= shift && begin - shift + 4 * QUADS * THREADS <= vocab;
#pragma unroll
  for (int j = 0; j < QUADS; ++j) q.first[j] = begin + 4 * (thread + j * THREADS) - shift;
  if (q.whole) {
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
      const Four four = *reinterpret_cast<const Four*>(row + q.first[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) q.value[j][i] = four[i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < QUADS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = q.first[j] + i;
        const float v = row[min(max(e, 0), vocab - 1)];
        q.value[j][i] = e >= 0 && e < vocab ? v : outside;
      }
  }
}

template <int LANES>
__device__ __forceinline__ double lanes_sum(double v) {
#pragma unroll
  for (int offset = LANES / 2; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, LANES);
  return v;
}

// (1) grid (chunks of a row, four to a workgroup; rows)
__global__ __launch_bounds__(kRowThreads) void verify_rows_kernel(Batch b, RowPart* __restrict__ parts) {
  constexpr int kQuads = kRowChunk / ms::kWave / 4;
  const int lane = threadIdx.x & 63;
  const int chunk = blockIdx.x * (kRowThreads / ms::kWave) + ms::uniform(threadIdx.x >> 6), row = blockIdx.y;
  if (chunk >= b.row_chunks) return;
  const float* logits = b.logits + static_cast<int64_t>(row) * b.vocab;
  constexpr float kOutside = -3.402823466e38f;          // finite, and no more than any finite number of the row
  Quads<kQuads> q;
  load_quads<kQuads, ms::kWave>(q, lane, logits, b.vocab, chunk * kRowChunk, shift_of(logits), kOutside);
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
  float best = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < kQuads; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bad |= not_finite(q.value[j][i]);
      best = fmaxf(best, q.value[j][i]);
    }
  best = ms::wave_max(best);
  bad = __any(bad);
  double sum = 0.0;
  int place = 0x7fffffff;
  if (temperature > 0.f) {
    const double rate = rate_of(temperature), least = floor_of(temperature), top = best;
    // what lies below the least is taken as 2^-1001: a sum that holds a mass of 1 does not see it
    const auto mass = [&](float logit) {
      return pow2_scaled<kSumDegree>(b.sum_power, fmax(static_cast<double>(logit) - top, least), rate);
    };
    if (q.whole) {
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += mass(q.value[j][i]);
    } else {
#pragma unroll
      for (int j = 0; j < kQuads; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = q.first[j] + i;
          const double here = mass(q.value[j][i]);
          sum += e >= 0 && e < b.vocab ? here : 0.0;
        }
    }
    sum = lanes_sum<ms::kWave>(sum);
  } else {
    // the lowest index of the maximum
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = q.first[j] + i;
        if (q.value[j][i] == best && e >= 0 && e < b.vocab) place = min(place, e);
      }
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1) place = min(place, __shfl_xor(place, offset, ms::kWave));
  }
  if (lane == 0) parts[static_cast<int64_t>(row) * b.row_chunks + chunk] = RowPart{sum, best, bad ? -1 : place};
}

struct RowSums {
  double sum;
  float max;
  int place;      // -1: not finite
};

// A row's maximum, its place and its sum from the chunks'; by 32 lanes, the same in all of them.
__device__ __forceinline__ RowSums row_sums(const Batch& b, const RowPart* __restrict__ parts, int row, double rate) {
  const int lane = threadIdx.x & 31;
  RowSums r{0.0, -INFINITY, 0x7fffffff};
  constexpr int kHeld = 3;        // chunks a lane keeps: 196,608 tokens of the vocabulary
  RowPart held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    const int c = lane + 32 * u;
    held[u] = c < b.row_chunks ? parts[static_cast<int64_t>(row) * b.row_chunks + c] : RowPart{0.0, -INFINITY, 0x7fffffff};
  }
  bool bad = false;
  const auto look = [&](const RowPart& part) {
    bad = bad || part.place < 0;
    if (part.max > r.max || (part.max == r.max && part.place < r.place)) r.max = part.max, r.place = part.place;
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u) look(held[u]);
  for (int c = lane + 32 * kHeld; c < b.row_chunks; c += 32) look(parts[static_cast<int64_t>(row) * b.row_chunks + c]);
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) {
    const float other = __shfl_xor(r.max, offset, 32);
    const int other_place = __shfl_xor(r.place, offset, 32);
    bad |= __shfl_xor(static_cast<int>(bad), offset, 32) != 0;
    if (other > r.max || (other == r.max && other_place < r.place)) r.max = other, r.place = other_place;
  }
  if (bad) r.place = -1;
  double sum = 0.0;
  const auto add = [&](const RowPart& part) {
    if (part.sum > 0.0) sum += part.sum * mass_of(b, part.max, r.max, rate);
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u) add(held[u]);
  for (int c = lane + 32 * kHeld; c < b.row_chunks; c += 32) add(parts[static_cast<int64_t>(row) * b.row_chunks + c]);
  r.sum = lanes_sum<32>(sum);
  return r;
}

// How a request ends; by a whole workgroup, the same in all its threads.
__device__ __forceinline__ Decision decide(const Batch& b, const RowPart* __restrict__ parts, int request, const Rows& rows,
                                           float temperature) {
  constexpr int kWaves = kChooseThreads / ms::kWave;
  constexpr int kAtOnce = kChooseThreads / 32;       // rows that are looked at together, 32 lanes each
  __shared__ RowSums sums_s[kAtOnce];
  __shared__ uint64_t ends_s[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = threadIdx.x >> 5;
  const bool greedy = !(temperature > 0.f);
  const double rate = greedy ? 0.0 : rate_of(temperature);
  // the first row whose draft is not taken; the row behind the last draft has none
  int end = 0;
  for (int first = 0;; first += kAtOnce) {
    const int i = first + half;
    bool ends = i == rows.drafts;
    if (i <= rows.drafts) {
      const int row = rows.first + i;
      const int64_t draft = rows.first_draft + i;
      double mass = 0.0, q = 1.0, u = 0.0;
      int token = -1;
      if (!ends) {
        token = b.draft_tokens[draft];
        if (!greedy && token >= 0 && token < b.vocab) {
          u = b.accept_uniform[draft];
          mass = b.logits[static_cast<int64_t>(row) * b.vocab + token];
          if (b.draft_probs != nullptr) q = b.draft_probs[draft * b.vocab + token];
        }
      }
      const RowSums sums = row_sums(b, parts, row, rate);
      if (!ends) {
        if (sums.place < 0 || token < 0 || token >= b.vocab) {
          ends = true;
        } else if (greedy) {
          ends = token != sums.place;
        } else {
          ends = !(u * q < mass_of(b, static_cast<float>(mass), sums.max, rate) / sums.sum);
        }
      }
      if ((threadIdx.x & 31) == 0) sums_s[half] = sums;
    }
    const uint64_t found = __ballot(ends);      // lane 0: the wave's first row, lane 32: its second
    if (lane == 0) ends_s[wave] = found;
    __syncthreads();
    int at = -1;
#pragma unroll
    for (int w = kWaves - 1; w >= 0; --w) {
      if (ends_s[w] >> 32 & 1) at = 2 * w + 1;
      if (ends_s[w] & 1) at = 2 * w;
    }
    if (at >= 0) {
      end = first + at;
      break;
    }
    __syncthreads();
  }
  const RowSums sums = sums_s[end % kAtOnce];
  const bool chosen = greedy || sums.place < 0;
  return Decision{1.0 / sums.sum, sums.max, rows.first + end, end, chosen ? sums.place : -2,
                  end < rows.drafts ? rows.first_draft + end : -1};
}

// What the request gets; by one wave.
__device__ __forceinline__ void give(const Batch& b, const Rows& rows, const Decision& d, int token, int request,
                                     int32_t* __restrict__ tokens, int32_t* __restrict__ accepted) {
  const int lane = threadIdx.x & 63;
  for (int i = lane; i <= rows.drafts; i += ms::kWave)
    tokens[rows.first + i] = i < d.accepted ? b.draft_tokens[rows.first_draft + i] : i == d.accepted ? token : -1;
  if (lane == 0) accepted[request] = d.accepted;
}

// (2a) grid (requests), for many requests: the decisions by themselves.  A workgroup of (2)
// takes some 5 us to make its request's, in which its unit draws nothing from memory; with
// few requests that is shorter than another kernel.
__global__ __launch_bounds__(kChooseThreads) void verify_decide_kernel(Batch b, const RowPart* __restrict__ parts,
                                                                       Decision* __restrict__ decisions) {
  const int request = blockIdx.x;
  const Decision d = decide(b, parts, request, rows_of(b, request), temperature_of(b, request));
  if (threadIdx.x == 0) decisions[request] = d;
}

// (2) grid (chunks, requests)
template <bool DECIDED>
__global__ __launch_bounds__(kChooseThreads) void verify_choose_kernel(Batch b, const RowPart* __restrict__ parts,
                                                                       Masses* __restrict__ masses,
                                                                       Decision* __restrict__ decisions) {
  constexpr int kWaves = kChooseThreads / ms::kWave, kQuads = kChunk / kChooseThreads / 4;
  __shared__ double residual_s[kWaves], plain_s[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int chunk = blockIdx.x, request = blockIdx.y;
  const float temperature = temperature_of(b, request);
  Decision d;
  if constexpr (DECIDED) {
    d = decisions[request];
  } else {
    d = decide(b, parts, request, rows_of(b, request), temperature);
    if (chunk == 0 && threadIdx.x == 0) decisions[request] = d;
  }
  if (d.token != -2) return;
  const double rate = rate_of(temperature), inverse = d.inverse_sum;
  const int64_t draft = d.draft;
  const float* logits = b.logits + static_cast<int64_t>(d.row) * b.vocab;
  const int shift = shift_of(logits);
  Quads<kQuads> l, q;
  load_quads<kQuads, kChooseThreads>(l, threadIdx.x, logits, b.vocab, chunk * kChunk, shift, 0.f);
  const bool subtract = draft >= 0 && b.draft_probs != nullptr;
  if (subtract) load_quads<kQuads, kChooseThreads>(q, threadIdx.x, b.draft_probs + draft * b.vocab, b.vocab, chunk * kChunk, shift, 0.f);
  const int without = draft >= 0 && b.draft_probs == nullptr ? b.draft_tokens[draft] : -1;
  double residual = 0.0, plain = 0.0;
#pragma unroll
  for (int j = 0; j < kQuads; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = l.first[j] + i;
      if (e < 0 || e >= b.vocab) continue;
      const double p = mass_of(b, l.value[j][i], d.max, rate) * inverse;
      plain += p;
      residual += subtract ? fmax(p - static_cast<double>(q.value[j][i]), 0.0) : (e == without ? 0.0 : p);
    }
  residual = lanes_sum<ms::kWave>(residual);
  plain = lanes_sum<ms::kWave>(plain);
  if (lane == 0) residual_s[wave] = residual, plain_s[wave] = plain;
  __syncthreads();
  if (threadIdx.x == 0) {
    Masses m{0.0, 0.0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m.residual += residual_s[w], m.plain += plain_s[w];
    masses[static_cast<int64_t>(request) * b.chunks + chunk] = m;
  }
}

// Running sums over the lanes of a wave, this lane's included.
__device__ __forceinline__ double wave_running_sum(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int offset = 1; offset < ms::kWave; offset <<= 1) {
    const double other = __shfl_up(v, offset, ms::kWave);
    if (lane >= offset) v += other;
  }
  return v;
}

// (3) grid (requests)
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(Batch b, const Masses* __restrict__ masses,
                                                                   const Decision* __restrict__ decisions,
                                                                   int32_t* __restrict__ tokens,
                                                                   int32_t* __restrict__ accepted) {
  constexpr int kWaves = kDrawThreads / ms::kWave;
  __shared__ double wave_s[kWaves];
  __shared__ int passed_s[kWaves], last_s[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int request = blockIdx.x;
  const Rows rows = rows_of(b, request);
  const Decision d = decisions[request];
  int token = d.token;
  if (token == -2) {
    // the chunk in which the running sum passes the target; by every wave for itself
    const Masses* m = masses + static_cast<int64_t>(request) * b.chunks;
    const double uniform = b.draw_uniform[request];
    const Masses mine = lane < b.chunks ? m[lane] : Masses{0.0, 0.0};
    double residual = mine.residual, plain = mine.plain;
    for (int c = lane + ms::kWave; c < b.chunks; c += ms::kWave) residual += m[c].residual, plain += m[c].plain;
    residual = lanes_sum<ms::kWave>(residual);
    plain = lanes_sum<ms::kWave>(plain);
    const bool use = residual > 0.0;
    const double target = uniform * (use ? residual : plain);
    double carried = 0.0, before = 0.0;
    int chunk = 0;
    for (int c0 = 0; c0 < b.chunks; c0 += ms::kWave) {
      const int c = c0 + lane;
      const Masses here = c0 == 0 ? mine : c < b.chunks ? m[c] : Masses{0.0, 0.0};
      const double mass = use ? here.residual : here.plain;
      const double upto = wave_running_sum(mass);
      const uint64_t some = __ballot(mass > 0.0), past = __ballot(mass > 0.0 && carried + upto > target);
      if (some != 0) {
        // where rounding leaves no chunk that passes, the last one with a mass
        const int at = past != 0 ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
        chunk = c0 + at;
        before = carried + __shfl(upto - mass, at, ms::kWave);
        if (past != 0) break;
      }
      carried += __shfl(upto, ms::kWave - 1, ms::kWave);
    }
    // the chunk's elements in their order, four neighbours a thread
    const float* logits = b.logits + static_cast<int64_t>(d.row) * b.vocab;
    const int shift = shift_of(logits);
    const double rate = rate_of(temperature_of(b, request));
    const bool subtract = use && d.draft >= 0 && b.draft_probs != nullptr;
    const int without = use && d.draft >= 0 && b.draft_probs == nullptr ? b.draft_tokens[d.draft] : -1;
    Quads<1> l, q;
    load_quads<1, kDrawThreads>(l, threadIdx.x, logits, b.vocab, chunk * kChunk, shift, 0.f);
    if (subtract) load_quads<1, kDrawThreads>(q, threadIdx.x, b.draft_probs + static_cast<int64_t>(d.draft) * b.vocab, b.vocab, chunk * kChunk, shift, 0.f);
    double mass[4], sum = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = l.first[0] + i;
      mass[i] = 0.0;
      if (e >= 0 && e < b.vocab && e != without) {
        const double p = mass_of(b, l.value[0][i], d.max, rate) * d.inverse_sum;
        mass[i] = subtract ? fmax(p - static_cast<double>(q.value[0][i]), 0.0) : p;
      }
      sum += mass[i];
    }
    const double upto = wave_running_sum(sum);
    if (lane == ms::kWave - 1) wave_s[wave] = upto;
    __syncthreads();
    double running = before + upto - sum;
    for (int w = 0; w < wave; ++w) running += wave_s[w];
    // the first element at which the running sum passes the target; where rounding leaves
    // none (the target lies at the chunk's very end), the last one with a mass
    int passed = 0x7fffffff, last = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      running += mass[i];
      if (mass[i] > 0.0) {
        last = l.first[0] + i;
        if (running > target && passed == 0x7fffffff) passed = l.first[0] + i;
      }
    }
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1) {
      passed = min(passed, __shfl_xor(passed, offset, ms::kWave));
      last = max(last, __shfl_xor(last, offset, ms::kWave));
    }
    if (lane == 0) passed_s[wave] = passed, last_s[wave] = last;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w) passed = min(passed, passed_s[w]), last = max(last, last_s[w]);
      token = passed != 0x7fffffff ? passed : last;
    }
  }
  if (wave == 0) give(b, rows, d, token, request, tokens, accepted);
}

// (2) and (3) where no request has a temperature: the best token of the row where the drafts
// end is known with the decision, and nothing is drawn (one request of 4 drafts, recorded, 8.2 us,
// and 11.0 by the way of the draws; an eager call 12.5 and 15.6).
__global__ __launch_bounds__(kChooseThreads) void verify_greedy_kernel(Batch b, const RowPart* __restrict__ parts,
                                                                       int32_t* __restrict__ tokens,
                                                                       int32_t* __restrict__ accepted) {
  const Rows rows = rows_of(b, blockIdx.x);
  const Decision d = decide(b, parts, blockIdx.x, rows, 0.f);
  if (threadIdx.x < ms::kWave) give(b, rows, d, d.token, blockIdx.x, tokens, accepted);
}

int chunks_of(int vocab, int chunk) { return (vocab + 3 + chunk - 1) / chunk; }      // a row may begin at any float of a quad

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

// Bytes of workspace that ms_verify_drafts takes for this many rows, requests and tokens of
// the vocabulary.
extern "C" size_t ms_verify_drafts_workspace_bytes(int rows, int requests, int vocab) {
  if (rows <= 0 || requests <= 0 || vocab <= 0) return 0;
  return aligned(sizeof(RowPart) * rows * chunks_of(vocab, kRowChunk)) +
         aligned(sizeof(Masses) * requests * chunks_of(vocab, kChunk)) + aligned(sizeof(Decision) * requests);
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
  for (int n = 0; n <= kDegree; ++n) b.power[n] = kPowerOfTwo[n];
  for (int n = 0; n <= kSumDegree; ++n) b.sum_power[n] = kSumPowerOfTwo[n];
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
  b.row_chunks = chunks_of(vocab, kRowChunk);
  b.chunks = chunks_of(vocab, kChunk);
  char* at = static_cast<char*>(workspace);
  RowPart* parts = reinterpret_cast<RowPart*>(at);
  at += aligned(sizeof(RowPart) * rows * b.row_chunks);
  Masses* masses = reinterpret_cast<Masses*>(at);
  at += aligned(sizeof(Masses) * requests * b.chunks);
  Decision* decisions = reinterpret_cast<Decision*>(at);
  hipLaunchKernelGGL(verify_rows_kernel, dim3((b.row_chunks + kRowThreads / ms::kWave - 1) / (kRowThreads / ms::kWave), rows),
                     dim3(kRowThreads), 0, stream, b, parts);
  MS_CHECK_LAUNCH("verify_drafts (rows)");
  if (temperature == nullptr) {
    hipLaunchKernelGGL(verify_greedy_kernel, dim3(requests), dim3(kChooseThreads), 0, stream, b,
                       static_cast<const RowPart*>(parts), static_cast<int32_t*>(tokens), static_cast<int32_t*>(accepted));
    MS_CHECK_LAUNCH("verify_drafts (greedy)");
    return 0;
  }
  const dim3 grid(b.chunks, requests);
  // decisions apart where the workgroups of (2) run in several turns (vocabulary 151,936, all
  // kernels: 64 requests of 8 drafts 108 us apart and 115 together, 32 of 4 the same, 16 of 4
  // 35.5 and 33.0, one 19.9 and 18.2)
  if (static_cast<int64_t>(b.chunks) * requests > 4 * ms_compute_units()) {
    hipLaunchKernelGGL(verify_decide_kernel, dim3(requests), dim3(kChooseThreads), 0, stream, b,
                       static_cast<const RowPart*>(parts), decisions);
    MS_CHECK_LAUNCH("verify_drafts (decide)");
    hipLaunchKernelGGL((verify_choose_kernel<true>), grid, dim3(kChooseThreads), 0, stream, b,
                       static_cast<const RowPart*>(parts), masses, decisions);
  } else {
    hipLaunchKernelGGL((verify_choose_kernel<false>), grid, dim3(kChooseThreads), 0, stream, b,
                       static_cast<const RowPart*>(parts), masses, decisions);
  }
  MS_CHECK_LAUNCH("verify_drafts (choose)");
  hipLaunchKernelGGL(verify_draw_kernel, dim3(requests), dim3(kDrawThreads), 0, stream, b, static_cast<const Masses*>(masses),
                     static_cast<const Decision*>(decisions), static_cast<int32_t*>(tokens),
                     static_cast<int32_t*>(accepted));
  MS_CHECK_LAUNCH("verify_drafts (draw)");
  return 0;
}
