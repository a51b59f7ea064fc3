// Copies of whole cache pages inside their pools, in every call (layer) at once: pool[c,
// destination[i]] = pool[c, source[i]] for all c and i.  Sources and destinations are
// disjoint and the destinations distinct (checked below), so the copies may run in any
// order; one source may have several destinations.
//
// The page numbers travel with the launch itself, as its arguments: a table in device
// memory would cost a copy from the host before the kernel could start, which for a fork's
// one page takes longer than the copy of the page.
//
// Bound by memory: each thread has four 16-byte loads under way and then stores them, so that
// the workgroups of a unit, whose loads and stores alternate, keep both directions busy.
// Measured on MI355X (pages of 16 keys, 8 kv heads of 128, bf16): 1,000 pages in 28 layers,
// 3.7 GB read and written, 700 us = 5.2 TB/s (a large copy in one piece: 4.9); 48 pages in 36
// layers 35 us; one page in 28 layers 3 us.
#include <cstdlib>

#include "common.hpp"

namespace {

constexpr int kPools = 4;        // of one launch (keys and values, or a mixer's own planes)
constexpr int kThreads = 256;
constexpr int kUnroll = 4;       // accesses a thread has in flight

typedef uint32_t Quad __attribute__((ext_vector_type(4)));

struct Pool {
  char* base;
  int64_t page_bytes, call_bytes;
  int64_t calls;
};

// The launch's arguments; most launches of a server carry few pages, so there is a small form
// (an eager call with one page takes the host 8.7 us, and 9.2 with the large form).
template <int PAIRS>
struct Plan {
  Pool pools[kPools];
  int32_t pairs[PAIRS][2];       // source, destination
};

constexpr int kFewPairs = 32, kMostPairs = 480;      // 384 and 3,968 bytes of arguments

// One workgroup copies kThreads * kUnroll accesses of one page of one call.
template <typename Word, int PAIRS>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(Plan<PAIRS> plan, int chunks) {
  const int pair = blockIdx.x / chunks, chunk = blockIdx.x - pair * chunks;
  const Pool pool = plan.pools[blockIdx.z];
  const int source = plan.pairs[pair][0], destination = plan.pairs[pair][1];
  if (blockIdx.y >= pool.calls) return;
  const int64_t words = pool.page_bytes / static_cast<int64_t>(sizeof(Word));
  char* in_call = pool.base + blockIdx.y * pool.call_bytes;
  const Word* from = reinterpret_cast<const Word*>(in_call + source * pool.page_bytes);
  Word* to = reinterpret_cast<Word*>(in_call + destination * pool.page_bytes);
  const int64_t first = static_cast<int64_t>(chunk) * kThreads * kUnroll + threadIdx.x;
  if (first - threadIdx.x + kThreads * kUnroll <= words) {
    Word kept[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) kept[u] = from[first + u * kThreads];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) to[first + u * kThreads] = kept[u];
  } else {
    for (int64_t at = first; at < words; at += kThreads) to[at] = from[at];       // the page's last workgroup
  }
}

template <int PAIRS>
void launch(const Pool* pools, int num_pools, const int32_t* source, const int32_t* destination, int count, int word,
            int chunks, int calls, hipStream_t stream) {
  Plan<PAIRS> plan = {};
  for (int p = 0; p < num_pools; ++p) plan.pools[p] = pools[p];
  for (int i = 0; i < count; ++i) plan.pairs[i][0] = source[i], plan.pairs[i][1] = destination[i];
  const dim3 grid(static_cast<unsigned>(chunks) * count, calls, num_pools);
  if (word == 16)
    hipLaunchKernelGGL((copy_pages_kernel<Quad, PAIRS>), grid, dim3(kThreads), 0, stream, plan, chunks);
  else if (word == 4)
    hipLaunchKernelGGL((copy_pages_kernel<uint32_t, PAIRS>), grid, dim3(kThreads), 0, stream, plan, chunks);
  else
    hipLaunchKernelGGL((copy_pages_kernel<uint8_t, PAIRS>), grid, dim3(kThreads), 0, stream, plan, chunks);
}

}  // namespace

extern "C" int ms_copy_pages_most_pools() { return kPools; }

// pools: four numbers each, of one [calls, pages, page_bytes]: its address, page_bytes, calls
// and pages; source, destination: `count` page numbers each.  All in host memory, read before the
// call returns.  (What the numbers must be is checked here, before anything is launched: for
// some hundred pages a check in Python takes longer than the copy.)
extern "C" int ms_copy_pages(const int64_t* pools, int num_pools, const int32_t* source, const int32_t* destination,
                             int count, hipStream_t stream) {
  MS_REQUIRE(num_pools >= 1 && num_pools <= kPools, "copy_pages: %d pools are outside 1..%d", num_pools, kPools);
  MS_REQUIRE(count >= 1, "copy_pages: no pages");
  Pool described[kPools] = {};
  int64_t most_bytes = 0, most_calls = 0, least_pages = 0;
  uint64_t alignment = 0;
  for (int p = 0; p < num_pools; ++p) {
    const int64_t base = pools[4 * p], page_bytes = pools[4 * p + 1], calls = pools[4 * p + 2], pages = pools[4 * p + 3];
    MS_REQUIRE(base != 0 && page_bytes > 0 && calls > 0 && calls <= 65535 && pages > 0 && pages < (1LL << 31),
               "copy_pages: pool %d has no pages, 2^31 of them, or more than 65535 calls", p);
    described[p] = Pool{reinterpret_cast<char*>(base), page_bytes, page_bytes * pages, calls};
    most_bytes = page_bytes > most_bytes ? page_bytes : most_bytes;
    most_calls = calls > most_calls ? calls : most_calls;
    least_pages = p == 0 || pages < least_pages ? pages : least_pages;
    alignment |= static_cast<uint64_t>(base) | static_cast<uint64_t>(page_bytes);
  }
  const int fewest_pages = static_cast<int>(least_pages);
  for (int i = 0; i < count; ++i)
    MS_REQUIRE(source[i] >= 0 && source[i] < fewest_pages && destination[i] >= 0 && destination[i] < fewest_pages,
               "copy_pages: page %d or %d lies outside the pools' %d", source[i], destination[i], fewest_pages);
  int twice = -1, both = -1;
  uint8_t* written = static_cast<uint8_t*>(calloc(fewest_pages, 1));
  MS_REQUIRE(written != nullptr, "copy_pages: no memory for a list of %d pages", fewest_pages);
  for (int i = 0; i < count; ++i) {
    if (written[destination[i]]) twice = destination[i];
    written[destination[i]] = 1;
  }
  for (int i = 0; i < count; ++i)
    if (written[source[i]]) both = source[i];
  free(written);
  MS_REQUIRE(twice < 0, "copy_pages: page %d is the destination of two copies", twice);
  MS_REQUIRE(both < 0, "copy_pages: page %d is the source of one copy and the destination of another", both);
  const int word = alignment % 16 == 0 ? 16 : alignment % 4 == 0 ? 4 : 1;
  const int64_t per_group = static_cast<int64_t>(word) * kThreads * kUnroll;
  const int64_t chunks = (most_bytes + per_group - 1) / per_group;
  MS_REQUIRE(chunks * kMostPairs * kThreads < (1LL << 32), "copy_pages: pages of %lld bytes", static_cast<long long>(most_bytes));
  for (int at = 0; at < count; at += kMostPairs) {
    const int here = count - at < kMostPairs ? count - at : kMostPairs;
    if (here <= kFewPairs)
      launch<kFewPairs>(described, num_pools, source + at, destination + at, here, word, static_cast<int>(chunks), static_cast<int>(most_calls), stream);
    else
      launch<kMostPairs>(described, num_pools, source + at, destination + at, here, word, static_cast<int>(chunks), static_cast<int>(most_calls), stream);
    MS_CHECK_LAUNCH("copy_pages");
  }
  return 0;
}
