// Copies of whole cache pages inside their pools, in every call (layer) at once: pool[c,
// destination[i]] = pool[c, source[i]] for all c and i.  Sources and destinations are
// disjoint and the destinations distinct (the caller checks), so the copies may run in any
// order; one source may have several destinations.
//
// The page numbers travel with the launch itself, as its arguments: a table in device
// memory would cost a copy from the host before the kernel could start, which for a fork's
// one page takes longer than the copy of the page.  A launch carries kPairs of them.
#include "common.hpp"

namespace {

constexpr int kPools = 4;        // of one launch (keys and values, or a mixer's own planes)
constexpr int kPairs = 480;      // together 4,000 bytes of arguments
constexpr int kThreads = 256;
constexpr int kUnroll = 4;       // accesses a thread has in flight

struct Plan {
  char* base[kPools];
  int64_t page_bytes[kPools];
  int64_t call_bytes[kPools];
  int32_t calls[kPools];
  int32_t source[kPairs];
  int32_t destination[kPairs];
};

// One workgroup copies kThreads * kUnroll accesses of one page of one call.
template <typename Word>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(Plan plan, int chunks) {
  const int pair = blockIdx.x / chunks, chunk = blockIdx.x - pair * chunks;
  const int call = blockIdx.y, pool = blockIdx.z;
  if (call >= plan.calls[pool]) return;
  const int64_t words = plan.page_bytes[pool] / static_cast<int64_t>(sizeof(Word));
  char* in_call = plan.base[pool] + call * plan.call_bytes[pool];
  const Word* from = reinterpret_cast<const Word*>(in_call + plan.source[pair] * plan.page_bytes[pool]);
  Word* to = reinterpret_cast<Word*>(in_call + plan.destination[pair] * plan.page_bytes[pool]);
  const int64_t first = static_cast<int64_t>(chunk) * kThreads * kUnroll + threadIdx.x;
  Word kept[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t at = first + u * kThreads;
    if (at < words) kept[u] = from[at];
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t at = first + u * kThreads;
    if (at < words) to[at] = kept[u];
  }
}

}  // namespace

extern "C" int ms_copy_pages_most_pools() { return kPools; }

// bases, page_bytes, calls, pages: one entry a pool [calls, pages, page_bytes]; source,
// destination: `count` page numbers each.  All in host memory, read before the call returns.
extern "C" int ms_copy_pages(const void* const* bases, const int64_t* page_bytes, const int32_t* calls,
                             const int32_t* pages, int num_pools, const int32_t* source, const int32_t* destination,
                             int count, hipStream_t stream) {
  MS_REQUIRE(num_pools >= 1 && num_pools <= kPools, "copy_pages: %d pools are outside 1..%d", num_pools, kPools);
  MS_REQUIRE(count >= 1, "copy_pages: no pages");
  Plan plan = {};
  int64_t most_bytes = 0;
  int32_t most_calls = 0;
  uint64_t alignment = 0;
  for (int p = 0; p < num_pools; ++p) {
    MS_REQUIRE(bases[p] != nullptr && page_bytes[p] > 0 && calls[p] > 0 && calls[p] <= 65535 && pages[p] > 0,
               "copy_pages: pool %d has no pages, or more than 65535 calls", p);
    plan.base[p] = static_cast<char*>(const_cast<void*>(bases[p]));
    plan.page_bytes[p] = page_bytes[p];
    plan.call_bytes[p] = page_bytes[p] * pages[p];
    plan.calls[p] = calls[p];
    most_bytes = page_bytes[p] > most_bytes ? page_bytes[p] : most_bytes;
    most_calls = calls[p] > most_calls ? calls[p] : most_calls;
    alignment |= reinterpret_cast<uint64_t>(bases[p]) | static_cast<uint64_t>(page_bytes[p]);
    for (int i = 0; i < count; ++i)
      MS_REQUIRE(source[i] >= 0 && source[i] < pages[p] && destination[i] >= 0 && destination[i] < pages[p],
                 "copy_pages: page %d or %d lies outside the pool's %d", source[i], destination[i], pages[p]);
  }
  const int word = alignment % 16 == 0 ? 16 : alignment % 4 == 0 ? 4 : 1;
  const int64_t per_group = static_cast<int64_t>(word) * kThreads * kUnroll;
  const int64_t chunks = (most_bytes + per_group - 1) / per_group;
  MS_REQUIRE(chunks * kPairs < (1LL << 31), "copy_pages: pages of %lld bytes", static_cast<long long>(most_bytes));
  for (int at = 0; at < count; at += kPairs) {
    const int here = count - at < kPairs ? count - at : kPairs;
    for (int i = 0; i < here; ++i) {
      plan.source[i] = source[at + i];
      plan.destination[i] = destination[at + i];
    }
    const dim3 grid(static_cast<unsigned>(chunks * here), most_calls, num_pools);
    if (word == 16)
      hipLaunchKernelGGL((copy_pages_kernel<uint4>), grid, dim3(kThreads), 0, stream, plan, static_cast<int>(chunks));
    else if (word == 4)
      hipLaunchKernelGGL((copy_pages_kernel<uint32_t>), grid, dim3(kThreads), 0, stream, plan, static_cast<int>(chunks));
    else
      hipLaunchKernelGGL((copy_pages_kernel<uint8_t>), grid, dim3(kThreads), 0, stream, plan, static_cast<int>(chunks));
    MS_CHECK_LAUNCH("copy_pages");
  }
  return 0;
}
