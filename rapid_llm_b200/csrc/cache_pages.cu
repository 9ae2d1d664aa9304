// Copies of cache pages: pages[layer, target] = pages[layer, source] for a list of (source, target) pairs, all layers of a
// group in one launch.  What a fork needs for the page its branches go on writing in, what compaction moves.
//
// A pure stream: it reads and writes every byte once, so the copy rate bounds it: 600 pages of 64 KB in 36 layers take 427 us,
// 6.6 TB/s; one page's seven copies in 36 layers 4.3 us, 19 MB, most of it the launch.  The pairs ride in the launch's parameters, so a
// call uploads nothing and waits for nothing, and a captured call keeps them.  The host has made sure
// that no page is written twice and none both read and written, so the order of the CTAs does not matter.  Rows of any size are
// taken (per-request states are copied by the same kernel): the unit of a copy is the largest of 16, 8, 4, 2 and 1
// bytes that a page is a multiple of and its address aligned to.
#include <stdlib.h>

#include "common.cuh"

namespace rl {

constexpr int kCopyThreads = 256;
constexpr int kCopyUnits = 4;                    // units a thread has in flight

template <int kPairs>
struct PagePairs {
  int2 of[kPairs];
};
// A list travels in a block of constants of the launch: a short one keeps the launch short, a long one keeps launches few.
constexpr int kFewPairs = 60, kSomePairs = 500, kManyPairs = 3900;

template <typename U, int kPairs>
__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(const __grid_constant__ PagePairs<kPairs> pairs, U* pages, long long layer_units, long long page_units) {
  // (No early start for what follows: attention may fetch cached keys before it waits, and these are some.)
  const int2 pair = pairs.of[blockIdx.y];
  U* layer = pages + static_cast<long long>(blockIdx.z) * layer_units;
  const U* src = layer + pair.x * page_units;
  U* dst = layer + pair.y * page_units;
  pdl_wait();
  for (long long base = static_cast<long long>(blockIdx.x) * (kCopyThreads * kCopyUnits); base < page_units;
       base += static_cast<long long>(gridDim.x) * (kCopyThreads * kCopyUnits)) {
    U held[kCopyUnits];
#pragma unroll
    for (int i = 0; i < kCopyUnits; ++i) {
      const long long at = base + i * kCopyThreads + threadIdx.x;
      if (at < page_units) held[i] = src[at];
    }
#pragma unroll
    for (int i = 0; i < kCopyUnits; ++i) {
      const long long at = base + i * kCopyThreads + threadIdx.x;
      if (at < page_units) dst[at] = held[i];
    }
  }
}

template <typename U, int kPairs>
static int launch_copy(void* pages, const int* pairs, int count, int layers, long long layer_bytes, long long page_bytes, bool pdl,
                       cudaStream_t stream) {
  PagePairs<kPairs> list;
  for (int i = 0; i < count; ++i) list.of[i] = make_int2(pairs[2 * i], pairs[2 * i + 1]);
  for (int i = count; i < kPairs; ++i) list.of[i] = make_int2(0, 0);
  const long long units = page_bytes / static_cast<long long>(sizeof(U));
  const long long per_block = kCopyThreads * kCopyUnits;
  long long blocks = (units + per_block - 1) / per_block;
  if (blocks > 65536) blocks = 65536;
  return launch_kernel(copy_pages_kernel<U, kPairs>, dim3(static_cast<unsigned>(blocks), count, layers), dim3(kCopyThreads), 0, stream, pdl,
                       list, static_cast<U*>(pages), layer_bytes / static_cast<long long>(sizeof(U)), units);
}

template <typename U>
static int copy_as(void* pages, const int* pairs, int count, int layers, long long layer_bytes, long long page_bytes, bool pdl,
                   cudaStream_t stream) {
  for (int at = 0; at < count;) {
    const int left = count - at, take = left <= kFewPairs ? left : left < kManyPairs ? left : kManyPairs;
    const int status = take <= kFewPairs
                           ? launch_copy<U, kFewPairs>(pages, pairs + 2 * at, take, layers, layer_bytes, page_bytes, pdl, stream)
                       : take <= kSomePairs
                           ? launch_copy<U, kSomePairs>(pages, pairs + 2 * at, take, layers, layer_bytes, page_bytes, pdl, stream)
                           : launch_copy<U, kManyPairs>(pages, pairs + 2 * at, take, layers, layer_bytes, page_bytes, pdl, stream);
    if (status != 0) return status;
    at += take;
  }
  return 0;
}

}  // namespace rl

extern "C" {

// Launches a list of `count` pairs takes.
int rl_copy_pages_launches(int count) { return (count + rl::kManyPairs - 1) / rl::kManyPairs; }

// What the pairs of a list break: 0 nothing, -1 a page outside the `known`, -2 a page that is written twice, or read and written,
// -3 no memory for the check.
int rl_copy_pages_check(const int* pairs, int count, long long known) {
  for (int i = 0; i < 2 * count; ++i)
    if (pairs[i] < 0 || pairs[i] >= known) return -1;
  if (count <= 32) {
    for (int i = 0; i < count; ++i)
      for (int j = 0; j < count; ++j)
        if ((i != j && pairs[2 * i + 1] == pairs[2 * j + 1]) || pairs[2 * i + 1] == pairs[2 * j]) return -2;
    return 0;
  }
  unsigned char* used = static_cast<unsigned char*>(calloc(static_cast<size_t>(known), 1));
  if (used == nullptr) return -3;
  int status = 0;
  for (int i = 0; i < count; ++i) used[pairs[2 * i]] = 1;
  for (int i = 0; i < count && status == 0; ++i) {
    if (used[pairs[2 * i + 1]]) status = -2;
    used[pairs[2 * i + 1]] = 1;
  }
  free(used);
  return status;
}

// pages: `layers` blocks of layer_bytes, page p of each at p * page_bytes; pairs: [count, 2] int32 in host memory, read
// before the call returns.  The caller has had the pairs checked.
int rl_copy_pages(void* pages, const int* pairs, int count, int layers, long long layer_bytes, long long page_bytes, int pdl,
                  cudaStream_t stream) {
  if (count == 0 || layers == 0 || page_bytes == 0) return 0;
  if (count < 0 || layers < 0 || layers > 65535 || page_bytes < 0 || layer_bytes < page_bytes) return static_cast<int>(cudaErrorInvalidValue);
  const unsigned long long all = static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(pages)) |
                                 static_cast<unsigned long long>(layer_bytes) | static_cast<unsigned long long>(page_bytes);
  if (all % 16 == 0) return rl::copy_as<uint4>(pages, pairs, count, layers, layer_bytes, page_bytes, pdl != 0, stream);
  if (all % 8 == 0) return rl::copy_as<uint2>(pages, pairs, count, layers, layer_bytes, page_bytes, pdl != 0, stream);
  if (all % 4 == 0) return rl::copy_as<unsigned>(pages, pairs, count, layers, layer_bytes, page_bytes, pdl != 0, stream);
  if (all % 2 == 0) return rl::copy_as<unsigned short>(pages, pairs, count, layers, layer_bytes, page_bytes, pdl != 0, stream);
  return rl::copy_as<unsigned char>(pages, pairs, count, layers, layer_bytes, page_bytes, pdl != 0, stream);
}

}  // extern "C"
