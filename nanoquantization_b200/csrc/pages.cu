// Copies of pages in many pools at once: what a fork, its copy on write and a compaction of a paged cache move.
//
// Bound by memory, and for a page or two by the launch: one launch for up to 64 pools and 192 pairs, whose pointers and numbers
// travel as the kernel's parameters (2.5 KB), so that nothing is copied to the device ahead of it.  32 pages of 147 KB in 56 pools: 81 us,
// 6.5 TB/s, the copy rate; one page 4.5 us.
#include "common.cuh"
#include <algorithm>
#include <new>
#include <vector>

namespace nqb200 {
namespace {

constexpr int kPools = 64, kPairs = 192, kThreads = 256, kDeep = 8;

struct CopyArgs {
  uint8_t* pool[kPools];
  int64_t bytes[kPools];
  int32_t source[kPairs], target[kPairs];
};

// A CTA copies kThreads * kDeep words of a row, all of a thread's loads ahead of its stores.
template <typename W>
__device__ __forceinline__ void copy_piece(const uint8_t* src, uint8_t* dst, int64_t bytes) {
  const int64_t words = bytes / (int64_t)sizeof(W), step = (int64_t)gridDim.x * kThreads * kDeep;
  const W* s = reinterpret_cast<const W*>(src);
  W* d = reinterpret_cast<W*>(dst);
  for (int64_t first = (int64_t)blockIdx.x * kThreads * kDeep + threadIdx.x; first < words; first += step) {
    W v[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (first + i * kThreads < words) v[i] = s[first + i * kThreads];
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (first + i * kThreads < words) d[first + i * kThreads] = v[i];
  }
}

__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int p = blockIdx.z;
  const int64_t bytes = a.bytes[p];
  const uint8_t* src = a.pool[p] + a.source[blockIdx.y] * bytes;
  uint8_t* dst = a.pool[p] + a.target[blockIdx.y] * bytes;
  const uint64_t on = reinterpret_cast<uintptr_t>(a.pool[p]) | (uint64_t)bytes;
  if (on % 16 == 0) copy_piece<uint4>(src, dst, bytes);
  else if (on % 4 == 0) copy_piece<uint32_t>(src, dst, bytes);
  else copy_piece<uint8_t>(src, dst, bytes);
}

}  // namespace
}  // namespace nqb200

using namespace nqb200;

extern "C" int nqb200_copy_pages(void* const* pools, const int64_t* row_bytes, int64_t n_pools, int64_t rows, const int32_t* sources, const int32_t* targets,
                                 int64_t n_pairs, void* stream) {
  if (n_pools < 0 || n_pairs < 0 || rows <= 0 || rows > INT32_MAX) return NQB200_ERR_BAD_SHAPE;
  if (n_pools == 0 || n_pairs == 0) return NQB200_OK;
  if (!pools || !row_bytes || !sources || !targets) return NQB200_ERR_NULL_POINTER;
  if (n_pairs > rows) return NQB200_ERR_BAD_INDEX;         // some target comes twice
  int64_t most = 0;
  for (int64_t p = 0; p < n_pools; ++p) {
    if (row_bytes[p] <= 0) return NQB200_ERR_BAD_SHAPE;
    if (!pools[p]) return NQB200_ERR_NULL_POINTER;
    most = std::max(most, row_bytes[p]);
  }
  for (int64_t i = 0; i < n_pairs; ++i)
    if (sources[i] < 0 || sources[i] >= rows || targets[i] < 0 || targets[i] >= rows) return NQB200_ERR_BAD_INDEX;
  try {
    std::vector<int32_t> s(sources, sources + n_pairs), t(targets, targets + n_pairs);
    std::sort(s.begin(), s.end());
    std::sort(t.begin(), t.end());
    if (std::adjacent_find(t.begin(), t.end()) != t.end()) return NQB200_ERR_BAD_INDEX;
    for (int32_t x : t)
      if (std::binary_search(s.begin(), s.end(), x)) return NQB200_ERR_BAD_INDEX;
  } catch (const std::bad_alloc&) {
    return NQB200_ERR_TOO_LARGE;
  }
  const int64_t piece = (int64_t)kThreads * kDeep * 16;
  const unsigned chunks = (unsigned)std::min<int64_t>((most + piece - 1) / piece, 4096);
  for (int64_t p = 0; p < n_pools; p += kPools) {
    for (int64_t i = 0; i < n_pairs; i += kPairs) {
      CopyArgs a = {};
      const int np = (int)std::min<int64_t>(kPools, n_pools - p), ni = (int)std::min<int64_t>(kPairs, n_pairs - i);
      for (int k = 0; k < np; ++k) { a.pool[k] = (uint8_t*)pools[p + k]; a.bytes[k] = row_bytes[p + k]; }
      for (int k = 0; k < ni; ++k) { a.source[k] = sources[i + k]; a.target[k] = targets[i + k]; }
      const int rc = launch_overlapped(copy_pages_kernel, dim3(chunks, (unsigned)ni, (unsigned)np), dim3(kThreads), 0, (cudaStream_t)stream, a);
      if (rc != NQB200_OK) return rc;
    }
  }
  return NQB200_OK;
}
