// Copies of whole pages inside the paged KV pools for gfx950: page src[i] onto page dst[i] of
// K and of V in one launch (copy on write of forked sequences, moves of a compaction).
//
// Bound by HBM: each byte is read and written once, in 16-byte units, one per thread; the pieces
// of a page have consecutive ids. The destinations must be distinct and none of them a source
// (the pieces run in any order).
//
// Measured on MI355X: 1009 pages of 128 KB in each of two pools (529 MB read and written) take
// 93 us, 5.7 TB/s; 16 pages of 32 KB 2.4 us. With 1 / 2 / 4 / 8 units per thread, all loads
// ahead of the stores, 92 / 104 / 109 / 144 us: more waves beat more loads per wave. Stores past
// the caches (nontemporal) leave the sources there: 79 us where the Infinity Cache holds part
// of them, 93 where it does not, 92 and 94 with ordinary ones.

#include "ffa_common.h"
#include "ffa_internal.h"

namespace ffa {
namespace {

constexpr int kCopyThreads = 256;
constexpr int64_t kCopyGroups = (1 << 24) - 1;  // workgroups of a launch (2^32 threads at most)

template <typename U>
__global__ __launch_bounds__(kCopyThreads) void page_copy_kernel(U* __restrict__ k, U* __restrict__ v,
                                                                 const int32_t* __restrict__ src,
                                                                 const int32_t* __restrict__ dst,
                                                                 int pieces, int64_t page_units, int num_pages) {
  const int pair = static_cast<int>(blockIdx.x) / pieces;
  const int piece = static_cast<int>(blockIdx.x) - pair * pieces;
  const int from = src[pair];
  const int to = dst[pair];
  // ids outside the pool address nothing; a page onto itself is no copy
  if (from < 0 || from >= num_pages || to < 0 || to >= num_pages || from == to) return;
  U* const pool = blockIdx.y == 0 ? k : v;
  const int64_t at = static_cast<int64_t>(piece) * kCopyThreads + threadIdx.x;
  if (at < page_units) __builtin_nontemporal_store(pool[from * page_units + at], pool + to * page_units + at);
}

template <typename U>
int run_copy(const ffa_paged_copy_args& a, hipStream_t s) {
  const int64_t units = a.page_bytes / static_cast<int64_t>(sizeof(U));
  const int64_t pieces = (units + kCopyThreads - 1) / kCopyThreads;
  if (pieces > kCopyGroups) return FFA_ERR_TOO_LARGE;
  const int64_t most = kCopyGroups / pieces;  // pairs of a launch
  for (int64_t first = 0; first < a.n_pairs; first += most) {
    const int64_t n = a.n_pairs - first < most ? a.n_pairs - first : most;
    const dim3 grid(static_cast<unsigned>(pieces * n), a.v_pages != nullptr ? 2 : 1);
    hipLaunchKernelGGL((page_copy_kernel<U>), grid, dim3(kCopyThreads), 0, s, static_cast<U*>(a.k_pages),
                       static_cast<U*>(a.v_pages), a.src + first, a.dst + first, static_cast<int>(pieces),
                       units, a.num_pages);
    if (hipGetLastError() != hipSuccess) return FFA_ERR_LAUNCH;
  }
  return FFA_OK;
}

}  // namespace

int launch_paged_copy(const ffa_paged_copy_args& a, hipStream_t stream) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages) |
                        static_cast<uint64_t>(a.page_bytes);
  if (bits % 16 == 0) return run_copy<u32x4>(a, stream);
  if (bits % 4 == 0) return run_copy<uint32_t>(a, stream);
  return run_copy<uint16_t>(a, stream);
}

}  // namespace ffa
