// Copies of whole pages inside the paged KV pools for gfx950: page src[i] onto page dst[i] of
// K and of V in one launch (copy on write of forked sequences, moves of a compaction).
//
// Bound by HBM: each byte is read and written once, in 16-byte units. A workgroup copies a
// piece of kUnits units per thread of one page of one pool, its loads issued together; the
// pieces of a page have consecutive ids. The destinations must be distinct and none of them a
// source (the pieces run in any order).

#include "ffa_common.h"
#include "ffa_internal.h"

namespace ffa {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kUnits = 4;

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
  const U* const in = pool + from * page_units;
  U* const out = pool + to * page_units;
  const int64_t first = static_cast<int64_t>(piece) * (kCopyThreads * kUnits) + threadIdx.x;
  U x[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t at = first + u * kCopyThreads;
    if (at < page_units) x[u] = in[at];
  }
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t at = first + u * kCopyThreads;
    if (at < page_units) out[at] = x[u];
  }
}

template <typename U>
int run_copy(const ffa_paged_copy_args& a, hipStream_t s) {
  const int64_t units = a.page_bytes / static_cast<int64_t>(sizeof(U));
  const int64_t pieces = (units + kCopyThreads * kUnits - 1) / (kCopyThreads * kUnits);
  if (pieces * a.n_pairs > 0x7fffffff) return FFA_ERR_TOO_LARGE;
  const dim3 grid(static_cast<unsigned>(pieces * a.n_pairs), a.v_pages != nullptr ? 2 : 1);
  hipLaunchKernelGGL((page_copy_kernel<U>), grid, dim3(kCopyThreads), 0, s, static_cast<U*>(a.k_pages),
                     static_cast<U*>(a.v_pages), a.src, a.dst, static_cast<int>(pieces), units, a.num_pages);
  return hipGetLastError() == hipSuccess ? FFA_OK : FFA_ERR_LAUNCH;
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
