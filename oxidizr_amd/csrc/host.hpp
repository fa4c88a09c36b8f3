// Host helpers that the C-ABI sources share: errors, sizes, and the launch plans
// of dense weight gradients and of row tiles.
#pragma once
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/moe_hip.h"
#include "kernels.hpp"

namespace moe {

// Leaves the message for moe_last_error (thread-local) and returns st.
moe_status fail(moe_status st, const char* fmt, ...);

#define HIP_TRY(expr)                                                                   \
  do {                                                                                  \
    hipError_t _e = (expr);                                                             \
    if (_e != hipSuccess)                                                               \
      return fail(_e == hipErrorOutOfMemory ? MOE_ERR_OOM : MOE_ERR_HIP, "%s: %s (%s:%d)", \
                  #expr, hipGetErrorString(_e), __FILE__, __LINE__);                    \
  } while (0)

#define LAUNCH_CHECK()                                                                   \
  do {                                                                                   \
    hipError_t _e = hipGetLastError();                                                   \
    if (_e != hipSuccess)                                                                \
      return fail(MOE_ERR_HIP, "kernel launch: %s (%s:%d)", hipGetErrorString(_e), __FILE__, \
                  __LINE__);                                                             \
  } while (0)

constexpr size_t kAlign = 256;
inline size_t align_up(size_t v) { return (v + kAlign - 1) / kAlign * kAlign; }

// Bump allocator over a caller buffer: records offsets of named regions.
struct Carve {
  size_t off = 0;
  size_t take(size_t bytes) {
    size_t o = off;
    off = align_up(off + bytes);
    return o;
  }
};

inline int elt_size(int dtype) { return dtype == MOE_DTYPE_F32 ? 4 : 2; }

// Buffer loads take 32-bit byte offsets and kOobOffset (2^31) must lie beyond
// every resource: no operand extent may reach this many bytes.
constexpr int64_t kMaxExtentBytes = int64_t(1) << 31;
inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Clears n bytes of device memory at q on stream s with a kernel (graph
// capture records no memset node for it).
static inline moe_status zero_async(hipStream_t s, void* q, size_t n) {
  if (!q) return MOE_OK;
  constexpr size_t kMost = size_t(1) << 35;  // 2^31 threads of 16 bytes, half of what a launch takes
  for (size_t at = 0; at < n; at += kMost) {
    const int64_t part = (int64_t)std::min(kMost, n - at), vecs = (part + 15) / 16;
    hipLaunchKernelGGL(k_zero, dim3((unsigned)((vecs + 255) / 256)), dim3(256), 0, s, (uint8_t*)q + at, part);
  }
  LAUNCH_CHECK();
  return MOE_OK;
}

// Split of a dense (all-token) weight gradient over K = tokens into fixed
// chunks (each at least four k-tiles).  The count minimises a cost model in
// units of one workgroup k-tile: rounds of workgroups on 256 CUs times k-tiles
// per chunk, plus, when split, the fp32 partial tiles written and read back by
// k_splitk_reduce (8 bytes per output element and chunk at ~5 TB/s, against
// ~3.9 TFLOP/s of MFMA work per CU: 3.1 * M * N / (BM * BN * BK) units per
// chunk).  These are the bf16 tilings' rates; fp32 does ~0.6 TFLOP/s per CU and
// holds several workgroups there, so its chunks are priced some six times too
// high and it splits less than would be fastest (M = 776, N = 680, T = 1999: one
// chunk, 144 workgroups).  The split depends only on the shapes, never on timing.
struct SplitPlan {
  int nsplit, kchunk;
};
template <class C>
SplitPlan plan_split(int M, int N, int K) {
  if (K <= 0) return {1, C::BK};  // no tokens: nothing to split
  const int tiles = ceil_div(M, C::BM) * ceil_div(N, C::BN);
  const int nkt = ceil_div(K, C::BK);
  const int most = K / (4 * C::BK) > 1 ? K / (4 * C::BK) : 1;
  const double red = 3.1 * (double)M * N / ((double)C::BM * C::BN * C::BK);
  int best = 1;
  double best_cost = 0;
  for (int ns = 1; ns <= most && ns <= 64; ++ns) {
    const double cost = (double)ceil_div((int64_t)tiles * ns, 256) * ceil_div(nkt, ns) +
                        (ns > 1 ? red * ns : 0.0);
    if (ns == 1 || cost < best_cost) {
      best = ns;
      best_cost = cost;
    }
  }
  const int chunk = ceil_div(ceil_div(K, best), C::BK) * C::BK;
  return {ceil_div(K, chunk), chunk};
}

// The split of one dense weight gradient (NA outputs of M x N over T tokens).
// It also decides how many terms one running fp32 sum holds.  The fp32 pair runs
// 64 x 64 tiles of 16-deep k-tiles, several to a CU, and is planned as 64 x 128
// tiles of 32-deep ones: the cost model has one workgroup to a CU, and on the
// launch's own tile it splits less (a tenth of the shapes with M and N up to some
// thousands).  M = 680, N = 776, T = 1999: 1 chunk instead of 3, and gradients
// 7.9e-7 off a 64-bit sum instead of 4.6e-7 (69 us alone; with 3 chunks 49, and 5
// for their sum).
template <typename D, int NA>
SplitPlan plan_dense_wgrad(int M, int N, int T) {
  using C = WgradTiling<D, NA>;
  using P = typename std::conditional<std::is_same<D, float>::value && NA == 2,
                                      Tiling<float, 64, 128, 32>, C>::type;
  static_assert(P::BK % C::BK == 0, "chunks are whole k-tiles of the launch");
  return plan_split<P>(M, N, T);
}

// fp32 partial-tile bytes of one dense weight gradient (NA outputs of M x N
// over T tokens) as launch_dense_wgrad splits it: 0 when it runs unsplit.
template <typename D, int NA>
inline size_t dense_wgrad_partial_bytes(int M, int N, int T) {
  const SplitPlan sp = plan_dense_wgrad<D, NA>(M, N, T);
  return sp.nsplit > 1 ? (size_t)NA * sp.nsplit * (size_t)M * N * 4 : 0;
}

// Blocks of a K-grouped (weight-gradient) launch over `groups` groups or
// split chunks of an M x N output: each takes 8 * ceil(tiles / 8) blocks.
inline int kgrouped_grid(int groups, int M, int N, int BM, int BN) {
  return groups * 8 * ceil_div(ceil_div(M, BM) * ceil_div(N, BN), 8);
}

// Weight gradient of a dense (all-token) GEMM: out_x[m, n] = alpha * sum_t
// P_x[t, m] Q[t, n], split over tokens when that fills the GPU better.  The
// fp32 partials of a split must fit the partial_bytes of `partial` (else an
// error, before anything is launched).
template <typename D, int NA>
inline moe_status launch_dense_wgrad(hipStream_t s, const D* P0, const D* P1, int64_t ldp, const D* Q,
                              int64_t ldq, int T, int M, int N, float alpha, D* o0, D* o1,
                              float* partial, size_t partial_bytes) {
  using C = WgradTiling<D, NA>;
  const SplitPlan sp = plan_dense_wgrad<D, NA>(M, N, T);
  if (sp.nsplit > 1) {
    const size_t need = dense_wgrad_partial_bytes<D, NA>(M, N, T);
    if (need > partial_bytes)
      return fail(MOE_ERR_UNSUPPORTED,
                  "weight-gradient split of %d chunks needs %zu bytes of partials, the workspace "
                  "holds %zu",
                  sp.nsplit, need, partial_bytes);
  }
  const KGroups kg{nullptr, 1, T, sp.nsplit, sp.kchunk, 1, nullptr};
  const int grid = kgrouped_grid(sp.nsplit, M, N, C::BM, C::BN);
  hipLaunchKernelGGL((k_wgrad<D, NA, false>), dim3(grid), dim3(C::THREADS), 0, s, P0, P1, ldp, Q,
                     ldq, kg, M, N, alpha, nullptr, o0, nullptr, o1, partial, grid, 0);
  if (sp.nsplit > 1) {
    const int64_t MN = (int64_t)M * N;
    hipLaunchKernelGGL(k_splitk_reduce<D>, dim3(ceil_div(MN, 2048), NA), dim3(256), 0, s, partial,
                       sp.nsplit, MN, alpha, o0, o1);
  }
  LAUNCH_CHECK();
  return MOE_OK;
}

// Cost of rounds of row tiles, in units of a tenth of a 256-row tile: `one` for a
// round of up to 256 tiles (one to a CU), `two` for one of up to 512.
struct TileCost {
  double one, two;
};
struct TileCosts {
  double big;  // a round of 256-row tiles
  TileCost mid, small;
};
inline double round_cost(double tiles, const TileCost& c) {
  const double full = std::floor(tiles / 512.0), rest = tiles - 512.0 * full;
  return full * c.two + (rest <= 0.0 ? 0.0 : rest <= 256.0 ? c.one : c.two);
}
inline double big_cost(double tiles, double c) { return std::ceil(tiles / 256.0) * c; }
// Row tiles of height bm over E groups of r rows on average.
inline double group_row_tiles(int E, double r, int bm) { return E * std::max(1.0, r / bm + 0.5); }

}  // namespace moe
