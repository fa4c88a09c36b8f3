// C ABI of the operators beside the MoE layer: tokens sorted by expert and back,
// expert products with bias, activation and residual, norms around a block.
// Declared in include/moe_hip.h.  The calls keep no state: sizes in, device
// pointers in, launches on the call's stream.
#include "host.hpp"
#include "linear.hpp"
#include "ops.hpp"

using namespace moe;

namespace {

// Makes `device` current for one call and the caller's device current after it.
struct DeviceScope {
  int before = -1, device;
  bool changed = false;
  explicit DeviceScope(int d) : device(d) {}
  hipError_t enter() {
    hipError_t e = hipGetDevice(&before);
    if (e != hipSuccess || before == device) return e;
    e = hipSetDevice(device);
    changed = e == hipSuccess;
    return e;
  }
  ~DeviceScope() {
    if (changed) (void)hipSetDevice(before);
  }
};

moe_status check_pointers(std::initializer_list<const void*> needed,
                          std::initializer_list<const void*> optional = {}) {
  for (const void* p : needed) {
    if (!p) return fail(MOE_ERR_INVALID, "a required pointer is NULL");
    if (!aligned16(p)) return fail(MOE_ERR_INVALID, "device pointers must be 16-byte aligned");
  }
  for (const void* p : optional)
    if (p && !aligned16(p)) return fail(MOE_ERR_INVALID, "device pointers must be 16-byte aligned");
  return MOE_OK;
}

moe_status check_dtype(int dtype) {
  if (dtype != MOE_DTYPE_F32 && dtype != MOE_DTYPE_BF16)
    return fail(MOE_ERR_INVALID, "unknown dtype %d", dtype);
  return MOE_OK;
}

// Integer arrays (indices, orders, offsets) need their own alignment only: they may be
// slices of one allocation.
moe_status check_ints(std::initializer_list<const void*> needed, size_t bytes = 4) {
  for (const void* p : needed) {
    if (!p) return fail(MOE_ERR_INVALID, "a required pointer is NULL");
    if ((uintptr_t)p % bytes) return fail(MOE_ERR_INVALID, "an integer array is not aligned");
  }
  return MOE_OK;
}

// Whether a launch of `blocks` workgroups of `threads` fits a grid.
constexpr int64_t kMaxGridThreads = int64_t(1) << 32;
moe_status check_grid(int64_t blocks, int threads) {
  if (blocks * threads >= kMaxGridThreads)
    return fail(MOE_ERR_UNSUPPORTED, "too many rows or tiles for one launch: split the batch");
  return MOE_OK;
}

// ---- sort by expert
constexpr int64_t kMaxAssignments = (int64_t(1) << 31) - 1;  // positions are int32
struct SortPlan {
  int64_t N, chunk;
  int blocks;
  size_t bytes;
};
SortPlan sort_plan(int64_t T, int k, int E) {
  SortPlan p{};
  p.N = T * k;
  const int64_t tiles = (p.N + kSortTile - 1) / kSortTile;
  p.chunk = kSortTile * std::max<int64_t>(1, (tiles + kSortMaxBlocks - 1) / kSortMaxBlocks);
  p.blocks = (int)std::max<int64_t>(1, (p.N + p.chunk - 1) / p.chunk);
  p.bytes = p.blocks > 1 ? align_up((size_t)p.blocks * (E + 1) * sizeof(int)) : 0;
  return p;
}
moe_status check_sort(int64_t T, int k, int E) {
  if (T < 0) return fail(MOE_ERR_INVALID, "num_tokens is negative");
  if (k < 1 || k > kMaxPerTok)
    return fail(MOE_ERR_INVALID, "experts_per_tok %d is outside 1..%d", k, kMaxPerTok);
  if (E < 1 || E > 1024) return fail(MOE_ERR_INVALID, "num_experts %d is outside 1..1024", E);
  if (T > kMaxAssignments / k)
    return fail(MOE_ERR_UNSUPPORTED, "num_tokens x experts_per_tok reaches 2^31");
  return MOE_OK;
}

template <typename I>
moe_status launch_sort(hipStream_t s, const SortPlan& p, int E, const I* idx, int* counts,
                       int* offsets, int* perm, int* inv, int* hist) {
  const size_t row = (size_t)(E + 1) * sizeof(int);
  if (p.blocks > 1)
    hipLaunchKernelGGL(k_sort_hist<I>, dim3(p.blocks), dim3(kSortThreads), row, s, idx, p.N, E,
                       p.chunk, hist);
  hipLaunchKernelGGL(k_sort_scatter<I>, dim3(p.blocks), dim3(kSortThreads), kSortWaves * row, s,
                     idx, p.N, E, p.chunk, hist, counts, offsets, perm, inv);
  LAUNCH_CHECK();
  return MOE_OK;
}

// ---- rows to experts and back
moe_status check_rows(int dtype, int64_t T, int k, int H) {
  moe_status st = check_dtype(dtype);
  if (st != MOE_OK) return st;
  if ((st = check_sort(T, k, 1)) != MOE_OK) return st;
  if (H < 8 || H % 8 != 0) return fail(MOE_ERR_INVALID, "hidden %d is not a positive multiple of 8", H);
  return MOE_OK;
}

// Calls f(integral constant >= k): the k rows of a token are held in registers.
template <class F>
void with_k(int k, F&& f) {
  if (k <= 2) f(std::integral_constant<int, 2>());
  else if (k <= 4) f(std::integral_constant<int, 4>());
  else if (k <= 8) f(std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 16>());
}

template <typename D>
moe_status launch_permute(hipStream_t s, int64_t T, int k, int H, const int* inv, const int* kept,
                          const D* x, D* xp) {
  const int64_t grid = (T * ceil_div(H, 64 * Vec16<D>::N) + 3) / 4;
  moe_status st = check_grid(grid, 256);
  if (st != MOE_OK) return st;
  hipLaunchKernelGGL(k_permute<D>, dim3((unsigned)grid), dim3(256), 0, s, x, inv, kept, T, k, H, xp);
  LAUNCH_CHECK();
  return MOE_OK;
}

template <typename D>
moe_status launch_unpermute(hipStream_t s, int64_t T, int k, int H, const int* inv,
                            const int* kept, const D* y, const float* w, D* out) {
  const int64_t grid = (T * ceil_div(H, 64 * Vec16<D>::N) + 3) / 4;
  moe_status st = check_grid(grid, 256);
  if (st != MOE_OK) return st;
  const bool stream = T * k * H * (int64_t)sizeof(D) > kStreamBytes;
  with_k(k, [&](auto kc) {
    constexpr int KM = decltype(kc)::value;
    if (stream)
      hipLaunchKernelGGL((k_unpermute<D, KM, true>), dim3((unsigned)grid), dim3(256), 0, s, y, inv, kept, w, T,
                         k, H, out);
    else
      hipLaunchKernelGGL((k_unpermute<D, KM, false>), dim3((unsigned)grid), dim3(256), 0, s, y, inv, kept, w, T,
                         k, H, out);
  });
  LAUNCH_CHECK();
  return MOE_OK;
}

template <typename D>
moe_status launch_unpermute_bwd(hipStream_t s, int64_t T, int k, int H, const int* inv,
                                const int* kept, const D* dout, const D* y, const float* w, D* dy,
                                float* dw) {
  const int slices = ceil_div(H, 64 * Vec16<D>::N);
  moe_status st = MOE_OK;
  with_k(k, [&](auto kc) {
    constexpr int KM = decltype(kc)::value;
    auto go = [&](auto wpt) {
      constexpr int W = decltype(wpt)::value;
      const int64_t grid = (T + 4 / W - 1) / (4 / W);
      if ((st = check_grid(grid, 256)) != MOE_OK) return;
      hipLaunchKernelGGL((k_unpermute_bwd<D, W, KM>), dim3((unsigned)grid), dim3(256), 0, s, dout, y, inv, kept, w, T,
                         k, H, dy, dw);
    };
    if (slices == 1) go(std::integral_constant<int, 1>());
    else if (slices == 2) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 4>());
  });
  if (st != MOE_OK) return st;
  LAUNCH_CHECK();
  return MOE_OK;
}

// ---- norms around a block
constexpr int kNormMaxHidden = 32768;
moe_status check_norm(int dtype, int64_t T, int H, int gate_kind, bool y, bool post, bool gate,
                      bool next, float scale) {
  moe_status st = check_dtype(dtype);
  if (st != MOE_OK) return st;
  if (T < 0 || T >= (int64_t(1) << 31)) return fail(MOE_ERR_INVALID, "num_tokens is outside 0..2^31-1");
  if (H < 8 || H % 8 != 0) return fail(MOE_ERR_INVALID, "hidden %d is not a positive multiple of 8", H);
  if (H > kNormMaxHidden)
    return fail(MOE_ERR_UNSUPPORTED, "hidden %d is above %d", H, kNormMaxHidden);
  if (gate_kind < kGateNone || gate_kind > kGateFull)
    return fail(MOE_ERR_INVALID, "unknown gate kind %d", gate_kind);
  if (T == 0) return MOE_OK;  // no rows: their tensors may have no address
  if ((gate_kind != kGateNone) != gate)
    return fail(MOE_ERR_INVALID, "gate and gate_kind do not go together");
  if (!y && (post || gate))
    return fail(MOE_ERR_INVALID, "a post norm or a gate needs the block's output y");
  if (!y && !next) return fail(MOE_ERR_INVALID, "neither y nor next_weight: nothing to compute");
  if (!y && scale != 1.0f) return fail(MOE_ERR_INVALID, "residual_scale needs the block's output y");
  return MOE_OK;
}

// Calls f(waves to a row, chunks to a thread) with 64 * 8 * WPR * NCH >= H. The backward
// holds more to a column, so it takes one chunk to a thread as long as a workgroup has
// the waves (H = 7168, T = 8192: 8 waves of two chunks 137 us, 16 of one 136; without
// the next row's loads in flight 270 and 183).
template <bool BWD, class F>
void with_norm_shape(int H, F&& f) {
  using std::integral_constant;
  if (H <= 512) f(integral_constant<int, 1>(), integral_constant<int, 1>());
  else if (H <= 2048) f(integral_constant<int, 4>(), integral_constant<int, 1>());
  else if (H <= 4096) f(integral_constant<int, 8>(), integral_constant<int, 1>());
  else if (H <= 8192) f(integral_constant<int, BWD ? 16 : 8>(), integral_constant<int, BWD ? 1 : 2>());
  else if (H <= 16384) f(integral_constant<int, 16>(), integral_constant<int, 2>());
  else f(integral_constant<int, 16>(), integral_constant<int, 4>());
}
constexpr int norm_waves(int wpr) { return wpr > 4 ? wpr : 4; }
constexpr int norm_rows(int wpr) { return norm_waves(wpr) / wpr; }

// Blocks of the backward: 16 waves to a CU, each adding its rows' column sums. bf16 ones all
// run at once (four waves to a SIMD); fp32 ones up to H = 4096 take 150 to 168 registers, three waves
// to a SIMD, so 768 of 1024 blocks (H <= 2048) or 256 of 512 run in the first round and the others
// behind them. More blocks write more partial rows and gain nothing (bf16 H = 7168, T = 8192: 256
// blocks 136 us, 512 143, 1024 153; H = 2048: 1024 43, 4096 47).
constexpr int kNormBwdWaves = 16 * 256;
int norm_bwd_blocks(int64_t T, int H) {
  int64_t blocks = 1;
  with_norm_shape<true>(H, [&](auto wpr, auto) {
    constexpr int W = decltype(wpr)::value;
    blocks = std::min<int64_t>(kNormBwdWaves / norm_waves(W), (T + norm_rows(W) - 1) / norm_rows(W));
  });
  return (int)blocks;
}

template <typename D>
moe_status launch_norm_fwd(hipStream_t s, const NormArgs<D>& a) {
  moe_status st = MOE_OK;
  with_norm_shape<false>(a.H, [&](auto wpr, auto nch) {
    constexpr int W = decltype(wpr)::value;
    const int64_t grid = (a.Tn + norm_rows(W) - 1) / norm_rows(W);
    if ((st = check_grid(grid, 64 * norm_waves(W))) != MOE_OK) return;
    hipLaunchKernelGGL((k_norm_fwd<D, W, decltype(nch)::value>), dim3((unsigned)grid),
                       dim3(64 * norm_waves(W)), 0, s, a);
  });
  if (st != MOE_OK) return st;
  LAUNCH_CHECK();
  return MOE_OK;
}

template <typename D>
moe_status launch_norm_bwd(hipStream_t s, const NormBwdArgs<D>& a, D* dw2, D* dgate_chan, D* dw3) {
  const int nb = norm_bwd_blocks(a.Tn, a.H);
  with_norm_shape<true>(a.H, [&](auto wpr, auto nch) {
    constexpr int W = decltype(wpr)::value;
    hipLaunchKernelGGL((k_norm_bwd<D, W, decltype(nch)::value>), dim3(nb), dim3(64 * norm_waves(W)), 0,
                       s, a);
  });
  if (a.need_a + a.need_b > 0)
    hipLaunchKernelGGL(k_norm_colsum<D>, dim3(ceil_div(a.H, kColsumCols), a.need_a + a.need_b), dim3(256), 0,
                       s, a.part, nb, a.H, a.need_a, a.need_b, a.w2,
                       a.gate_kind == kGateChannel ? a.gate : nullptr, dw2, dgate_chan, dw3);
  LAUNCH_CHECK();
  return MOE_OK;
}

// hn_given: h is the forward's h_out in place of its h.
moe_status norm_backward(int device, void* stream, int dtype, int64_t T, int H, bool hn_given,
                         const void* d_h_out, const void* d_n_out, const void* h, const void* y,
                         const void* post_weight, const void* gate, int gate_kind,
                         const void* next_weight, float residual_scale, const float* rstd_post,
                         const float* rstd_next, void* d_h, void* d_y, void* d_post_weight,
                         void* d_gate, void* d_next_weight, void* workspace) {
  moe_status st = check_norm(dtype, T, H, gate_kind, y, post_weight, gate, next_weight,
                             residual_scale);
  if (st != MOE_OK) return st;
  if ((st = check_pointers({}, {d_h_out, d_n_out, h, y, post_weight, gate, next_weight,
                                rstd_post, rstd_next, d_h, d_y, d_post_weight, d_gate,
                                d_next_weight, workspace})) != MOE_OK)
    return st;
  const size_t b = elt_size(dtype);
  DeviceScope dev(device);
  hipStream_t s = (hipStream_t)stream;
  if (T == 0) {  // sums over no row
    HIP_TRY(dev.enter());
    if ((st = zero_async(s, d_post_weight, H * b)) != MOE_OK) return st;
    if ((st = zero_async(s, gate_kind == kGateChannel ? d_gate : nullptr, H * b)) != MOE_OK) return st;
    return zero_async(s, d_next_weight, H * b);
  }
  if (!d_h || (y && !d_y) || !workspace || (post_weight && (!d_post_weight || !rstd_post)) ||
      (gate && !d_gate) || (next_weight && !d_next_weight) ||
      (next_weight && (!rstd_next || !h || !d_n_out)) || (!next_weight && !d_h_out))
    return fail(MOE_ERR_INVALID, "a required pointer is NULL");
  HIP_TRY(dev.enter());
  const bool chan = gate_kind == kGateChannel;
  auto go = [&](auto d) {
    using D = decltype(d);
    const NormBwdArgs<D> a{(const D*)d_h_out, (const D*)d_n_out, (const D*)h, (const D*)y,
                           (const D*)post_weight, (const D*)gate, (const D*)next_weight, gate_kind,
                           hn_given ? 1 : 0, residual_scale, T, H, rstd_post, rstd_next, (D*)d_h, (D*)d_y,
                           chan ? nullptr : (D*)d_gate, (float*)workspace,
                           post_weight || chan ? 1 : 0, next_weight ? 1 : 0};
    return launch_norm_bwd<D>(s, a, (D*)d_post_weight, chan ? (D*)d_gate : nullptr,
                              (D*)d_next_weight);
  };
  return dtype == MOE_DTYPE_BF16 ? go(bf16_t()) : go(float());
}

// ---- expert products
constexpr int kLinearMaxWidth = 1 << 20;
moe_status check_linear(int dtype, int64_t M, int K, int N, int E, bool grouped, int act) {
  moe_status st = check_dtype(dtype);
  if (st != MOE_OK) return st;
  if (M < 0) return fail(MOE_ERR_INVALID, "num_rows is negative");
  if (K < 8 || K % 8 != 0 || N < 8 || N % 8 != 0)
    return fail(MOE_ERR_INVALID, "in_features %d and out_features %d must be positive multiples of 8",
                K, N);
  if (grouped ? (E < 1 || E > 1024) : E != 1)
    return fail(MOE_ERR_INVALID, grouped ? "num_groups %d is outside 1..1024"
                                         : "num_groups %d without offsets is not 1", E);
  if (act < 0 || act >= kNumActs) return fail(MOE_ERR_INVALID, "unknown activation %d", act);
  if (K > kLinearMaxWidth || N > kLinearMaxWidth)
    return fail(MOE_ERR_UNSUPPORTED, "in_features %d or out_features %d is above %d", K, N,
                kLinearMaxWidth);
  const int64_t b = elt_size(dtype);
  if ((int64_t)K * N * b >= kMaxExtentBytes)
    return fail(MOE_ERR_UNSUPPORTED, "a weight matrix reaches 2^31 bytes");
  if (M > (int64_t(1) << 26) || M * std::max(K, N) * b >= kMaxExtentBytes * 8)
    return fail(MOE_ERR_UNSUPPORTED, "num_rows x max(in, out features) reaches 2^34 bytes");
  return MOE_OK;
}

// Waves of k_linear_skinny to a block of 16 weight rows: four with two k-chunks each at
// least, two where K holds fewer (4096 x 4096, one row: 12.0 -> 7.6 us; 64 experts of 1408 x
// 2048, one row each, six chunks: 40 -> 46; eight waves: 7.5 and 60).
template <typename D>
int skinny_split(int K) {
  return K >= 8 * kSkinnyChunkBytes / (int)sizeof(D) ? 4 : 2;
}
int64_t skinny_slots(int64_t M, int E, bool grouped) {
  return grouped ? std::min<int64_t>(E, M) + M / kLinearSkinnyRows : ceil_div(M, kLinearSkinnyRows);
}
int64_t skinny_blocks(int64_t M, int N, int E, bool grouped, int split) {
  return skinny_slots(M, E, grouped) * ceil_div(N, 64 / split) + (grouped ? 64 : 0);
}

// Whether a forward runs as the stream of its weights (k_linear_skinny): few rows to
// an expert (rows counted as evenly spread over the experts that can have any), or
// somewhat more where the row tiles would leave half of the CUs idle. us, tiles / this,
// at 1, 4, 8, 16 rows an expert: bf16 128 experts of 4096 x 1536 181 / 168, 267 / 258, 276 /
// 302, 288 / 404; 64 of 1408 x 2048 43 / 40, 68 / 70, 73 / 81, 74 / 104; 8 of 1024 x 512 14 /
// 4.4, 15 / 5.7, 15 / 5.7, 15 / 7.7; fp32 448 / 337, 756 / 537, 780 / 636, 809 / 802. One weight of
// 4096 x 4096 at 1, 16, 32, 64 rows: 24 / 7.6, 24 / 10.6, 25 / 16, 27 / 26; 1408 x 7168 11 / 5.7, 10
// / 8.3, 11 / 12, 13 / 19; fp32 81 / 18, 81 / 20, 82 / 29, 82 / 45 and 30 / 10, 30 / 14, 32 / 21, 32 / 33.
template <typename D>
bool linear_skinny(int64_t M, int K, int N, int E, bool grouped) {
  const int64_t groups = grouped ? std::min<int64_t>(E, M) : 1;
  // a thousand experts a million columns wide can be more workgroups than a launch holds
  if (skinny_blocks(M, N, E, grouped, skinny_split<D>(K)) * 256 >= kMaxGridThreads) return false;
  const bool idle = groups * ceil_div(N, 128) <= (grouped ? 128 : 32);
  if (sizeof(D) == 4) return M <= (grouped ? 16 * groups : kLinearSkinnyRows);
  if (grouped) return M <= (idle ? 16 : 4) * groups;
  return M <= (idle ? kLinearSkinnyRows : 24);
}

// Row tilings of a product alone on the GPU, in tenths of a round of 256-row tiles (one
// to a CU). Measured on dense products of random bf16 rows (zeros run at higher
// clocks), us, 256-row / 384-row / 128 x 128 / 64 x 128 tiles: M = 16384, N = 2048, K = 1408
// 82 / 106 / 95 / 125; 16384, 1408, 2048 107 / 140 / 97 / -; 8192, 2816, 2048 98 / 82 / 98 /
// 125; 8192, 2048, 2816 76 / 98 / 90 / 122; 4096, 2048, 2816 63 / 87 / 47 / 64; 4096, 1408,
// 2048 45 / 63 / 31 / 34; 1000, 2048, 2816 53 / 82 / 33 / 21; 300, 7168, 2048 41 / 51 / 25 / 23.
constexpr TileCosts kLinearCosts{10.0, {4.8, 6.3}, {2.9, 4.3}};
// A 384-row tile against a 256-row one (its kernel spills 40 registers, 84 bytes a lane, around the
// epilogue, and was measured so).
constexpr double kTallCost = 1.55;

enum class RowTiles { kBig, kTall, kMid, kSmall };
template <typename D>
double tile_count(bool grouped, int E, int64_t M, int N, int bm, int bn) {
  const int groups = grouped ? (int)std::min<int64_t>(E, M) : 1;
  return (grouped ? group_row_tiles(groups, (double)M / groups, bm) : (double)ceil_div(M, bm)) *
         ceil_div(N, bn);
}
// The row tiles of a product of M rows in E groups (or dense) with N output columns.
template <typename D>
RowTiles pick_tiles(bool grouped, int E, int64_t M, int N) {
  using C = typename Tilings<D>::Big;
  if constexpr (has_half_rows<D, C>()) {
    using CM = typename LowTilings<C>::Mid;
    using CS = typename LowTilings<C>::Small;
    auto tiles = [&](int bm, int bn) { return tile_count<D>(grouped, E, M, N, bm, bn); };
    const double big = big_cost(tiles(C::BM, C::BN), kLinearCosts.big);
    const double mid = round_cost(tiles(CM::BM, CM::BN), kLinearCosts.mid);
    const double small = round_cost(tiles(CS::BM, CS::BN), kLinearCosts.small);
    // groups of fewer rows would run most of their 384-row tiles as shorter ones
    const bool tall_ok = !grouped || M >= 2 * (int64_t)Rows384<C>::AR * E;
    const double tall =
        tall_ok ? big_cost(tiles(Rows384<C>::AR, C::BN), kLinearCosts.big * kTallCost) : 1e30;
    if (std::min(mid, small) < std::min(big, tall))
      return mid <= small ? RowTiles::kMid : RowTiles::kSmall;
    if (tall < big) return RowTiles::kTall;
  }
  return RowTiles::kBig;
}

// Blocks of a launch of C over M rows in E groups, or dense, with N output columns.
template <class C>
constexpr int prefix_rows() { return C::XR == 128 ? C::AR : C::BM; }
template <class C>
int64_t row_grid(bool grouped, int E, int64_t M, int N) {
  if (!grouped) return (int64_t)ceil_div(M, C::AR) * ceil_div(N, C::BN);
  const int64_t mt = ceil_div(M, prefix_rows<C>()) + E;
  return (mt * ceil_div(N, C::BN) + 7) / 8 * 8;
}

// Calls f(tiling).
template <typename D, class F>
void with_tiling(RowTiles kind, F&& f) {
  using C = typename Tilings<D>::Big;
  if constexpr (has_half_rows<D, C>()) {
    if (kind == RowTiles::kTall) return f(Rows384<C>{});
    if (kind == RowTiles::kMid) return f(typename LowTilings<C>::Mid{});
    if (kind == RowTiles::kSmall) return f(typename LowTilings<C>::Small{});
  }
  f(C{});
}
// Whether that launch, behind `before` other blocks, fits a grid.
template <typename D>
moe_status check_tiles(RowTiles kind, bool grouped, int E, int64_t M, int N, int64_t before = 0) {
  moe_status st = MOE_OK;
  with_tiling<D>(kind, [&](auto c) {
    using C = decltype(c);
    st = check_grid(before + row_grid<C>(grouped, E, M, N), C::THREADS);
  });
  return st;
}

// Calls f(tiling, row groups, grid) for a launch of M rows in E groups (offsets and
// prefixes of k_linear_prep), or dense (offsets null), with N output columns.
template <typename D, class F>
void with_row_tiles(RowTiles kind, const int* offsets, const int* prefixes, int E, int64_t M, int N,
                    F&& f) {
  with_tiling<D>(kind, [&](auto c) {
    using C = decltype(c);
    const bool grouped = offsets != nullptr;
    const int grid = (int)row_grid<C>(grouped, E, M, N);
    if (!grouped) return f(c, RowGroups{nullptr, nullptr, nullptr, nullptr, 1, (int)M, 0, 0}, grid);
    const int* tp = prefixes + prefix_slot(prefix_rows<C>()) * (E + 1);
    constexpr bool tall = C::XR == 128, big = std::is_same<C, typename Tilings<D>::Big>::value && sizeof(D) == 2;
    const int half_last = tall || (big && M >= 2 * (int64_t)C::BM * E);
    f(c, RowGroups{offsets, tp, tp + (E + 1), tp + 2 * (E + 1), E, (int)M, half_last, big ? tall_rows_for(C::BM) : 0},
      grid);
  });
}

// Both products of a backward as one launch (k_linear_bwd): its estimated time, in
// 64-deep k-tiles of a 256 x 256 tile. The weight gradient's tiles start first; work
// that is left when they end is dealt tile by tile, so the last tiles end half a tile
// apart on average. An epilogue costs about seven k-tiles.
constexpr double kEpilogueTiles = 7.0;
double bwd_cost(double wtiles, double wdepth, double dtiles, double ddepth) {
  const double w = wdepth + kEpilogueTiles, d = ddepth + kEpilogueTiles;
  return std::max(w, (wtiles * w + dtiles * d) / 256.0 + 0.5 * d);
}
struct BwdPlan {
  SplitPlan split;  // chunks of the weight gradient's rows (dense only)
  RowTiles tiles;   // of the input gradient
  bool fused;
};
template <typename D>
BwdPlan plan_bwd(bool grouped, int E, int64_t M, int K, int N) {
  using C = typename Tilings<D>::Big;
  BwdPlan p;
  p.split = grouped ? SplitPlan{1, 0} : plan_dense_wgrad<D, 1>(N, K, (int)M);
  p.tiles = pick_tiles<D>(grouped, E, M, K);
  p.fused = false;
  if (M == 0) return p;  // no rows to plan for: nothing is launched
  if constexpr (has_half_rows<D, C>()) {
    if (p.tiles != RowTiles::kBig && p.tiles != RowTiles::kTall) return p;
    p.fused = true;
    const int groups = grouped ? (int)std::min<int64_t>(E, M) : 1;
    const double wtiles = (double)groups * ceil_div(N, C::BM) * ceil_div(K, C::BN);
    const double red = 3.1 * (double)N * K / ((double)C::BM * C::BN * C::BK);  // see plan_split
    const int nkt = ceil_div((M + groups - 1) / groups, C::BK);
    const int most = grouped ? 1 : std::max(1, std::min(64, nkt / 4));
    const double dtiles = tile_count<D>(grouped, E, M, K, C::BM, C::BN);
    const double ttiles = tile_count<D>(grouped, E, M, K, Rows384<C>::AR, C::BN);
    const double depth = ceil_div(N, C::BK);
    const bool tall_ok = p.tiles == RowTiles::kTall;
    double best = 0;
    for (int ns = 1; ns <= most; ++ns) {
      const double d = ceil_div(nkt, ns), extra = ns > 1 ? red * ns : 0.0;
      const double big = bwd_cost(wtiles * ns, d, dtiles, depth) + extra;
      const double tall = tall_ok ? bwd_cost(wtiles * ns, d, ttiles, depth * kTallCost) + extra : 1e30;
      const double cost = std::min(big, tall);
      if (ns == 1 || cost < best) {
        best = cost;
        if (!grouped) {
          const int chunk = ceil_div(ceil_div(M, ns), C::BK) * C::BK;
          p.split = {ceil_div(M, chunk), chunk};
        }
        p.tiles = big <= tall ? RowTiles::kBig : RowTiles::kTall;
      }
    }
  }
  return p;
}

template <typename D>
int wgrad_blocks(const BwdPlan& p, bool grouped, int E, int K, int N) {
  using CW = WgradTiling<D, 1>;
  return kgrouped_grid(grouped ? E : p.split.nsplit, N, K, CW::BM, CW::BN);
}
// Whether the launches of a forward, or of a backward of dx and dw (as asked for), fit their grids.
template <typename D>
moe_status check_launches(bool backward, bool grouped, int E, int64_t M, int K, int N, bool dx, bool dw) {
  if (!backward)
    return linear_skinny<D>(M, K, N, E, grouped) ? MOE_OK
                                                 : check_tiles<D>(pick_tiles<D>(grouped, E, M, N), grouped, E, M, N);
  const BwdPlan p = plan_bwd<D>(grouped, E, M, K, N);
  const int64_t wblocks = dw ? wgrad_blocks<D>(p, grouped, E, K, N) : 0;
  moe_status st = check_grid(wblocks, WgradTiling<D, 1>::THREADS);
  if (st == MOE_OK && dx) st = check_tiles<D>(p.tiles, grouped, E, M, K, p.fused ? wblocks : 0);
  return st;
}
moe_status check_launches(int dtype, bool backward, bool grouped, int E, int64_t M, int K, int N, bool dx, bool dw) {
  return dtype == MOE_DTYPE_BF16 ? check_launches<bf16_t>(backward, grouped, E, M, K, N, dx, dw)
                                 : check_launches<float>(backward, grouped, E, M, K, N, dx, dw);
}

struct LinearWs {
  size_t offs, prefixes, w_tab, dw_tab, dz, part, splitk, splitk_bytes, total;
};
int64_t dz_chunks(int64_t M, int E, bool grouped) {
  return (M + kDzRows - 1) / kDzRows + (grouped ? E : 0);
}
LinearWs linear_ws(int dtype, int64_t M, int K, int N, int E, bool grouped, int act, bool backward) {
  LinearWs w{};
  Carve c;
  const size_t b = elt_size(dtype);
  if (grouped) {
    w.offs = c.take((size_t)(E + 1) * 4);
    w.prefixes = c.take((size_t)kNumTilePrefixes * (E + 1) * 4);
    w.w_tab = c.take((size_t)E * sizeof(void*));
    w.dw_tab = c.take((size_t)E * sizeof(void*));
  }
  if (backward) {
    if (act != kActNone) w.dz = c.take((size_t)M * N * b);
    w.part = c.take((size_t)dz_chunks(M, E, grouped) * N * 4);
    if (!grouped) {
      const SplitPlan sp = dtype == MOE_DTYPE_BF16 ? plan_bwd<bf16_t>(false, 1, M, K, N).split
                                                   : plan_bwd<float>(false, 1, M, K, N).split;
      w.splitk_bytes = sp.nsplit > 1 ? (size_t)sp.nsplit * N * K * 4 : 0;
      w.splitk = c.take(w.splitk_bytes);
    }
  }
  w.total = c.off;
  return w;
}

// Blocks of k_linear_prep: one for the prefixes, the others for the rows of no expert.
constexpr int kPrepBlocks = 1 + 128;

template <typename D>
moe_status linear_forward(hipStream_t s, int64_t M, int K, int N, int E, const int* offsets,
                          const D* x, const D* w, const LinearEpi<D>& epi, char* ws) {
  const bool grouped = offsets != nullptr;
  if (linear_skinny<D>(M, K, N, E, grouped)) {
    const int64_t nslot = skinny_slots(M, E, grouped);
    auto go = [&](auto nc, auto ks) {
      constexpr int KS = decltype(ks)::value;
      const unsigned grid = (unsigned)skinny_blocks(M, N, E, grouped, KS);
      hipLaunchKernelGGL((k_linear_skinny<D, decltype(nc)::value, KS>), dim3(grid), dim3(256), 0,
                         s, x, offsets, E, (int)M, (int)nslot, w, K, epi);
    };
    auto split = [&](auto nc) {
      if (skinny_split<D>(K) == 4) go(nc, std::integral_constant<int, 4>());
      else go(nc, std::integral_constant<int, 2>());
    };
    if (M <= 16) split(std::integral_constant<int, 1>());
    else split(std::integral_constant<int, 4>());
    LAUNCH_CHECK();
    return MOE_OK;
  }
  const LinearWs L = linear_ws(sizeof(D) == 2 ? MOE_DTYPE_BF16 : MOE_DTYPE_F32, M, K, N, E, grouped,
                               epi.act, false);
  int* offs = grouped ? (int*)(ws + L.offs) : nullptr;
  int* prefixes = grouped ? (int*)(ws + L.prefixes) : nullptr;
  const D** w_tab = grouped ? (const D**)(ws + L.w_tab) : nullptr;
  if (grouped)
    hipLaunchKernelGGL(k_linear_prep<D>, dim3(kPrepBlocks), dim3(1024), 0, s, offsets, E, (int)M,
                       offs, prefixes, w, (D*)nullptr, (int64_t)N * K, w_tab, (D**)nullptr, epi.res,
                       epi.y, epi.pre, N);
  with_row_tiles<D>(pick_tiles<D>(grouped, E, M, N), offs, prefixes, E, M, N,
                    [&](auto c, const RowGroups& r, int grid) {
    using C = decltype(c);
    hipLaunchKernelGGL((k_linear_fwd<D, C>), dim3(grid), dim3(C::THREADS), 0, s, x, r,
                       (const D* const*)w_tab, w, K, epi);
  });
  LAUNCH_CHECK();
  return MOE_OK;
}

template <typename D>
moe_status linear_backward(hipStream_t s, int64_t M, int K, int N, int E, const int* offsets,
                           const D* dy, const D* x, const D* w, const D* pre, int act, D* dx, D* dw,
                           D* db, char* ws) {
  const bool grouped = offsets != nullptr;
  const LinearWs L = linear_ws(sizeof(D) == 2 ? MOE_DTYPE_BF16 : MOE_DTYPE_F32, M, K, N, E, grouped,
                               act, true);
  int* offs = grouped ? (int*)(ws + L.offs) : nullptr;
  int* prefixes = grouped ? (int*)(ws + L.prefixes) : nullptr;
  const D** w_tab = grouped ? (const D**)(ws + L.w_tab) : nullptr;
  D** dw_tab = grouped ? (D**)(ws + L.dw_tab) : nullptr;
  if (grouped)
    hipLaunchKernelGGL(k_linear_prep<D>, dim3(kPrepBlocks), dim3(1024), 0, s, offsets, E,
                       (int)M, offs, prefixes, w, dw, (int64_t)N * K, w_tab, dw_tab,
                       (const D*)nullptr, dx, (D*)nullptr, K);
  const RowGroups chunks{offs, prefixes, nullptr, nullptr, E, (int)M, 0, 0};
  static_assert(prefix_slot(kDzRows) == 0, "the chunks' prefix is the first");
  const D* dz = dy;
  if (act != kActNone || db) {
    D* out = (D*)(ws + L.dz);
    float* part = db ? (float*)(ws + L.part) : nullptr;
    hipLaunchKernelGGL(k_linear_dz<D>, dim3((unsigned)dz_chunks(M, E, grouped), ceil_div(N, kDzCols)),
                       dim3(256), 0, s, dy, pre, act, chunks, N, out, part);
    if (act != kActNone) dz = out;
    if (db)
      hipLaunchKernelGGL(k_linear_db<D>, dim3(ceil_div(N, 64), E), dim3(256), 0, s, part, chunks, N,
                         db);
  }
  LAUNCH_CHECK();
  using CW = WgradTiling<D, 1>;
  const BwdPlan bp = plan_bwd<D>(grouped, E, M, K, N);
  const SplitPlan& sp = bp.split;
  const KGroups kg{offs, E, (int)M, sp.nsplit, sp.kchunk, 1, nullptr};
  const int wgrid = wgrad_blocks<D>(bp, grouped, E, K, N);
  float* partial = (float*)(ws + L.splitk);
  auto wgrad = [&](auto g) {
    hipLaunchKernelGGL((k_wgrad<D, 1, decltype(g)::value>), dim3(wgrid), dim3(CW::THREADS), 0, s, dz,
                       (const D*)nullptr, (int64_t)N, x, (int64_t)K, kg, N, K, 1.0f,
                       (D* const*)dw_tab, dw, (D* const*)nullptr, (D*)nullptr, partial, wgrid, 0);
  };
  bool done = false;  // the weight gradient rides with the input gradient
  if (dx)
    with_row_tiles<D>(bp.tiles, offs, prefixes, E, M, K, [&](auto c, const RowGroups& r, int grid) {
      using C = decltype(c);
      if constexpr (C::THREADS == CW::THREADS && sizeof(D) == 2) {
        if (dw && bp.fused) {
          auto both = [&](auto g) {
            hipLaunchKernelGGL((k_linear_bwd<D, C, decltype(g)::value>), dim3(wgrid + grid),
                               dim3(C::THREADS), 0, s, dz, x, r, (const D* const*)w_tab, w, N, K,
                               dx, kg, wgrid, (D* const*)dw_tab, dw, partial);
          };
          if (grouped) both(std::true_type());
          else both(std::false_type());
          done = true;
          return;
        }
      }
      hipLaunchKernelGGL((k_linear_dgrad<D, C>), dim3(grid), dim3(C::THREADS), 0, s, dz, r,
                         (const D* const*)w_tab, w, N, K, dx);
    });
  if (dw && !done) {
    if (grouped) wgrad(std::true_type());
    else wgrad(std::false_type());
  }
  if (dw && sp.nsplit > 1)
    hipLaunchKernelGGL(k_splitk_reduce<D>, dim3(ceil_div((int64_t)N * K, 2048), 1), dim3(256), 0, s,
                       partial, sp.nsplit, (int64_t)N * K, 1.0f, dw, (D*)nullptr);
  LAUNCH_CHECK();
  return MOE_OK;
}

}  // namespace

extern "C" {

size_t moe_sort_workspace_bytes(int64_t T, int32_t k, int32_t E) {
  return check_sort(T, k, E) == MOE_OK ? sort_plan(T, k, E).bytes : 0;
}

moe_status moe_sort_tokens(int32_t device, void* stream, int64_t T, int32_t k, int32_t E,
                           int32_t index_bytes, const void* topk_idx, int32_t* counts,
                           int32_t* offsets, int32_t* perm, int32_t* inv_perm, void* workspace) {
  moe_status st = check_sort(T, k, E);
  if (st != MOE_OK) return st;
  if (index_bytes != 4 && index_bytes != 8)
    return fail(MOE_ERR_INVALID, "index_bytes %d is neither 4 nor 8", index_bytes);
  if ((st = check_ints({counts, offsets})) != MOE_OK) return st;
  const SortPlan p = sort_plan(T, k, E);
  if (T > 0 && ((st = check_ints({perm, inv_perm})) != MOE_OK ||
                (st = check_ints({topk_idx}, index_bytes)) != MOE_OK))
    return st;
  if (p.bytes && (st = check_pointers({workspace})) != MOE_OK) return st;
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  hipStream_t s = (hipStream_t)stream;
  if (index_bytes == 4)
    return launch_sort<int32_t>(s, p, E, (const int32_t*)topk_idx, counts, offsets, perm, inv_perm,
                                (int*)workspace);
  return launch_sort<int64_t>(s, p, E, (const int64_t*)topk_idx, counts, offsets, perm, inv_perm,
                              (int*)workspace);
}

moe_status moe_permute(int32_t device, void* stream, int32_t dtype, int64_t T, int32_t k,
                       int32_t H, const int32_t* inv_perm, const int32_t* num_kept, const void* x,
                       void* x_perm) {
  moe_status st = check_rows(dtype, T, k, H);
  if (st != MOE_OK || T == 0) return st;
  if ((st = check_pointers({x, x_perm})) != MOE_OK) return st;
  if ((st = check_ints({inv_perm, num_kept})) != MOE_OK) return st;
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  if (dtype == MOE_DTYPE_BF16)
    return launch_permute<bf16_t>((hipStream_t)stream, T, k, H, inv_perm, num_kept,
                                  (const bf16_t*)x, (bf16_t*)x_perm);
  return launch_permute<float>((hipStream_t)stream, T, k, H, inv_perm, num_kept, (const float*)x,
                               (float*)x_perm);
}

moe_status moe_unpermute(int32_t device, void* stream, int32_t dtype, int64_t T, int32_t k,
                         int32_t H, const int32_t* inv_perm, const int32_t* num_kept,
                         const void* y, const float* weights, void* out) {
  moe_status st = check_rows(dtype, T, k, H);
  if (st != MOE_OK || T == 0) return st;
  if ((st = check_pointers({y, out}, {weights})) != MOE_OK) return st;
  if ((st = check_ints({inv_perm, num_kept})) != MOE_OK) return st;
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  if (dtype == MOE_DTYPE_BF16)
    return launch_unpermute<bf16_t>((hipStream_t)stream, T, k, H, inv_perm, num_kept,
                                    (const bf16_t*)y, weights, (bf16_t*)out);
  return launch_unpermute<float>((hipStream_t)stream, T, k, H, inv_perm, num_kept, (const float*)y,
                                 weights, (float*)out);
}

moe_status moe_unpermute_backward(int32_t device, void* stream, int32_t dtype, int64_t T,
                                  int32_t k, int32_t H, const int32_t* inv_perm,
                                  const int32_t* num_kept, const void* d_out, const void* y,
                                  const float* weights, void* d_y, float* d_weights) {
  moe_status st = check_rows(dtype, T, k, H);
  if (st != MOE_OK || T == 0) return st;
  if ((st = check_pointers({d_out, d_y}, {y, weights, d_weights})) != MOE_OK) return st;
  if ((st = check_ints({inv_perm, num_kept})) != MOE_OK) return st;
  if (d_weights && !y) return fail(MOE_ERR_INVALID, "d_weights needs y");
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  if (dtype == MOE_DTYPE_BF16)
    return launch_unpermute_bwd<bf16_t>((hipStream_t)stream, T, k, H, inv_perm, num_kept,
                                        (const bf16_t*)d_out, (const bf16_t*)y, weights,
                                        (bf16_t*)d_y, d_weights);
  return launch_unpermute_bwd<float>((hipStream_t)stream, T, k, H, inv_perm, num_kept,
                                     (const float*)d_out, (const float*)y, weights, (float*)d_y,
                                     d_weights);
}

size_t moe_linear_workspace_bytes(int32_t dtype, int64_t M, int32_t K, int32_t N, int32_t E,
                                  int32_t grouped, int32_t activation, int32_t backward) {
  if (check_linear(dtype, M, K, N, E, grouped != 0, activation) != MOE_OK) return 0;
  if (M > 0 && check_launches(dtype, backward != 0, grouped != 0, E, M, K, N, true, true) != MOE_OK) return 0;
  return linear_ws(dtype, M, K, N, E, grouped != 0, activation, backward != 0).total;
}

moe_status moe_linear_forward(int32_t device, void* stream, int32_t dtype, int64_t M, int32_t K,
                              int32_t N, int32_t E, const int32_t* offsets, const void* x,
                              const void* weight, const void* bias, const void* residual,
                              int32_t activation, void* y, void* pre_act, void* workspace) {
  moe_status st = check_linear(dtype, M, K, N, E, offsets != nullptr, activation);
  if (st != MOE_OK || M == 0) return st;
  if ((st = check_launches(dtype, false, offsets != nullptr, E, M, K, N, false, false)) != MOE_OK) return st;
  if ((st = check_pointers({x, weight, y}, {bias, residual, pre_act})) != MOE_OK) return st;
  if (offsets && ((st = check_ints({offsets})) != MOE_OK ||
                  (st = check_pointers({workspace})) != MOE_OK))
    return st;
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MOE_DTYPE_BF16)
    return linear_forward<bf16_t>(s, M, K, N, E, offsets, (const bf16_t*)x, (const bf16_t*)weight,
                                  {(const bf16_t*)bias, (const bf16_t*)residual, (bf16_t*)y,
                                   (bf16_t*)pre_act, activation, N},
                                  (char*)workspace);
  return linear_forward<float>(s, M, K, N, E, offsets, (const float*)x, (const float*)weight,
                               {(const float*)bias, (const float*)residual, (float*)y,
                                (float*)pre_act, activation, N},
                               (char*)workspace);
}

moe_status moe_linear_backward(int32_t device, void* stream, int32_t dtype, int64_t M, int32_t K,
                               int32_t N, int32_t E, const int32_t* offsets, const void* d_y,
                               const void* x, const void* weight, const void* pre_act,
                               int32_t activation, void* dx, void* d_weight, void* d_bias,
                               void* workspace) {
  moe_status st = check_linear(dtype, M, K, N, E, offsets != nullptr, activation);
  if (st != MOE_OK) return st;
  const int64_t b = elt_size(dtype);
  // the weight gradient's operands reach over all rows of a group; the others' over a tile's
  if (d_weight && M * std::max(K, N) * b >= kMaxExtentBytes)
    return fail(MOE_ERR_UNSUPPORTED, "num_rows x max(in, out features) reaches 2^31 bytes");
  if ((st = check_pointers({}, {dx, d_weight, d_bias, workspace})) != MOE_OK) return st;
  if (M > 0) {
    if ((st = check_launches(dtype, true, offsets != nullptr, E, M, K, N, dx, d_weight)) != MOE_OK) return st;
    if ((st = check_pointers({d_y, x, weight}, {pre_act})) != MOE_OK) return st;
    if (activation != kActNone && !pre_act)
      return fail(MOE_ERR_INVALID, "the activation's backward needs pre_act");
    if (offsets && (st = check_ints({offsets})) != MOE_OK) return st;
    if (linear_ws(dtype, M, K, N, E, offsets != nullptr, activation, true).total && !workspace)
      return fail(MOE_ERR_INVALID, "a required pointer is NULL");
  }
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  hipStream_t s = (hipStream_t)stream;
  if (M == 0) {  // sums over no row
    if ((st = zero_async(s, d_weight, (size_t)E * N * K * b)) != MOE_OK) return st;
    return zero_async(s, d_bias, (size_t)E * N * b);
  }
  if (dtype == MOE_DTYPE_BF16)
    return linear_backward<bf16_t>(s, M, K, N, E, offsets, (const bf16_t*)d_y, (const bf16_t*)x,
                                   (const bf16_t*)weight, (const bf16_t*)pre_act, activation,
                                   (bf16_t*)dx, (bf16_t*)d_weight, (bf16_t*)d_bias,
                                   (char*)workspace);
  return linear_backward<float>(s, M, K, N, E, offsets, (const float*)d_y, (const float*)x,
                                (const float*)weight, (const float*)pre_act, activation, (float*)dx,
                                (float*)d_weight, (float*)d_bias, (char*)workspace);
}

moe_status moe_residual_norm(int32_t device, void* stream, int32_t dtype, int64_t T, int32_t H,
                             const void* h, const void* y, const void* post_weight,
                             const void* gate, int32_t gate_kind, const void* next_weight,
                             float residual_scale, float eps, void* h_out, void* n_out,
                             float* rstd_post, float* rstd_next) {
  moe_status st = check_norm(dtype, T, H, gate_kind, y, post_weight, gate, next_weight,
                             residual_scale);
  if (st != MOE_OK || T == 0) return st;
  if ((st = check_pointers({h}, {y, post_weight, gate, next_weight, h_out, n_out, rstd_post,
                                 rstd_next})) != MOE_OK)
    return st;
  if ((y && !h_out) || (next_weight && !n_out))
    return fail(MOE_ERR_INVALID, "a required pointer is NULL");
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  auto go = [&](auto d) {
    using D = decltype(d);
    return launch_norm_fwd<D>((hipStream_t)stream,
                              {(const D*)h, (const D*)y, (const D*)post_weight, (const D*)gate,
                               (const D*)next_weight, gate_kind, residual_scale, eps, T, H,
                               (D*)h_out, (D*)n_out, rstd_post, rstd_next});
  };
  return dtype == MOE_DTYPE_BF16 ? go(bf16_t()) : go(float());
}

size_t moe_residual_norm_workspace_bytes(int64_t T, int32_t H) {
  if (check_norm(MOE_DTYPE_F32, T, H, kGateNone, false, false, false, true, 1.0f) != MOE_OK) return 0;
  return (size_t)norm_bwd_blocks(T, H) * 2 * H * sizeof(float);
}

moe_status moe_residual_norm_backward(int32_t device, void* stream, int32_t dtype, int64_t T,
                                      int32_t H, const void* d_h_out, const void* d_n_out,
                                      const void* h_out, const void* y, const void* post_weight,
                                      const void* gate, int32_t gate_kind, const void* next_weight,
                                      float residual_scale, const float* rstd_post,
                                      const float* rstd_next, void* d_h, void* d_y,
                                      void* d_post_weight, void* d_gate, void* d_next_weight,
                                      void* workspace) {
  return norm_backward(device, stream, dtype, T, H, true, d_h_out, d_n_out, h_out, y, post_weight, gate,
                       gate_kind, next_weight, residual_scale, rstd_post, rstd_next, d_h, d_y,
                       d_post_weight, d_gate, d_next_weight, workspace);
}

moe_status moe_residual_norm_backward_from_input(int32_t device, void* stream, int32_t dtype, int64_t T,
                                      int32_t H, const void* d_h_out, const void* d_n_out,
                                      const void* h, const void* y, const void* post_weight,
                                      const void* gate, int32_t gate_kind, const void* next_weight,
                                      float residual_scale, const float* rstd_post,
                                      const float* rstd_next, void* d_h, void* d_y,
                                      void* d_post_weight, void* d_gate, void* d_next_weight,
                                      void* workspace) {
  return norm_backward(device, stream, dtype, T, H, false, d_h_out, d_n_out, h, y, post_weight, gate,
                       gate_kind, next_weight, residual_scale, rstd_post, rstd_next, d_h, d_y,
                       d_post_weight, d_gate, d_next_weight, workspace);
}

}  // extern "C"
