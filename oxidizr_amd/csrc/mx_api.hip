// C ABI of microscaled 4-bit numbers: quantisation and back, and expert products over 4-bit weights.
// Declared in include/moe_hip.h.  The calls keep no state.
#include "entry.hpp"
#include "mx.hpp"

using namespace moe;

namespace {

// ---- quantisation
moe_status check_mx(int dtype, int64_t blocks) {
  moe_status st = check_dtype(dtype);
  if (st != MOE_OK) return st;
  if (blocks < 0) return fail(MOE_ERR_INVALID, "num_blocks is negative");
  // up to eight lanes to a block
  return blocks >= kMaxGridThreads / 8 ? fail(MOE_ERR_UNSUPPORTED, "num_blocks reaches 2^29: split the tensor") : MOE_OK;
}

// ---- products
constexpr int kMxMaxWidth = 1 << 20;
constexpr int kMxNoGroupBlocks = 64;  // of a launch, for the rows of no group
moe_status check_mx_linear(int x_format, int dtype, int64_t M, int K, int N, int E, bool grouped, int act) {
  moe_status st = check_dtype(dtype);
  if (st != MOE_OK) return st;
  if (x_format != MOE_MX_ROWS_BF16 && x_format != MOE_MX_ROWS_FOUR_BIT)
    return fail(MOE_ERR_INVALID, "unknown row format %d", x_format);
  if (x_format == MOE_MX_ROWS_BF16 && dtype != MOE_DTYPE_BF16)
    return fail(MOE_ERR_INVALID, "bf16 rows have bf16 results");
  if (M < 0) return fail(MOE_ERR_INVALID, "num_rows is negative");
  if (K < kMxBlock || K % kMxBlock != 0)
    return fail(MOE_ERR_INVALID, "in_features %d is not a positive multiple of %d", K, kMxBlock);
  if (N < 8 || N % 8 != 0) return fail(MOE_ERR_INVALID, "out_features %d is not a positive multiple of 8", N);
  if (grouped ? (E < 1 || E > 1024) : E != 1)
    return fail(MOE_ERR_INVALID, grouped ? "num_groups %d is outside 1..1024"
                                         : "num_groups %d without offsets is not 1", E);
  if (act < 0 || act >= kNumActs) return fail(MOE_ERR_INVALID, "unknown activation %d", act);
  if (K > kMxMaxWidth || N > kMxMaxWidth)
    return fail(MOE_ERR_UNSUPPORTED, "in_features %d or out_features %d is above %d", K, N, kMxMaxWidth);
  if ((int64_t)K * N >= int64_t(1) << 30)
    return fail(MOE_ERR_UNSUPPORTED, "a weight matrix reaches 2^30 elements");
  if (M > (int64_t(1) << 26) || M * std::max(K, N) * elt_size(dtype) >= kMaxExtentBytes * 8)
    return fail(MOE_ERR_UNSUPPORTED, "num_rows x max(in, out features) reaches 2^34 bytes");
  return MOE_OK;
}

// Shape of a few-row launch: waves that share the K of their weight rows, blocks of 16 weight rows to a wave.  More
// blocks read the token rows less often (bf16 rows are four times the weight's bytes), fewer make more workgroups, and so
// do more waves.  us at (4 waves, 1 block) / (4, 2) / (2, 4), and with both sides in 4 bits (4, 1) / (4, 2) / (2, 2): 2 rows in
// 16 experts of 1408 x 2048 4.2 / 4.8 / 9.3 and 3.8 / 4.5 / 5.4; one weight of 4096 x 4096, 16 rows 7.7 / 9.0 / 19.0 and 5.0 / 6.4
// / 9.0, 32 rows 12.1 / 9.2 / 19.0 and 6.8 / 6.5 / 9.0, 64 rows 21 / 14 / 19 and 10.7 / 9.2 / 9.0; 128 rows in 16 experts 14.1 / 11.5 /
// 13.3 and 8.7 / 8.2 / 9.3, 256 20 / 16 / 14 and 10.9 / 10.2 / 10.1; 512 in 128 of 1536 x 4096 125 / 95 / 85 and 82 / 70 / 70.
struct MxSkinny {
  int ks, rw;
};
int64_t mx_skinny_slots(int64_t M, int E, bool grouped) {
  return grouped ? std::min<int64_t>(E, M) + M / kMxSkinnyRows : ceil_div(M, kMxSkinnyRows);
}
MxSkinny mx_skinny_shape(bool four, int64_t M, int N, int E, bool grouped) {
  const int64_t blocks = mx_skinny_slots(M, E, grouped) * ceil_div(N, 16);
  if (blocks < 512) return {4, 1};
  if (blocks < 2500) return {4, 2};
  return {2, four ? 2 : 4};
}
// Calls f(waves, blocks), constants.
template <bool X4, class F>
void with_mx_skinny(const MxSkinny& p, F&& f) {
  using std::integral_constant;
  if (p.ks == 2) f(integral_constant<int, 2>(), integral_constant<int, X4 ? 2 : 4>());
  else if (p.rw == 2) f(integral_constant<int, 4>(), integral_constant<int, 2>());
  else f(integral_constant<int, 4>(), integral_constant<int, 1>());
}
int64_t mx_skinny_blocks(const MxSkinny& p, int64_t M, int N, int E, bool grouped) {
  return mx_skinny_slots(M, E, grouped) * ceil_div(N, 64 / p.ks * p.rw) + (grouped ? kMxNoGroupBlocks : 0);
}
// Whether a forward runs as the stream of its weights.  us, tiles / this: bf16 rows, 512, 1024 and 2048 in 128 experts of 1536 x
// 4096 159 / 85, 167 / 104, 175 / 136; 128, 256 and 512 in 16 of 1408 x 2048 19 / 12, 19 / 14, 19 / 22; 64, 128 and 256 of one weight
// of 4096 x 4096 32 / 14, 32 / 25, 32 / 34.  Both sides in 4 bits: 85 / 70, 87 / 80, 89 / 108; 9.4 / 8.2, 9.3 / 10.1, 9.6 / 16;
// 13 / 9.2, 13 / 15, 14 / 26.
bool mx_skinny(bool four, int64_t M, int K, int N, int E, bool grouped) {
  // the tiles' scales are loaded 16 bytes at once
  if (four && std::min(M, (int64_t)E * N) * (K / kMxBlock) < 16) return true;
  if (mx_skinny_blocks(mx_skinny_shape(four, M, N, E, grouped), M, N, E, grouped) * 256 >= kMaxGridThreads) return false;
  return grouped ? M <= (four ? 9 : 20) * std::min<int64_t>(E, M) : M <= (four ? 80 : 160);
}

// Row tiles by height, by their cost in tenths of a full round of 256-row tiles; the tiles behind the last full round are cut
// (mx_slot).  us, 256 / 128 / 64 rows, over bf16 rows: 16384 rows in 16 experts, 2048 -> 1408 102 / 112 / 146; 65536 in 128, 4096 ->
// 1536 840 / 1028 / 1344; 12000 in 12, 1376 -> 1368 70 / 74 / 81 (uncut 82); 8192 in 64, 2048 -> 1408 85 / 86 / 88; 2048 in 16 32 / 27 /
// 26 (44); 1999 of one weight, 2784 -> 2056 45 / 48 / 56 (57); 512 of 4096 -> 4096 50 / 45 / 35 (80); 1024 60 / 50 / 52 (81); their input
// gradients 115 / 133 / 181 (120), 893 / 1107 / 1561, 66 / 75 / 98 (78), 92 / 83 / 107, 38 / 29 / 40, 42 / 38 / 59 (53), 65 / 54 / 43
// (96), 66 / 54 / 59 (96).  Both sides in 4 bits 44 / 45 / 62, 343 / 402 / 571, 46 / 48 / 44 (51), 40 / 40 / 43, 16 / 14 / 13 (20), 22 / 21 / 25 (26), 18 / 17 / 18 (29), 20 / 22 /
// 21 (31).  (Those are of the loop as it stands, which waits for all its loads in each k-tile: mainloop_mxmx.)
// An input gradient takes tiles at any number of rows: 512 rows in 128 experts of 1536 x 4096 195 us, where the stream of few
// rows gives the forward in 88; 64 rows there 87 and 39, 256 rows in 256 experts of 768 x 2048 69 and 32.
enum class MxTiles { kBig, kMid, kSmall };
MxTiles mx_tiles(bool four, bool grouped, int E, int64_t M, int N) {
  const int groups = grouped ? (int)std::min<int64_t>(E, M) : 1;
  auto count = [&](int bm, int bn) {
    return (grouped ? group_row_tiles(groups, (double)M / groups, bm) : (double)ceil_div(M, bm)) * ceil_div(N, bn);
  };
  const double tiles = count(256, 256), full = std::floor(tiles / 256.0), rest = tiles - 256.0 * full;
  const double big = 10.0 * full + (rest <= 0.0 ? 0.0 : rest <= 64.0 ? (four ? 4.6 : 5.6) : rest <= 128.0 ? 7.2 : 10.0);
  const double mid = round_cost(count(128, 128), four ? TileCost{5.0, 5.9} : TileCost{4.2, 7.0});
  const double small = round_cost(count(64, 128), four ? TileCost{4.2, 4.6} : TileCost{3.0, 4.9});
  return big <= std::min(mid, small) ? MxTiles::kBig : mid <= small ? MxTiles::kMid : MxTiles::kSmall;
}
template <class F>
void with_mx_tiling(MxTiles kind, F&& f) {
  if (kind == MxTiles::kMid) return f(Tilings<bf16_t>::BigMid{});
  if (kind == MxTiles::kSmall) return f(Tilings<bf16_t>::BigSmall{});
  f(Tilings<bf16_t>::Big{});
}
// Blocks of tiles, and behind them (grouped) those for the rows of no group.
template <class C>
int64_t mx_tile_blocks(bool grouped, int E, int64_t M, int N) {
  const int64_t xcd = ((int64_t)(ceil_div(M, C::BM) + (grouped ? E : 0)) * ceil_div(N, C::BN) + 7) / 8;  // tiles of one, at most
  return 8 * (C::BM == 256 ? xcd / 32 * 32 + 32 : xcd);  // mx_slot: parts behind the last full 32
}
moe_status check_mx_tiles(MxTiles kind, bool grouped, int E, int64_t M, int N) {
  moe_status st = MOE_OK;
  with_mx_tiling(kind, [&](auto c) {
    using C = decltype(c);
    st = check_grid(mx_tile_blocks<C>(grouped, E, M, N) + kMxNoGroupBlocks, C::THREADS);
  });
  return st;
}
moe_status check_mx_launches(bool backward, bool four, bool grouped, int E, int64_t M, int K, int N) {
  if (backward) return check_mx_tiles(mx_tiles(false, grouped, E, M, K), grouped, E, M, K);
  return mx_skinny(four, M, K, N, E, grouped) ? MOE_OK : check_mx_tiles(mx_tiles(four, grouped, E, M, N), grouped, E, M, N);
}
// Calls f(tiling, blocks of tiles, grid).
template <class F>
void with_mx_launch(MxTiles kind, const MxRows& r, int N, F&& f) {
  with_mx_tiling(kind, [&](auto c) {
    const bool grouped = r.offsets != nullptr;
    const int tiles = (int)mx_tile_blocks<decltype(c)>(grouped, r.G, r.M, N);
    f(c, tiles, dim3(tiles + (grouped ? kMxNoGroupBlocks : 0)));
  });
}

// Scratch of a backward: dz, and the chunks' sums of it.
struct MxWs {
  size_t dz, part, total;
};
int64_t mx_dz_chunks(int64_t M, int E, bool grouped) { return (M + kDzRows - 1) / kDzRows + (grouped ? E : 0); }
MxWs mx_ws(int64_t M, int N, int E, bool grouped, int act) {
  MxWs w{};
  Carve c;
  if (act != kActNone) w.dz = c.take((size_t)M * N * 2);
  w.part = c.take((size_t)mx_dz_chunks(M, E, grouped) * N * 4);
  w.total = c.off;
  return w;
}

template <bool X4, typename T>
moe_status mx_forward(hipStream_t s, int64_t M, int E, const int* offsets, const void* x, const uint8_t* xs,
                      const MxWeights& w, const LinearEpi<T>& epi) {
  const bool grouped = offsets != nullptr;
  const int N = w.N, K = w.K;
  if (mx_skinny(X4, M, K, N, E, grouped)) {
    const MxSkinny p = mx_skinny_shape(X4, M, N, E, grouped);
    const int nslot = (int)mx_skinny_slots(M, E, grouped);
    const dim3 grid((unsigned)mx_skinny_blocks(p, M, N, E, grouped));
    with_mx_skinny<X4>(p, [&](auto ks, auto rw) {
      hipLaunchKernelGGL((k_mx_skinny<X4, T, decltype(ks)::value, decltype(rw)::value>), grid, dim3(256), 0, s, x, xs,
                         offsets, E, (int)M, nslot, w, epi);
    });
    LAUNCH_CHECK();
    return MOE_OK;
  }
  const MxRows r{offsets, E, (int)M};
  with_mx_launch(mx_tiles(X4, grouped, E, M, N), r, N, [&](auto c, int tiles, dim3 grid) {
    using C = decltype(c);
    if constexpr (X4)
      hipLaunchKernelGGL((k_mxmx_fwd<C, T>), grid, dim3(C::THREADS), 0, s, (const uint8_t*)x, xs, r, tiles, w, epi);
    else
      hipLaunchKernelGGL((k_mx_fwd<C>), grid, dim3(C::THREADS), 0, s, (const bf16_t*)x, r, tiles, w, epi);
  });
  LAUNCH_CHECK();
  return MOE_OK;
}

moe_status mx_backward(hipStream_t s, int64_t M, int E, const int* offsets, const bf16_t* dy, const MxWeights& w,
                       const bf16_t* pre, int act, bf16_t* dx, bf16_t* db, char* ws) {
  const bool grouped = offsets != nullptr;
  const int N = w.N, K = w.K;
  const MxWs L = mx_ws(M, N, E, grouped, act);
  const MxRows r{offsets, E, (int)M};
  const bf16_t* dz = dy;
  if (act != kActNone || db) {
    bf16_t* out = (bf16_t*)(ws + L.dz);
    float* part = db ? (float*)(ws + L.part) : nullptr;
    const int chunks = (int)mx_dz_chunks(M, E, grouped);
    hipLaunchKernelGGL(k_mx_dz, dim3(chunks, ceil_div(N, kDzCols)), dim3(256), 0, s, dy, pre, act, r, N, out, part);
    if (act != kActNone) dz = out;
    if (db) hipLaunchKernelGGL(k_mx_db, dim3(ceil_div(N, 64), E), dim3(256), 0, s, part, r, chunks, N, db);
  }
  if (dx)
    with_mx_launch(mx_tiles(false, grouped, E, M, K), r, K, [&](auto c, int tiles, dim3 grid) {
      using C = decltype(c);
      hipLaunchKernelGGL((k_mx_dgrad<C>), grid, dim3(C::THREADS), 0, s, dz, r, tiles, w, dx);
    });
  LAUNCH_CHECK();
  return MOE_OK;
}

}  // namespace

extern "C" {

moe_status moe_mx_quantize(int32_t device, void* stream, int32_t dtype, int64_t num_blocks, const void* x,
                           uint8_t* codes, uint8_t* scales) {
  moe_status st = check_mx(dtype, num_blocks);
  if (st != MOE_OK || num_blocks == 0) return st;
  if ((st = check_pointers({x, codes})) != MOE_OK || (st = check_ints({scales}, 1)) != MOE_OK) return st;
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  const int64_t nvec = num_blocks * 4;
  const dim3 grid((unsigned)((nvec + 255) / 256));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MOE_DTYPE_BF16)
    hipLaunchKernelGGL(k_mx_quantize<bf16_t>, grid, dim3(256), 0, s, (const bf16_t*)x, nvec, (uint32_t*)codes, scales);
  else
    hipLaunchKernelGGL(k_mx_quantize<float>, grid, dim3(256), 0, s, (const float*)x, nvec, (uint32_t*)codes, scales);
  LAUNCH_CHECK();
  return MOE_OK;
}

moe_status moe_mx_dequantize(int32_t device, void* stream, int32_t dtype, int64_t num_blocks, const uint8_t* codes,
                             const uint8_t* scales, void* y) {
  moe_status st = check_mx(dtype, num_blocks);
  if (st != MOE_OK || num_blocks == 0) return st;
  if ((st = check_pointers({codes, y})) != MOE_OK || (st = check_ints({scales}, 1)) != MOE_OK) return st;
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  const int64_t nvec = num_blocks * (dtype == MOE_DTYPE_BF16 ? 4 : 8);  // 16 bytes each
  const dim3 grid((unsigned)((nvec + 255) / 256));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == MOE_DTYPE_BF16)
    hipLaunchKernelGGL(k_mx_dequantize<bf16_t>, grid, dim3(256), 0, s, (const uint32_t*)codes, scales, nvec, (bf16_t*)y);
  else
    hipLaunchKernelGGL(k_mx_dequantize<float>, grid, dim3(256), 0, s, (const uint32_t*)codes, scales, nvec, (float*)y);
  LAUNCH_CHECK();
  return MOE_OK;
}

size_t moe_mx_linear_workspace_bytes(int64_t M, int32_t K, int32_t N, int32_t E, int32_t grouped, int32_t activation) {
  if (check_mx_linear(MOE_MX_ROWS_BF16, MOE_DTYPE_BF16, M, K, N, E, grouped != 0, activation) != MOE_OK) return 0;
  if (M > 0 && check_mx_launches(true, false, grouped != 0, E, M, K, N) != MOE_OK) return 0;
  return mx_ws(M, N, E, grouped != 0, activation).total;
}

moe_status moe_mx_linear_forward(int32_t device, void* stream, int32_t x_format, int32_t dtype, int64_t M, int32_t K,
                                 int32_t N, int32_t E, const int32_t* offsets, const void* x, const uint8_t* x_scales,
                                 const uint8_t* w_codes, const uint8_t* w_scales, const void* bias,
                                 const void* residual, int32_t activation, void* y, void* pre_act) {
  moe_status st = check_mx_linear(x_format, dtype, M, K, N, E, offsets != nullptr, activation);
  if (st != MOE_OK || M == 0) return st;
  if ((st = check_mx_launches(false, x_format == MOE_MX_ROWS_FOUR_BIT, offsets != nullptr, E, M, K, N)) != MOE_OK) return st;
  if ((st = check_pointers({x, w_codes, y}, {bias, residual, pre_act})) != MOE_OK) return st;
  if ((st = check_ints({w_scales}, 1)) != MOE_OK) return st;
  const bool four = x_format == MOE_MX_ROWS_FOUR_BIT;
  if (four && (st = check_ints({x_scales}, 1)) != MOE_OK) return st;
  if (offsets && (st = check_ints({offsets})) != MOE_OK) return st;
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  hipStream_t s = (hipStream_t)stream;
  const MxWeights w{w_codes, w_scales, N, K};
  auto go = [&](auto x4, auto d) {
    using D = decltype(d);
    return mx_forward<decltype(x4)::value, D>(s, M, E, offsets, x, x_scales, w,
                                              LinearEpi<D>{(const D*)bias, (const D*)residual, (D*)y, (D*)pre_act,
                                                           activation, N});
  };
  if (!four) return go(std::false_type(), bf16_t());
  return dtype == MOE_DTYPE_BF16 ? go(std::true_type(), bf16_t()) : go(std::true_type(), float());
}

moe_status moe_mx_linear_backward(int32_t device, void* stream, int64_t M, int32_t K, int32_t N, int32_t E,
                                  const int32_t* offsets, const void* d_y, const uint8_t* w_codes,
                                  const uint8_t* w_scales, const void* pre_act, int32_t activation, void* dx,
                                  void* d_bias, void* workspace) {
  moe_status st = check_mx_linear(MOE_MX_ROWS_BF16, MOE_DTYPE_BF16, M, K, N, E, offsets != nullptr, activation);
  if (st != MOE_OK) return st;
  if ((st = check_pointers({}, {dx, d_bias, workspace})) != MOE_OK) return st;
  if (M > 0) {
    if ((st = check_mx_launches(true, false, offsets != nullptr, E, M, K, N)) != MOE_OK) return st;
    if ((st = check_pointers({d_y, w_codes}, {pre_act})) != MOE_OK) return st;
    if ((st = check_ints({w_scales}, 1)) != MOE_OK) return st;
    if (activation != kActNone && !pre_act)
      return fail(MOE_ERR_INVALID, "the activation's backward needs pre_act");
    if (offsets && (st = check_ints({offsets})) != MOE_OK) return st;
    if (!workspace) return fail(MOE_ERR_INVALID, "a required pointer is NULL");
  }
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  hipStream_t s = (hipStream_t)stream;
  if (M == 0) return zero_async(s, d_bias, (size_t)E * N * 2);  // sums over no row
  return mx_backward(s, M, E, offsets, (const bf16_t*)d_y, {w_codes, w_scales, N, K}, (const bf16_t*)pre_act,
                     activation, (bf16_t*)dx, (bf16_t*)d_bias, (char*)workspace);
}

}  // extern "C"
