// HIP kernels of expert_linear (gfx950 / CDNA4): a matrix product with bias,
// activation and residual in its epilogue, over rows sorted by expert or with one
// weight for all rows.
//   z[r] = x[r] W_e^T + b_e,  y[r] = act(z[r]) + res[r]   for r in expert e's rows,
//   dz = dy act'(z),  dx = dz W_e,  dW_e = dz^T x,  db_e = sum_r dz[r],  dres = dy.
// W_e is [N, K] row-major (out, in).  Rows of no expert (before the first one's or
// behind the last one's) have y = res (or 0), dx = 0 and no part in dW and db.  The GEMM main loop is gemm.hpp's.
#pragma once
#include "kernels.hpp"

namespace moe {

enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4, kNumActs = 5 };

// Activations and their derivatives in fp32.  gelu: z Phi(z) with the error
// function; gelu_tanh: 0.5 z (1 + tanh(c (z + 0.044715 z^3))), written with the
// logistic function: 0.5 (1 + tanh(v)) = 1 / (1 + exp(-2 v)).  For float tensors by the device
// library's expf, erfcf and a division; for bf16 ones, whose results keep 8 bits, by v_exp_f32,
// v_rcp_f32 and a polynomial, within 2^-16 of the value.
constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
// 1 / (1 + exp(-z)); bf16 with v_rcp_f32 (one step) instead of a division (ten instructions):
// an epilogue runs it 128 times a lane, alone (8192 x 2048 outputs, K = 2816) 9 us of 88.
MOE_DEV float logistic(float z, bf16_t) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }
MOE_DEV float logistic(float z, float) { return 1.0f / (1.0f + expf(-z)); }
// Phi(z) and exp(-z^2 / 2).  No tail is formed as 1 - erf, which cancels: a value is off by a few
// fp32 steps of itself, and by z^2 more for the rounding of the exponent's argument.
MOE_DEV float normal_cdf(float z, float& e, float) {
  e = expf(-0.5f * z * z);
  return 0.5f * erfcf(-0.7071067811865476f * z);
}
// Phi(-|z|) exp(z^2 / 2) = t P(t), t = 1 / (1 + p |z|): p and P by linear programming for the
// smallest largest relative error over |z| <= 14, 6.5e-7 (9e-7 in fp32 arithmetic); below -14 Phi is
// under 2^-146.  With erff the slope of 500 x 2816 outputs took 18.8 us.
MOE_DEV float normal_cdf(float z, float& e, bf16_t) {
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.265f * fabsf(z));
  e = __expf(-0.5f * z * z);
  const float q = e * t *
                  (0.105599158f +
                   t * (0.107845433f +
                        t * (0.0829029307f +
                             t * (0.142605081f +
                                  t * (-0.066516608f + t * (0.195381135f + t * -0.0678174347f))))));
  return z < 0.0f ? q : 1.0f - q;
}
template <typename T>
MOE_DEV float act_value(float z, int act) {
  switch (act) {
    case kActRelu: return z <= 0.0f ? 0.0f : z;  // a NaN stays one
    case kActSilu: return z * logistic(z, T());
    case kActGelu: {
      float e;
      return z * normal_cdf(z, e, T());
    }
    case kActGeluTanh: return z * logistic(2.0f * kGeluC * (z + 0.044715f * z * z * z), T());
    default: return z;
  }
}
template <typename T>
MOE_DEV float act_slope(float z, int act) {
  switch (act) {
    case kActRelu: return z <= 0.0f ? 0.0f : 1.0f;
    case kActSilu: {
      const float s = logistic(z, T());
      return s * (1.0f + z * (1.0f - s));
    }
    case kActGelu: {
      float e;
      const float cdf = normal_cdf(z, e, T());
      return cdf + z * 0.3989422804014327f * e;
    }
    case kActGeluTanh: {
      const float s = logistic(2.0f * kGeluC * (z + 0.044715f * z * z * z), T());
      // s (1 - s) is 0 from |z| = 10 on: squares beyond 1e6 would only make 0 inf a NaN
      const float zz = fminf(z * z, 1e6f);
      return s + s * (1.0f - s) * z * (2.0f * kGeluC * (1.0f + 3.0f * 0.044715f * zz));
    }
    default: return 1.0f;
  }
}

// Eight at once: one branch on the activation, which is the same for the launch.
template <typename T>
MOE_DEV void act_value8(const float (&z)[8], float (&y)[8], int act) {
  auto all = [&](auto a) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = act_value<T>(z[i], decltype(a)::value);
  };
  switch (act) {
    case kActRelu: return all(std::integral_constant<int, kActRelu>());
    case kActSilu: return all(std::integral_constant<int, kActSilu>());
    case kActGelu: return all(std::integral_constant<int, kActGelu>());
    case kActGeluTanh: return all(std::integral_constant<int, kActGeluTanh>());
    default: return all(std::integral_constant<int, kActNone>());
  }
}
// d *= act'(z)
template <typename T>
MOE_DEV void act_slope8(const float (&z)[8], float (&d)[8], int act) {
  auto all = [&](auto a) {
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] *= act_slope<T>(z[i], decltype(a)::value);
  };
  switch (act) {
    case kActRelu: return all(std::integral_constant<int, kActRelu>());
    case kActSilu: return all(std::integral_constant<int, kActSilu>());
    case kActGelu: return all(std::integral_constant<int, kActGelu>());
    default: return all(std::integral_constant<int, kActGeluTanh>());
  }
}

// What the epilogue of a forward needs.  bias: [G, N] (or [N]) or null; res, pre: row r
// at r N, or null.
template <typename T>
struct LinearEpi {
  const T *bias, *res;
  T *y, *pre;
  int act, N;
};

// Eight outputs of row r from column n on.  The pre-activation is kept in the dtype.  A bf16 z is
// off by up to 2^-8 of itself and act'(z) by up to |z act''(z)| 2^-8, which is more than dz's own
// rounding where the slope is small: silu 5 times it at z = -1, gelu 3 at -2 and 20 at -5.  A choice:
// kept in fp32 it takes twice the memory of a tensor that lives until the backward and a tenth more
// traffic, and since dz is rounded to bf16 for the products in any case, gradients over N(0, 1)
// data come to 2.42e-3 instead of 2.35e-3 (relative L2).
template <typename T, bool RES>
MOE_DEV void linear_store8(const LinearEpi<T>& e, int64_t r, int n, const float (&z)[8],
                           const float (&res)[8]) {
  const int64_t o = r * e.N + n;
  float y[8];
  if (e.pre) store8(e.pre + o, z);
  act_value8<T>(z, y, e.act);
  if constexpr (RES) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] += res[i];
  }
  store8_stream(e.y + o, y);
}

// ------------------------------------------------------------------ preparation
// Before the tiled launches of a grouped call.  Block 0: a clean copy of the offsets
// (clamped to [0, M] and made ascending, so that no offsets make a launch leave its
// buffers), the tile prefixes, and the experts' weight (and weight gradient)
// addresses.  The blocks after it: rows of no expert, which are out = res (or
// zeros), `cols` wide, and out2 = 0; and zeros for the weight gradient of an
// expert without rows.
template <typename T>
__global__ __launch_bounds__(1024) void k_linear_prep(const int* __restrict__ offsets, int E, int M,
                                                      int* __restrict__ offs_out,
                                                      int* __restrict__ prefixes,
                                                      const T* w, T* dw, int64_t stride,
                                                      const T** __restrict__ w_tab,
                                                      T** __restrict__ dw_tab,
                                                      const T* __restrict__ res,
                                                      T* __restrict__ out, T* __restrict__ out2,
                                                      int cols) {
  __shared__ int cnt[1024], offs[1024], wsum[16 * kScanCount], wmaxs[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // running maximum of the offsets clamped to [0, M]: offset e + 1 in thread e
  const int o0 = min(max(offsets[0], 0), M);
  int v = tid < E ? min(max(offsets[tid + 1], o0), M) : o0;
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(v, d, 64);
    if (lane >= d) v = max(v, u);
  }
  if (lane == 63) wmaxs[wave] = v;
  __syncthreads();
  for (int i = 0; i < wave; ++i) v = max(v, wmaxs[i]);
  offs[tid] = v;
  __syncthreads();
  const int lo = tid == 0 ? o0 : offs[tid - 1];
  if (tid < E) cnt[tid] = v - lo;
  __syncthreads();
  if (blockIdx.x > 0) {
    const int64_t first = (int64_t)(blockIdx.x - 1) * 1024 + tid;
    const int64_t step = (int64_t)(gridDim.x - 1) * 1024;
    const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    // vectors [0, head) and [tail, M cols / 8)
    const int64_t head = (int64_t)o0 * cols / 8, tail = (int64_t)offs[E - 1] * cols / 8;
    const int64_t none = head + (int64_t)M * cols / 8 - tail;
    if (out)
      for (int64_t j = first; j < none; j += step) {
        const int64_t i = j < head ? j : j - head + tail;
        float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (res) load8(res + i * 8, f);
        store8(out + i * 8, f);
        if (out2) store8(out2 + i * 8, zero);
      }
    if (dw)
      for (int e = 0; e < E; ++e)
        if (cnt[e] == 0)
          for (int64_t i = first; i < stride / 8; i += step) store8(dw + e * stride + i * 8, zero);
    return;
  }
  if (tid < E) {
    w_tab[tid] = w + tid * stride;
    if (dw) dw_tab[tid] = dw + tid * stride;
  }
  // the scan writes offsets from zero; rows before the first offset are no expert's
  scan_counts(cnt, E, offs_out, prefixes, offs, wsum);
  if (tid < E) offs_out[tid] += o0;
  if (tid == 1023) offs_out[E] += o0;  // the thread that wrote it
}

// ------------------------------------------------------------------ tiled products
// Adds bias[0..nv) (of the tile's first column on) to the accumulators where they are:
// a lane holds four consecutive columns in each quarter of a block, so it needs 16
// bytes' worth per block and no second pass; all loads are in flight together.
template <class C, typename T>
MOE_DEV void add_bias(f32x16 (&acc)[1][C::TN][C::TM], f32x16 (&xacc)[1][C::XTN], const T* bias,
                      int nv) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / C::WGN, wn = wave % C::WGN;
  const int n0 = wn * C::WN + 4 * (lane >> 5);
  // the extra blocks of a 320-row tile are the lower or the upper half of the columns
  const bool hi = C::XR == 64 && (wm >> 1) != 0;
#pragma unroll
  for (int tn = 0; tn < C::TN; ++tn) {
    float b[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = n0 + tn * 32 + 8 * q;
#pragma unroll
      for (int i = 0; i < 4; ++i) b[q][i] = 0.0f;
      if (n < nv) load4(bias + n, b[q]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int tm = 0; tm < C::TM; ++tm) acc[0][tn][tm][4 * q + i] += b[q][i];
        if constexpr (C::XR == 128) xacc[0][tn][4 * q + i] += b[q][i];
        if constexpr (C::XR == 64) {
          constexpr int half = C::XTN;
          if ((tn >= half) == hi) xacc[0][tn % half][4 * q + i] += b[q][i];
        }
      }
  }
}

// fp32 sums run over k in the order 0, 4, 8, 12, 1, 5, .. of 16-deep steps, in which a 16 x 16
// x 4 MFMA fed by 16-byte vectors takes it: that of a wave of k_linear_skinny, and, by
// their bits, of torch's fp32 products in most shapes.  relu's slope jumps at 0, so a sum
// that rounding puts on its other side has another gradient: of 7.8 million outputs (5697 x
// 1368, K = 776) about one a batch is on the other side of the exact sum, in torch as here.
// With one order they are the same ones: in 24 batches no sign differed, in 8-deep steps
// (0, 4, 1, 5, ..) one did in 8 of them.  No slower: 394 -> 388 us a training pass.
constexpr int kF32StepVectors = 2;

// y tile by tile.  Bound by the matrix cores and, one 256-row tile to a CU, by its
// epilogue, which nothing overlaps: 8192 x 2048, K = 2816 with bias and residual 85-90 us
// (1050-1110 TFLOP/s; the library's product alone 69), of which the k-loop is some 70;
// 16 experts of 1024 rows, 1408 x 2048, silu, two outputs, 128-row tiles 115-125 us.
// The residual of the whole tile is requested when the main loop has
// ended (in the fragments' registers; a 384-row tile has none left, takes it a pass ahead and
// spills 40 of its 256 registers, 84 bytes a lane).
template <typename T, class C>
__global__ __launch_bounds__(C::THREADS) void k_linear_fwd(const T* __restrict__ X, RowGroups groups,
                                                           const T* const* w_tab, const T* w_one,
                                                           int K, LinearEpi<T> epi) {
  __shared__ __align__(16) T smem[rowcol_smem_elems<T, C, 1, 1, 1>()];
  int grp, row0, mv, n0;
  const int N = epi.N;
  if (!resolve_rows(groups, N, C::AR, C::BN, grp, row0, mv, n0)) return;
  const T* w = pick(w_tab, w_one, grp);
  const T* bias = epi.bias ? epi.bias + (int64_t)grp * N + n0 : nullptr;
  with_tile_shape<T, C>(mv, N - n0, [&](auto ct) {
    using CT = decltype(ct);
    OpDesc<T> a[1] = {{X + (int64_t)row0 * K, K, mv, K}};
    OpDesc<T> b[1] = {{w + (int64_t)n0 * K, K, N - n0, K}};
    f32x16 acc[1][CT::TN][CT::TM], xacc[1][CT::XTN];
    zero_acc<CT, 1>(acc, xacc);
    constexpr int KW = sizeof(T) == 4 ? kF32StepVectors : 1;
    mainloop_x<CT, T, false, false, 1, 1, false, KW>(acc, xacc, a, b, K, smem);
    static_assert(epi_lds_floats<CT, 1>() * 4 <= (int)sizeof(smem), "epilogue LDS");
    if (bias) add_bias<CT, T>(acc, xacc, bias, N - n0);
    if (epi.res) {
      constexpr int V = Vec16<T>::N;
      struct Pre { u32x4 r[8 / V]; };
      for_each_row8_xpre<CT, 1, Pre, CT::XR == 0 && sizeof(T) == 2>(acc, xacc, reinterpret_cast<float*>(smem),
                                     [&](int m, int n, Pre& q) {
        if (m >= mv || n0 + n >= N) return;
        const T* p = epi.res + ((int64_t)row0 + m) * N + n0 + n;
#pragma unroll
        for (int i = 0; i < 8 / V; ++i) q.r[i] = *gptr(reinterpret_cast<const u32x4*>(p + i * V));
      }, [&](int m, int n, auto& v, const Pre& q) {
        if (m >= mv || n0 + n >= N) return;
        float r[8];
#pragma unroll
        for (int i = 0; i < 8 / V; ++i) unpack16(q.r[i], r + i * V, T());
        linear_store8<T, true>(epi, (int64_t)row0 + m, n0 + n, v[0], r);
      });
    } else {
      for_each_row8_x<CT, 1>(acc, xacc, reinterpret_cast<float*>(smem),
                             [&](int m, int n, auto& v) {
        if (m >= mv || n0 + n >= N) return;
        linear_store8<T, false>(epi, (int64_t)row0 + m, n0 + n, v[0], v[0]);
      });
    }
  });
}

// One tile of dx = dz W (K-major weight operand), as block blk of a launch.
template <typename T, class C>
MOE_DEV void dgrad_tile(T* smem, int blk, const T* __restrict__ dZ, const RowGroups& groups,
                        const T* const* w_tab, const T* w_one, int N, int K, T* __restrict__ dX) {
  int grp, row0, mv, k0;
  if (!resolve_rows(groups, K, C::AR, C::BN, grp, row0, mv, k0, blk)) return;
  const T* w = pick(w_tab, w_one, grp);  // element (k, n) of the operand at w + n K + k
  with_tile_shape<T, C>(mv, K - k0, [&](auto ct) {
    using CT = decltype(ct);
    OpDesc<T> a[1] = {{dZ + (int64_t)row0 * N, N, mv, N}};
    OpDesc<T> b[1] = {{w + k0, K, K - k0, N}};
    f32x16 acc[1][CT::TN][CT::TM], xacc[1][CT::XTN];
    zero_acc<CT, 1>(acc, xacc);
    mainloop_x<CT, T, false, true, 1, 1>(acc, xacc, a, b, N, smem);
    for_each_row8_x<CT, 1>(acc, xacc, reinterpret_cast<float*>(smem), [&](int m, int n, auto& v) {
      if (m >= mv || k0 + n >= K) return;
      store8_stream(dX + ((int64_t)row0 + m) * K + k0 + n, v[0]);
    });
  });
}
template <typename T, class C>
__global__ __launch_bounds__(C::THREADS) void k_linear_dgrad(const T* __restrict__ dZ,
                                                             RowGroups groups,
                                                             const T* const* w_tab, const T* w_one,
                                                             int N, int K, T* __restrict__ dX) {
  __shared__ __align__(16) T smem[rowcol_smem_elems<T, C, 1, 1, 1>()];
  dgrad_tile<T, C>(smem, (int)blockIdx.x, dZ, groups, w_tab, w_one, N, K, dX);
}

// Both products of a backward in one launch: the wblocks (a multiple of 8) weight
// gradient tiles, then the input gradient's.  One workgroup fills a CU, so a launch of
// its own ends with a partial round; here the second product's tiles start as the
// first's end, and one partial round is left: 16 experts of 1024 rows, 1408 x 2048, 248 ->
// 209 us; 8192 rows of 2816 x 2048 205 -> 161-181.
template <typename T, class C, bool GROUPED>
__global__ __launch_bounds__(C::THREADS) void k_linear_bwd(const T* __restrict__ dZ,
                                                           const T* __restrict__ X,
                                                           RowGroups groups,
                                                           const T* const* w_tab, const T* w_one,
                                                           int N, int K, T* __restrict__ dX,
                                                           KGroups kgroups, int wblocks,
                                                           T* const* dw_tab, T* dw_one,
                                                           float* __restrict__ partial) {
  using CW = WgradTiling<T, 1>;
  static_assert(C::THREADS == CW::THREADS, "one workgroup size");
  constexpr int A = rowcol_smem_elems<T, C, 1, 1, 1>(), B = kernel_smem_elems<CW, T, 1, 1, 1>();
  __shared__ __align__(16) T smem[A > B ? A : B];
  if ((int)blockIdx.x < wblocks)
    wgrad_tile<T, 1, GROUPED>(smem, (int)blockIdx.x, dZ, (const T*)nullptr, N, X, K, kgroups, N, K,
                              1.0f, dw_tab, dw_one, (T* const*)nullptr, (T*)nullptr, partial);
  else
    dgrad_tile<T, C>(smem, (int)blockIdx.x - wblocks, dZ, groups, w_tab, w_one, N, K, dX);
}

// ------------------------------------------------------------------ few rows
// A launch with few rows to an expert is the stream of the weights that it
// touches.  As in the layer's small-batch kernels a wave multiplies 16 weight rows
// with the rows of the expert (up to four chunks of 16) by 16 x 16 MFMAs straight
// from memory: lane l supplies 16-byte vector l / 16 + 4 q of weight row l % 16 and
// of token row l % 16 in step q, so four lanes read 64 contiguous bytes.  KS waves of
// a workgroup share a block of 16 weight rows and take every KS-th k-chunk of 8
// steps; their sums are added through LDS in wave order.  Bound by the weights: 128
// experts of 4096 x 1536 bf16, 512 rows (1.61 GB) 231-240 us, 6.7-7.0 TB/s.
constexpr int kLinearSkinnyRows = 64;  // rows of an expert that one workgroup takes
constexpr int kSkinnyChunkBytes = 512;  // of a weight row, in one k-chunk
// Slot s of a launch: the s-th (expert, 64 rows of it) pair with rows, experts
// ascending.  Every wave finds its own from the offsets: lane l counts the chunks of
// experts l E/64 .., a prefix sum over the lanes finds the lane that holds slot s.
// False for a slot past the last.
MOE_DEV bool skinny_slot(const int* __restrict__ offsets, int E, int M, int s, int& grp, int& r0,
                         int& rows) {
  const int lane = threadIdx.x & 63;
  const int per = (E + 63) >> 6, e0 = lane * per;
  constexpr int R = kLinearSkinnyRows;
  int n = 0;
  for (int i = 0; i < per; ++i) {
    const int e = e0 + i;
    if (e < E) {
      const int a = min(max(offsets[e], 0), M), b = min(max(offsets[e + 1], a), M);
      n += (b - a + R - 1) / R;
    }
  }
  const int incl = wave_incl_scan(n);
  const uint64_t m = __ballot(incl > s);
  if (m == 0) return false;
  const int l = __ffsll((unsigned long long)m) - 1;
  int left = s - (__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(n, l));
  // the experts of lane l, walked by every lane (uniform)
  for (int i = 0; i < per; ++i) {
    const int e = l * per + i;
    if (e >= E) break;
    const int a = uni(min(max(offsets[e], 0), M)), b = uni(min(max(offsets[e + 1], a), M));
    const int c = (b - a + R - 1) / R;
    if (left < c) {
      grp = e;
      r0 = a + left * R;
      rows = min(R, b - r0);
      return true;
    }
    left -= c;
  }
  return false;
}

// NC: chunks of 16 rows (1 for calls of at most 16 rows, else 4).  Blocks below
// nslot x nNb are (slot, row blocks) pairs; the others write the rows of no
// expert.  offsets null: one weight, rows s 64 .. .
template <typename T, int NC, int KS>
__global__ __launch_bounds__(256) void k_linear_skinny(const T* __restrict__ X,
                                                       const int* __restrict__ offsets, int E,
                                                       int M, int nslot, const T* __restrict__ W,
                                                       int K, LinearEpi<T> epi) {
  constexpr int RB = 4 / KS, V = Vec16<T>::N, KC = kSkinnyChunkBytes / sizeof(T);
  static_assert(KC == 32 * V, "eight steps of four vectors");
  __shared__ f32x4 red[(KS - 1) * RB * NC * 64];
  const int N = epi.N;
  const int nNb = (N + 16 * RB - 1) / (16 * RB);
  const int slot = uni(blockIdx.x / nNb), nb = uni(blockIdx.x % nNb);
  if (slot >= nslot) {
    int m = 0;
    for (int e = threadIdx.x & 63; e <= E; e += 64) m = max(m, offsets[e]);
    m = min(wave_max(m), M);
    const int64_t head = (int64_t)min(max(offsets[0], 0), M) * N / 8, tail = (int64_t)m * N / 8;
    const int64_t none = head + (int64_t)M * N / 8 - tail;
    const int64_t step = ((int64_t)gridDim.x - (int64_t)nslot * nNb) * 256;
    for (int64_t j = ((int64_t)blockIdx.x - (int64_t)nslot * nNb) * 256 + threadIdx.x; j < none;
         j += step) {
      const int64_t v = j < head ? j : j - head + tail;
      float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (epi.res) load8(epi.res + v * 8, f);
      store8(epi.y + v * 8, f);
      if (epi.pre) store8(epi.pre + v * 8, zero);
    }
    return;
  }
  int grp = 0, r0 = slot * kLinearSkinnyRows, rows = min(kLinearSkinnyRows, M - r0);
  if (offsets && !skinny_slot(offsets, E, M, slot, grp, r0, rows)) return;  // workgroup-uniform
  grp = uni(grp); r0 = uni(r0); rows = uni(rows);
  const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int rb = wave / KS, ks = wave % KS;
  const int n0 = (nb * RB + rb) * 16;
  const int nrows = uni(min(16, N - n0));
  const int g = lane >> 4, rl = lane & 15;
  const int nch = (rows + 15) / 16;
  f32x4 acc[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) acc[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (nrows > 0) {
    const rsrc_t rx = make_rsrc(uni_ptr(X + (int64_t)r0 * K), (uint32_t)uni(rows * K * (int)sizeof(T)));
    const rsrc_t rw = make_rsrc(uni_ptr(W + ((int64_t)grp * N + n0) * K),
                                (uint32_t)uni(nrows * K * (int)sizeof(T)));
    const uint32_t vw = (uint32_t)((rl * K + V * g) * (int)sizeof(T));
    uint32_t vx[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
      vx[c] = c * 16 + rl < rows ? (uint32_t)(((c * 16 + rl) * K + V * g) * (int)sizeof(T)) : kOobOffset;
    for (int kc = ks; kc * KC < K; kc += KS) {
      const uint32_t soff = (uint32_t)kc * kSkinnyChunkBytes;
      u32x4 wa[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const bool kin = kc * KC + 4 * V * q + V * g < K;
        wa[q] = buf_ld16(rw, kin ? vw + 64 * q : kOobOffset, soff);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (c >= nch) break;
        u32x4 xa[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const bool kin = kc * KC + 4 * V * q + V * g < K;
          xa[q] = buf_ld16(rx, kin ? vx[c] + 64 * q : kOobOffset, soff);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < 8; ++q) mfma16(acc[c], xa[q], wa[q], T());
      }
    }
  }
  if (ks > 0) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (c < nch) red[((ks - 1) * RB + rb) * NC * 64 + c * 64 + lane] = acc[c];
  }
  __syncthreads();
  if (ks > 0) return;
#pragma unroll
  for (int q = 1; q < KS; ++q)
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (c < nch) acc[c] += red[((q - 1) * RB + rb) * NC * 64 + c * 64 + lane];
  // lane holds row 16 c + 4 g + r, column n0 + rl
  if (rl >= nrows) return;
  const int n = n0 + rl;
  const float bias = epi.bias ? to_f<T>(epi.bias[(int64_t)grp * N + n]) : 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (c >= nch) break;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = c * 16 + 4 * g + r;
      if (t >= rows) continue;
      const int64_t o = ((int64_t)r0 + t) * N + n;
      const float z = acc[c][r] + bias;
      if (epi.pre) epi.pre[o] = from_f<T>(z);
      const float y = act_value<T>(z, epi.act);
      epi.y[o] = from_f<T>(epi.res ? y + to_f<T>(epi.res[o]) : y);
    }
  }
}

// ------------------------------------------------------------------ backward, element-wise part
// dz = dy act'(z) (written when act is not none) and, per 64-row chunk of a group,
// the column sums of dz for the bias gradient, from the unrounded products.  Block
// (chunk, 64 columns): thread (r, c) takes rows r and r + 32 of 8 columns, so that a
// few rows fill the CUs as well; the 32 row lanes are added in order.  Bound by its
// reads and writes (16384 x 1408 bf16, 138 MB: 26 us, 5.2 TB/s).
constexpr int kDzRows = kF32RowTile;  // rows of a chunk: the prefix of 64-row tiles counts them
constexpr int kDzCols = 64;
template <typename T>
__global__ __launch_bounds__(256) void k_linear_dz(const T* __restrict__ dY,
                                                   const T* __restrict__ pre, int act, RowGroups g,
                                                   int N, T* __restrict__ dZ,
                                                   float* __restrict__ part) {
  __shared__ float col[32][kDzCols];
  int r0, rows;
  const int chunk = blockIdx.x;
  if (g.offsets) {
    if (chunk >= g.tile_prefix[g.G]) return;
    const int grp = uni(find_group(g.tile_prefix, g.G, chunk));
    r0 = g.offsets[grp] + (chunk - g.tile_prefix[grp]) * kDzRows;
    rows = min(kDzRows, g.offsets[grp + 1] - r0);
  } else {
    r0 = chunk * kDzRows;
    rows = min(kDzRows, g.M - r0);
  }
  const int rl = threadIdx.x >> 3, c8 = (threadIdx.x & 7) * 8;
  const int n = blockIdx.y * kDzCols + c8;
  float d[2][8], z[2][8], s[8];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = rl + 32 * j;
#pragma unroll
    for (int i = 0; i < 8; ++i) d[j][i] = z[j][i] = 0.0f;
    if (n < N && r < rows) {
      load8(dY + ((int64_t)r0 + r) * N + n, d[j]);
      if (act != kActNone) load8(pre + ((int64_t)r0 + r) * N + n, z[j]);
    }
  }
  if (act != kActNone) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      act_slope8<T>(z[j], d[j], act);
      if (n < N && rl + 32 * j < rows) store8(dZ + ((int64_t)r0 + rl + 32 * j) * N + n, d[j]);
    }
  }
  if (!part) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = d[0][i] + d[1][i];
#pragma unroll
  for (int i = 0; i < 8; ++i) col[rl][c8 + i] = s[i];
  __syncthreads();
  const int cc = blockIdx.y * kDzCols + threadIdx.x;
  if (threadIdx.x >= kDzCols || cc >= N) return;
  float t = 0.0f;
#pragma unroll
  for (int r = 0; r < 32; ++r) t += col[r][threadIdx.x];
  part[(int64_t)chunk * N + cc] = t;
}

// db[g] = the sum of group g's chunks, in order (zeros for a group without rows).
// Block (group, 64 columns): four row lanes of 64 columns each.
template <typename T>
__global__ __launch_bounds__(256) void k_linear_db(const float* __restrict__ part, RowGroups g,
                                                   int N, T* __restrict__ db) {
  __shared__ float col[4][64];
  const int grp = blockIdx.y;
  const int p0 = g.offsets ? g.tile_prefix[grp] : 0;
  const int p1 = g.offsets ? g.tile_prefix[grp + 1] : (g.M + kDzRows - 1) / kDzRows;
  const int n = blockIdx.x * 64 + (threadIdx.x & 63), rl = threadIdx.x >> 6;
  float s = 0.0f;
  if (n < N) {
#pragma unroll 8
    for (int p = p0 + rl; p < p1; p += 4) s += part[(int64_t)p * N + n];
  }
  col[rl][threadIdx.x & 63] = s;
  __syncthreads();
  if (rl != 0 || n >= N) return;
  db[(int64_t)grp * N + n] =
      from_f<T>((col[0][n & 63] + col[1][n & 63]) + (col[2][n & 63] + col[3][n & 63]));
}

}  // namespace moe
