// HIP kernels of the router's losses over given logits and experts (gfx950 / CDNA4).
//
// Logits [T, E], experts [T, k].  A token is real when one of its k indices is in [0, E) (others have no
// expert: padding, or dropped).  For each sequence of tokens, with n real ones and M_e assignments to expert e:
//   x = logits / tau,  p = softmax(x),  lse = log sum exp(x),
//   q = p, or sigmoid(x) over its sum,
//   P_e = sum_t q_te / n,  f_e = M_e / (k n),
//   balance = E sum_e (c_sw f_e P_e + c_sq P_e^2),  z = sum_t lse_t^2 / n   (0 for n = 0).
// Gradient, with g_e = d_balance E (c_sw f_e + 2 c_sq P_e) / n and h = 2 d_z / n:
//   dlogits_te = (q_te c_te (g_e - sum_j q_tj g_j) + h lse_t p_te) / tau,  c = 1, or 1 - sigmoid(x_te).
// Rows of tokens that are not real, or in no sequence, have none.
//
// Each direction reads the logits once.  The forward keeps a lane's columns in registers and adds them
// up over the rows of its block; the blocks' sums are added in block order, so no result depends on
// scheduling.  Sums within a block are fp32 (some 1e-7 of a loss), those over blocks 64 bits.  Exponentials are v_exp_f32
// of a logit times log2(e) / tau, off by |x| 2^-23 of themselves for the factor's and the product's roundings and a step
// more (exact to fp32 where they matter, near the largest), quotients v_rcp_f32: with the device library's expf and
// divisions 65536 rows of 160 sigmoid scores took 45 us forward and 55 back (24 and 29 with these).
#pragma once
#include "kernels.hpp"

namespace moe {

constexpr float kLog2E = 1.4426950408889634f;

// The larger, or NaN if one of them is (fmaxf passes over it).
MOE_DEV float max_of_all(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// v of lane l ^ X, any power of two below 64.
template <int X>
MOE_DEV float group_xor(float v) {
  if constexpr (X == 32) {
    const uint32_t u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(threadIdx.x & 32 ? s[0] : s[1]);
  } else if constexpr (X == 16) {
    const uint32_t u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(threadIdx.x & 16 ? s[0] : s[1]);
  } else {
    return lane_xor<X>(v);
  }
}
// Over lanes whose numbers differ in the bits below HI and not below LO.
template <int LO, int HI, class OP>
MOE_DEV float group_reduce(float v, OP&& op) {
  if constexpr (LO < HI) {
    v = op(v, group_xor<HI / 2>(v));
    return group_reduce<LO, HI / 2>(v, op);
  }
  return v;
}
template <int N>
MOE_DEV float group_sum(float v) { return group_reduce<1, N>(v, [](float a, float b) { return a + b; }); }
template <int N>
MOE_DEV float group_max(float v) { return group_reduce<1, N>(v, max_of_all); }

enum { kScoreSoftmax = 0, kScoreSigmoid = 1 };

template <typename T, typename I>
struct RouterRows {
  const T* logits;
  const I* idx;
  const int* offsets;  // [S + 1], or null: one sequence of all rows
  int64_t Tn;
  int E, k, S, score;
  float inv_tau;
};

// How a wave holds rows: LPR lanes to a row, NCH chunks of V consecutive columns to a lane.  Few lanes with many columns
// each: sums over a row then take fewer steps and the lanes of a wave are used (160 columns: 8 lanes of 5 chunks, not 40 of 64).
template <int V_, int LPR_, int NCH_>
struct RouterShape {
  static constexpr int V = V_, LPR = LPR_, NCH = NCH_, C = V_ * NCH_;
  static constexpr int RPW = 64 / LPR;        // rows to a wave
  static constexpr int COLS = C * LPR;        // columns held, E at most
};

// A row's chunks.  bf16 ones are converted where they are loaded, in a branch each, so hipcc waits for every chunk before the
// next is requested; fp32 ones are in flight together.
template <class S, typename T>
MOE_DEV void router_load(const T* row, int E, int j, float (&x)[S::C]) {
#pragma unroll
  for (int i = 0; i < S::NCH; ++i) {
    const int c = (i * S::LPR + j) * S::V;
    if constexpr (S::V == 4) {
      float f[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (c < E) load4(row + c, f);
#pragma unroll
      for (int v = 0; v < 4; ++v) x[4 * i + v] = f[v];
    } else {
      x[i] = c < E ? to_f<T>(row[c]) : -INFINITY;
    }
  }
}

// Of a row whose logits x are spread over S::LPR lanes: q and p, normalised, the largest logit m and the log of the sum, so
// that lse = m / tau + log_sum.  The largest is taken off before the division by tau: logits of the type's lowest value
// over a tau below 1 are beyond fp32, their differences are not.  Of an infinite m, p is NaN and lse m itself.  scale: log2(e) / tau.
template <class S>
MOE_DEV void router_scores(const float (&x)[S::C], int score, float scale, float (&q)[S::C], float (&p)[S::C], float& m,
                           float& log_sum) {
  m = -INFINITY;
#pragma unroll
  for (int i = 0; i < S::C; ++i) m = max_of_all(m, x[i]);
  m = group_max<S::LPR>(m);
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < S::C; ++i) {
    p[i] = __builtin_amdgcn_exp2f((x[i] - m) * scale);
    sum += p[i];
  }
  if (score == kScoreSoftmax) {
    sum = group_sum<S::LPR>(sum);
    const float r = __builtin_amdgcn_rcpf(sum);
#pragma unroll
    for (int i = 0; i < S::C; ++i) {
      p[i] *= r;
      q[i] = p[i];
    }
  } else {
    // sigmoid(x / tau) over sigmoid's size at the row's largest, min(1, exp(m / tau)): rows of very negative logits have
    // scores as well
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < S::C; ++i) {
      const float t = __builtin_amdgcn_exp2f(-fabsf(x[i]) * scale);
      const float below = m > 0.0f ? t : p[i];
      q[i] = (x[i] > 0.0f ? 1.0f : below) * __builtin_amdgcn_rcpf(1.0f + t);
      total += q[i];
    }
    sum = group_sum<S::LPR>(sum);
    total = group_sum<S::LPR>(total);
    const float r = __builtin_amdgcn_rcpf(sum), rq = __builtin_amdgcn_rcpf(total);
#pragma unroll
    for (int i = 0; i < S::C; ++i) {
      p[i] *= r;
      q[i] *= rq;
    }
  }
  log_sum = isinf(m) ? 0.0f : logf(sum);
}

// Whether the row's token is real (all lanes of a wave call this; `in`: there is a row), and f(e) for each of its
// experts, once.
template <class S, typename I, class F>
MOE_DEV bool router_real(const I* idx, int k, int E, int j, bool in, F&& f) {
  bool any = false;
  if (in)
    for (int i = j; i < k; i += S::LPR) {
      const I e = idx[i];
      if (e >= 0 && e < (I)E) {
        any = true;
        f((int)e);
      }
    }
  const uint64_t b = __ballot(any);
  const int sub = (threadIdx.x & 63) / S::LPR;
  constexpr uint64_t mask = S::LPR == 64 ? ~0ull : (1ull << S::LPR) - 1;
  return ((b >> (sub * S::LPR)) & mask) != 0;
}

// The first sequence, from lo on, that ends behind row r.
MOE_DEV int router_first(const int* offsets, int S, int64_t r, int lo = 0) {
  int hi = S;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid + 1] > r) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
// Calls f(sequence, first row, end) for the parts of sequences in rows [r0, r1), in order, and none(first row, end) for
// rows of none.  A run of empty sequences is walked for eight and then searched for its end: 131072 of them within a block's rows
// took it 13 ms, a load after another.  Offsets of any values end the walk.
template <class F, class G>
MOE_DEV void router_walk(const int* offsets, int S, int64_t r0, int64_t r1, F&& f, G&& none) {
  if (!offsets) return f(0, r0, r1);
  int64_t r = r0;
  for (int s = uni(router_first(offsets, S, r0)); r < r1; ++s) {
    int64_t end = 0;
    for (int empty = 0; s < S && (end = uni(offsets[s + 1])) <= r; ++empty)
      s = empty < 8 ? s + 1 : uni(router_first(offsets, S, r, s + 1));
    if (s >= S) break;
    const int64_t a = min(max(r, (int64_t)uni(offsets[s])), r1), b = min(r1, end);
    if (a > r) none(r, min(a, b));
    if (b > a) f(s, a, b);
    r = b;
  }
  if (r < r1) none(r, r1);
}

// ------------------------------------------------------------------ forward
// Block b takes rows [b rpb, (b + 1) rpb) and writes, for each sequence s that has rows there, its column sums
// of q, its counts and (z sum, real tokens) to slot b + s: such pairs ascend in both, so no two share a slot.
// Bound by round trips to memory: nothing of a step's rows is requested before the step, the indices are loaded behind the
// logits, and bf16 rows' chunks (router_load) one behind the other: 65536 x 160 bf16 sigmoid scores in 48 sequences 24 us (0.9
// TB/s; the loop's instructions some 9), 8192 x 256 fp32 softmax 5.1 (1.7 TB/s).  More rows to a block leave the reduction fewer
// slots and the CUs idle: one block to a CU.
constexpr int kRouterBlock = 512;
template <class S, typename T, typename I>
__global__ __launch_bounds__(kRouterBlock) void k_router_losses(RouterRows<T, I> in, int64_t rpb,
                                                                float* __restrict__ part_q,
                                                                int* __restrict__ part_c,
                                                                float* __restrict__ part_z,
                                                                int* __restrict__ part_n) {
  constexpr int NW = kRouterBlock / 64;
  __shared__ float cols[NW][S::COLS];
  __shared__ int hist[S::COLS];
  __shared__ float zs[NW];
  __shared__ int ns[NW];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, j = lane % S::LPR, sub = lane / S::LPR;
  const int E = in.E, k = in.k;
  const float scale = in.inv_tau * kLog2E;
  const int64_t r0 = blockIdx.x * rpb, r1 = min(r0 + rpb, in.Tn);
  router_walk(in.offsets, in.S, r0, r1, [&](int s, int64_t a, int64_t b) {
    for (int e = tid; e < E; e += kRouterBlock) hist[e] = 0;
    __syncthreads();
    float acc[S::C], z = 0.0f;
    int n = 0;
#pragma unroll
    for (int i = 0; i < S::C; ++i) acc[i] = 0.0f;
    for (int64_t base = a + wave * S::RPW; base < b; base += NW * S::RPW) {
      const int64_t row = base + sub;
      const bool has = row < b;
      const int64_t at = has ? row : b - 1;
      float x[S::C], q[S::C], p[S::C], m, log_sum;
      router_load<S>(in.logits + at * E, E, j, x);
      const bool real = router_real<S>(in.idx + at * k, k, E, j, has, [&](int e) { atomicAdd(&hist[e], 1); });
      router_scores<S>(x, in.score, scale, q, p, m, log_sum);
      if (real) {
#pragma unroll
        for (int i = 0; i < S::C; ++i) acc[i] += q[i];
        if (j == 0) {
          const float lse = m * in.inv_tau + log_sum;
          z += lse * lse;
          ++n;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < S::C; ++i) {
      acc[i] = group_reduce<S::LPR, 64>(acc[i], [](float u, float v) { return u + v; });
      if (sub == 0) cols[wave][((i / S::V) * S::LPR + j) * S::V + i % S::V] = acc[i];
    }
    z = wave_sum(z);
    n = wave_butterfly(n, [](int u, int v) { return u + v; });
    if (lane == 0) zs[wave] = z, ns[wave] = n;
    __syncthreads();
    const int64_t slot = (int64_t)blockIdx.x + s;
    for (int e = tid; e < E; e += kRouterBlock) {
      float t = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) t += cols[w][e];
      part_q[slot * E + e] = t;
      part_c[slot * E + e] = hist[e];
    }
    if (tid == 0) {
      float zz = 0.0f;
      int nn = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) zz += zs[w], nn += ns[w];
      part_z[slot] = zz;
      part_n[slot] = nn;
    }
    __syncthreads();
  }, [](int64_t, int64_t) {});
}

// Sequence s = blockIdx.x: its blocks' parts added in 64 bits (in block order within kRouterParts interleaved sums),
// and the losses.  One workgroup to a sequence, bound by its CU's reads: 256 slots of 256 experts (0.5 MB) 9.5 us, of 48 sequences 5.6.
constexpr int kRouterParts = 32;
template <int V>
__global__ __launch_bounds__(1024) void k_router_reduce(const float* __restrict__ part_q, const int* __restrict__ part_c,
                                                        const float* __restrict__ part_z, const int* __restrict__ part_n,
                                                        const int* __restrict__ offsets, int64_t Tn, int64_t rpb, int E,
                                                        int k, float c_sw, float c_sq, float* __restrict__ balance,
                                                        float* __restrict__ zloss, int* __restrict__ counts,
                                                        float* __restrict__ slope, float* __restrict__ inv_real) {
  __shared__ double sums[1024 * V];
  __shared__ int cnts[1024 * V];
  __shared__ int n_all;
  __shared__ float terms[16];
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int64_t o0 = offsets ? min(max((int64_t)offsets[s], (int64_t)0), Tn) : 0;
  const int64_t o1 = offsets ? min(max((int64_t)offsets[s + 1], (int64_t)0), Tn) : Tn;
  const int64_t b0 = o0 / rpb, b1 = o1 > o0 ? (o1 - 1) / rpb + 1 : b0;  // blocks with rows of it
  const int ncv = E / V, parts = min(kRouterParts, 1024 / ncv);
  const int cv = tid % ncv, pl = tid / ncv;
  if (pl < parts) {
    double a[V];
    int c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = 0.0, c[v] = 0;
    constexpr int U = 8;  // in flight at once
    for (int64_t b = b0 + pl; b < b1; b += U * parts) {
      float f[U][V];
      int g[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool in = b + u * parts < b1;
        const int64_t at = (in ? b + u * parts + s : b + s) * E + cv * V;
        if constexpr (V == 4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(part_q + at);
          const u32x4 y = *reinterpret_cast<const u32x4*>(part_c + at);
#pragma unroll
          for (int v = 0; v < 4; ++v) f[u][v] = in ? x[v] : 0.0f, g[u][v] = in ? (int)y[v] : 0;
        } else {
          f[u][0] = in ? part_q[at] : 0.0f;
          g[u][0] = in ? part_c[at] : 0;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] += (double)f[u][v], c[v] += g[u][v];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sums[pl * E + cv * V + v] = a[v];
      cnts[pl * E + cv * V + v] = c[v];
    }
  }
  float zt = 0.0f;
  if (tid < 64) {
    double z = 0.0;
    int n = 0;
    for (int64_t b = b0 + lane; b < b1; b += 64) z += (double)part_z[b + s], n += part_n[b + s];
    n = wave_butterfly(n, [](int u, int v) { return u + v; });
    zt = wave_sum((float)z);
    if (tid == 0) n_all = n;
  }
  __syncthreads();
  const int n = n_all;
  const float rn = n > 0 ? 1.0f / (float)n : 0.0f;
  float term = 0.0f;
  if (tid < E) {
    double a = 0.0;
    int c = 0;
    for (int p = 0; p < parts; ++p) a += sums[p * E + tid], c += cnts[p * E + tid];
    const float P = n > 0 ? (float)(a / (double)n) : 0.0f;
    const float f = (float)c / (float)k * rn;
    term = P * (c_sw * f + c_sq * P);
    counts[(int64_t)s * E + tid] = c;
    if (slope) slope[(int64_t)s * E + tid] = (float)E * (c_sw * f + 2.0f * c_sq * P) * rn;
  }
  term = wave_sum(term);
  if (lane == 0) terms[tid >> 6] = term;
  __syncthreads();
  if (tid != 0) return;
  float t = 0.0f;
#pragma unroll
  for (int w = 0; w < 16; ++w) t += terms[w];
  balance[s] = (float)E * t;
  zloss[s] = zt * rn;
  if (inv_real) inv_real[s] = rn;
}

// ------------------------------------------------------------------ backward
// As the forward bound by round trips: 65536 x 160 bf16 sigmoid scores 29 us, 8192 x 256 fp32 softmax 8.2 (2.0 TB/s).
// Block b: rows [b rpb, (b + 1) rpb) over four waves.  slope: of balance in q, [S, E].  d_balance, d_z: [S], or null (0).
constexpr int kRouterBwdBlock = 256;
template <class S, typename T, typename I>
__global__ __launch_bounds__(kRouterBwdBlock) void k_router_losses_bwd(
    RouterRows<T, I> in, int64_t rpb, const float* __restrict__ slope, const float* __restrict__ inv_real,
    const float* __restrict__ d_balance, const float* __restrict__ d_z, T* __restrict__ d_logits) {
  constexpr int NW = kRouterBwdBlock / 64;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, j = lane % S::LPR, sub = lane / S::LPR;
  const int E = in.E, k = in.k;
  const float scale = in.inv_tau * kLog2E;
  const int64_t r0 = blockIdx.x * rpb, r1 = min(r0 + rpb, in.Tn);
  auto store = [&](int64_t row, const float (&d)[S::C]) {
#pragma unroll
    for (int i = 0; i < S::NCH; ++i) {
      const int c = (i * S::LPR + j) * S::V;
      if (c >= E) continue;
      if constexpr (S::V == 4) store4(d_logits + row * E + c, d + 4 * i);
      else d_logits[row * E + c] = from_f<T>(d[i]);
    }
  };
  router_walk(in.offsets, in.S, r0, r1, [&](int s, int64_t a, int64_t b) {
    // a loss without an upstream gradient adds nothing, also where its own value is not finite
    const float gb = d_balance ? d_balance[s] * in.inv_tau : 0.0f;
    const float h = d_z ? 2.0f * d_z[s] * inv_real[s] * in.inv_tau : 0.0f;
    float g[S::C];
#pragma unroll
    for (int i = 0; i < S::C; ++i) {
      const int c = ((i / S::V) * S::LPR + j) * S::V + i % S::V;
      g[i] = c < E && gb != 0.0f ? gb * slope[(int64_t)s * E + c] : 0.0f;
    }
    for (int64_t base = a + wave * S::RPW; base < b; base += NW * S::RPW) {
      const int64_t row = base + sub;
      const bool has = row < b;
      const int64_t at = has ? row : b - 1;
      float x[S::C], q[S::C], p[S::C], m, log_sum, dot = 0.0f;
      router_load<S>(in.logits + at * E, E, j, x);
      const bool real = router_real<S>(in.idx + at * k, k, E, j, has, [](int) {});
      // from the row's largest again, not from a kept lse: x - lse carries lse's rounding, |lse| 2^-24, which is all of log sum
      // where a row's logits are large (1 in each p of a row of the type's lowest value)
      router_scores<S>(x, in.score, scale, q, p, m, log_sum);
      // h lse; where lse is beyond fp32 the product need not be
      const float lse = m * in.inv_tau + log_sum, hl = isinf(lse) ? h * in.inv_tau * m + h * log_sum : h * lse;
#pragma unroll
      for (int i = 0; i < S::C; ++i) dot += q[i] * g[i];
      dot = group_sum<S::LPR>(dot);
      float d[S::C];
#pragma unroll
      for (int i = 0; i < S::C; ++i) {
        float t = q[i] * (g[i] - dot);
        if (in.score == kScoreSigmoid) {
          const float e = __builtin_amdgcn_exp2f(-fabsf(x[i]) * scale);
          t *= (x[i] > 0.0f ? e : 1.0f) * __builtin_amdgcn_rcpf(1.0f + e);
        }
        d[i] = !real ? 0.0f : h != 0.0f ? t + hl * p[i] : t;
      }
      if (has) store(row, d);
    }
  }, [&](int64_t a, int64_t b) {
    float d[S::C];
#pragma unroll
    for (int i = 0; i < S::C; ++i) d[i] = 0.0f;
    for (int64_t row = a + wave * S::RPW + sub; row < b; row += NW * S::RPW) store(row, d);
  });
}

}  // namespace moe
