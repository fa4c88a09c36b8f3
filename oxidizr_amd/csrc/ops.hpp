// HIP kernels of the operators that stand beside the MoE layer (gfx950 / CDNA4):
// tokens sorted by expert and back, and the norms before and after a block with
// its gate and residual scale.  expert_linear's kernels are in linear.hpp.
// No floating-point atomics: every reduction has a fixed order.
#pragma once
#include "kernels.hpp"

namespace moe {

// ------------------------------------------------------------------ sort by expert
// A stable counting sort of N = T k assignments by expert, flat index i = t k + j:
// expert ascending, then i ascending.  An index outside [0, E) has no expert and
// goes to bucket E, behind every expert, so perm and inv_perm are bijections for
// every input and offsets[E] is the number of assignments that have an expert.
// Every key may occur any number of times in a token.
//
// Block b owns a chunk of kSortTile-entry tiles; its wave w a contiguous eighth.
// base(b, w, e) = (buckets before e) + (e in earlier blocks) + (e in earlier waves);
// a wave then walks its part 64 entries at a time, and a lane's place among the
// lanes with its key comes from one ballot per key bit.  Up to kSortTile entries one
// launch does it all (512 entries, 128 experts: 4.7 us).  Bound by its chain of loads,
// LDS counts and scans, not by bytes: 65536 entries, 256 experts 3.8 us for the
// histograms and 7.4 for the rest.
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr int kSortTile = 2048;
// Blocks read every block's histogram: at most this many, longer chunks beyond.
constexpr int kSortMaxBlocks = 512;

template <typename I>
MOE_DEV int sort_key(const I* __restrict__ idx, int64_t i, int E) {
  const I v = idx[i];
  return v >= 0 && v < (I)E ? (int)v : E;
}

// hist[b][e]: entries of block b's chunk in bucket e, e <= E.
template <typename I>
__global__ __launch_bounds__(kSortThreads) void k_sort_hist(const I* __restrict__ idx, int64_t N,
                                                            int E, int64_t chunk,
                                                            int* __restrict__ hist) {
  extern __shared__ int cnt[];
  for (int e = threadIdx.x; e <= E; e += kSortThreads) cnt[e] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * chunk, i1 = min(N, i0 + chunk);
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kSortThreads)
    atomicAdd(&cnt[sort_key(idx, i, E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += kSortThreads)
    hist[(int64_t)blockIdx.x * (E + 1) + e] = cnt[e];
}

// LDS: kSortWaves x (E + 1) running positions.  hist is not read when the grid
// has one block.
template <typename I>
__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(
    const I* __restrict__ idx, int64_t N, int E, int64_t chunk, const int* __restrict__ hist,
    int* __restrict__ counts, int* __restrict__ offsets, int* __restrict__ perm,
    int* __restrict__ inv_perm) {
  extern __shared__ int pos[];  // [wave][bucket]
  __shared__ int wsum[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6);
  const int B = E + 1, nb = gridDim.x, b = blockIdx.x;
  for (int i = tid; i < kSortWaves * B; i += kSortThreads) pos[i] = 0;
  __syncthreads();
  const int64_t part = chunk / kSortWaves;
  const int64_t i0 = min(N, (int64_t)b * chunk + wave * part);
  const int64_t i1 = min(N, i0 + part);
  int* mine = pos + wave * B;
  for (int64_t i = i0 + lane; i < i1; i += 64) atomicAdd(&mine[sort_key(idx, i, E)], 1);
  __syncthreads();
  int carry = 0;
  for (int r0 = 0; r0 < B; r0 += kSortThreads) {  // exclusive scan over the buckets
    const int e = r0 + tid;
    int before = 0, total = 0;
    if (e < B) {
      if (nb > 1) {
        int p = 0;
        for (; p + 8 <= nb; p += 8) {
          int v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) v[u] = hist[(int64_t)(p + u) * B + e];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            total += v[u];
            before += p + u < b ? v[u] : 0;
          }
        }
        for (; p < nb; ++p) {
          const int v = hist[(int64_t)p * B + e];
          total += v;
          before += p < b ? v : 0;
        }
      } else {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) total += pos[w * B + e];
      }
    }
    const int incl = wave_incl_scan(total);
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int start = carry + incl - total, all = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      start += w < wave ? wsum[w] : 0;
      all += wsum[w];
    }
    carry += all;
    __syncthreads();  // wsum is rewritten by the next round
    if (e < B) {
      if (b == 0) {
        offsets[e] = start;
        if (e < E) counts[e] = total;
      }
      int run = start + before;
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const int c = pos[w * B + e];
        pos[w * B + e] = run;
        run += c;
      }
    }
  }
  __syncthreads();
  const int bits = 32 - __clz(E);
  const uint64_t below = (1ull << lane) - 1;
  for (int64_t i = i0; i < i1; i += 64) {  // wave-uniform trip count
    const bool in = i + lane < i1;
    const int key = in ? sort_key(idx, i + lane, E) : 0;
    uint64_t same = __ballot(in);
    for (int k = 0; k < bits; ++k) {
      const bool on = (key >> k) & 1;
      const uint64_t m = __ballot(on);
      same &= on ? m : ~m;
    }
    const int rank = __popcll(same & below);
    const int base = in ? mine[key] : 0;
    // every lane has read its bucket's position before the first lane of each
    // bucket moves it (one wave: LDS operations keep their order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) mine[key] = base + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in) {
      perm[base + rank] = (int)(i + lane);
      inv_perm[i + lane] = base + rank;
    }
  }
}

// ------------------------------------------------------------------ rows to experts and back
// inv_perm[t k + j] says which row of the sorted order holds assignment (t, j);
// rows at or beyond *kept belong to no expert.  A position outside [0, T k) (no
// sort makes one) counts as such, and neither it nor a *kept beyond T k makes a kernel
// leave its buffers.
MOE_DEV int kept_rows(const int* kept, int64_t N) { return (int)min((int64_t)*kept, N); }
constexpr int kMaxPerTok = 16;

// xp[inv[t, j]] = x[t], or zeros for an assignment without an expert.  One wave
// per (token, 64 16-byte vectors): it reads its part of the row once and writes it k
// times.  Bound by memory: 8192 tokens of H = 7168, k = 8 (1.06 GB) 175 us, 6.0 TB/s; 64 of
// H = 4096, k = 8 3.6 us.
template <typename T>
__global__ __launch_bounds__(256) void k_permute(const T* __restrict__ x,
                                                 const int* __restrict__ inv,
                                                 const int* __restrict__ kept, int64_t Tn, int k,
                                                 int H, T* __restrict__ xp) {
  constexpr int V = Vec16<T>::N;
  const int nv = H / V, nsl = (nv + 63) / 64;
  const int64_t wid = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (wid >= Tn * nsl) return;
  const int64_t t = wid / nsl;
  const int lane = threadIdx.x & 63;
  const int c = (int)(wid - t * nsl) * 64 + lane;
  const bool in = c < nv;  // no early exit: lane j holds slot j's row
  const int64_t N = Tn * k;
  const int rows = kept_rows(kept, N);
  const int at = lane < k ? inv[t * k + lane] : -1;
  const u32x4 v = in ? ld16(x + t * H + (int64_t)c * V) : u32x4{0, 0, 0, 0};
  for (int j = 0; j < k; ++j) {
    const int p = __builtin_amdgcn_readlane(at, j);
    if (in && p >= 0 && p < N)
      st16_stream(xp + (int64_t)p * H + c * V, p < rows ? v : u32x4{0, 0, 0, 0});
  }
}

// out[t] = sum_j w[t, j] y[inv[t, j]] over the assignments that have an expert, j
// ascending, in fp32, rounded once (w null: every weight is 1).  One wave per
// (token, 64 vectors); a slice's k rows are all requested before the first is added.
// Bound by memory: H = 7168, k = 8 of 8192 tokens (1.06 GB) 173 us, 6.1 TB/s; H = 2048, k = 6
// of 16384 (470 MB) 70 us, 6.7 TB/s.  At least four waves to a SIMD: left alone the
// compiler takes 242 registers for fp32 and eight rows, two waves.
// STREAM: rows of more than kStreamBytes, which the caches would not hold anyway, are
// loaded with the nontemporal hint (939 MB, k = 8, H = 7168: 190 -> 176 us; 403 MB, k = 6:
// 86 -> 78; but 67 MB just written, k = 2: 14.8 -> 18.2).
constexpr int64_t kStreamBytes = int64_t(256) << 20;
template <typename T, int KMAX, bool STREAM>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void k_unpermute(const T* __restrict__ y,
                                                   const int* __restrict__ inv,
                                                   const int* __restrict__ kept,
                                                   const float* __restrict__ w, int64_t Tn, int k,
                                                   int H, T* __restrict__ out) {
  constexpr int V = Vec16<T>::N;
  const int nv = H / V, nsl = (nv + 63) / 64;
  const int64_t wid = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (wid >= Tn * nsl) return;
  const int64_t t = wid / nsl;
  const int lane = threadIdx.x & 63;
  const int c = (int)(wid - t * nsl) * 64 + lane;
  const int rows = kept_rows(kept, Tn * k);
  const int at = lane < k ? inv[t * k + lane] : -1;
  const float wt = lane < k ? (w ? w[t * k + lane] : 1.0f) : 0.0f;
  const bool in = c < nv;  // no early exit: lane j holds slot j's row and weight
  u32x4 v[KMAX];
#pragma unroll
  for (int j = 0; j < KMAX; ++j) {  // slots past k are -1
    const int p = __builtin_amdgcn_readlane(at, j);
    if (in && p >= 0 && p < rows) v[j] = ld16_maybe_stream<STREAM>(y + (int64_t)p * H + c * V);
  }
  float acc[V], f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.0f;
#pragma unroll
  for (int j = 0; j < KMAX; ++j) {
    const int p = __builtin_amdgcn_readlane(at, j);
    const float wj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wt), j));
    if (in && p >= 0 && p < rows) {
      unpack16(v[j], f, T());
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += wj * f[i];
    }
  }
  if (in) st16_stream(out + t * H + c * V, pack16(acc, T()));
}

// dy[inv[t, j]] = w[t, j] dout[t] (zeros without an expert) and, with y,
// dw[t, j] = <dout[t], y[inv[t, j]]> in fp32.  WPT waves to a token (4 / WPT tokens
// to a block): wave q takes slices q, q + WPT, .. of 64 vectors; the waves' parts
// of dw are added in order.  Bound by memory: H = 2048, k = 6 of 16384 tokens (872 MB) 162
// us, 5.4 TB/s.
template <typename T, int WPT, int KMAX>
__global__ __launch_bounds__(256) void k_unpermute_bwd(
    const T* __restrict__ dout, const T* __restrict__ y, const int* __restrict__ inv,
    const int* __restrict__ kept, const float* __restrict__ w, int64_t Tn, int k, int H,
    T* __restrict__ dy, float* __restrict__ dw) {
  constexpr int V = Vec16<T>::N, TPB = 4 / WPT;
  __shared__ float red[4][kMaxPerTok];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int q = wave % WPT;
  const int64_t t = (int64_t)blockIdx.x * TPB + wave / WPT, N = Tn * k;
  const bool live = t < Tn;
  const int nv = H / V;
  const int rows = kept_rows(kept, Tn * k);
  const int at = live && lane < k ? inv[t * k + lane] : -1;
  const float wt = live && lane < k ? (w ? w[t * k + lane] : 1.0f) : 0.0f;
  float dot[KMAX];
#pragma unroll
  for (int j = 0; j < KMAX; ++j) dot[j] = 0.0f;
  if (live)
    for (int c = q * 64 + lane; c - lane < nv; c += 64 * WPT) {
      const bool in = c < nv;
      float d[V];
      u32x4 v[KMAX];
      const u32x4 raw = in ? ld16(dout + t * H + (int64_t)c * V) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < KMAX; ++j)
        if (j < k && dw) {
          const int p = __builtin_amdgcn_readlane(at, j);
          if (in && p >= 0 && p < rows) v[j] = ld16(y + (int64_t)p * H + c * V);
        }
      unpack16(raw, d, T());
#pragma unroll
      for (int j = 0; j < KMAX; ++j)
        if (j < k) {
          const int p = __builtin_amdgcn_readlane(at, j);
          if (p < 0 || p >= N) continue;
          const bool real = p < rows;
          const float wj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wt), j));
          if (in && real && dw) {
            float f[V];
            unpack16(v[j], f, T());
#pragma unroll
            for (int i = 0; i < V; ++i) dot[j] += d[i] * f[i];
          }
          if (in) {
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = real ? wj * d[i] : 0.0f;
            st16_stream(dy + (int64_t)p * H + c * V, pack16(o, T()));
          }
        }
    }
  if (!dw) return;
#pragma unroll
  for (int j = 0; j < KMAX; ++j)
    if (j < k) {
      const float s = wave_sum(dot[j]);
      if (WPT == 1) {
        if (live && lane == 0) dw[t * k + j] = s;
      } else if (lane == 0) {
        red[wave][j] = s;
      }
    }
  if constexpr (WPT > 1) {
    __syncthreads();
    if (live && q == 0 && lane < k) {
      float s = red[wave][lane];
#pragma unroll
      for (int i = 1; i < WPT; ++i) s += red[wave + i][lane];
      dw[t * k + lane] = s;
    }
  }
}

// ------------------------------------------------------------------ norms around a block
//   u = y rstd(y) w2 (or y without a norm after the block), rstd(v) = 1 / sqrt(mean(v^2) + eps)
//   hn = scale h + g u,  n = hn rstd(hn) w3
// g: none (1), a channel vector [H], one number to a token [T] or a full [T, H].
// Without y: hn = h (scale 1, not written), a plain RMSNorm.  Statistics and products
// in fp32; hn and n are each rounded once, n from the unrounded hn.
//
// WPR waves share a row, in chunks of 8 elements: thread i of the row owns chunks
// i, i + 64 WPR, .. (NCH of them), which stay in registers between the two
// statistics: every tensor is read once and written once.  Bound by memory: 8192 x 7168
// bf16 (470 MB) 85 us, 5.5 TB/s; one row of 2048 2.8 us.
enum { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };

template <typename T>
struct NormArgs {
  const T *h, *y, *w2, *gate, *w3;
  int gate_kind;
  float scale, eps;
  int64_t Tn;
  int H;
  T *hn, *n;
  float *r2, *r3;  // [T]; null when no backward follows
};

// Sum over the row's 64 WPR threads, waves in order.  red: one float to a wave, a
// buffer of its own for each call between two barriers.
template <int WPR>
MOE_DEV float row_sum(float v, float* red, int wave) {
  v = wave_sum(v);
  if constexpr (WPR == 1) return v;
  if ((threadIdx.x & 63) == 0) red[wave] = v;
  __syncthreads();
  const float* r = red + wave / WPR * WPR;
  float s = r[0];
#pragma unroll
  for (int i = 1; i < WPR; ++i) s += r[i];
  return s;
}

template <typename T, int WPR, int NCH>
__global__ __launch_bounds__(WPR > 4 ? 64 * WPR : 256) void k_norm_fwd(NormArgs<T> a) {
  constexpr int NW = WPR > 4 ? WPR : 4, RPB = NW / WPR, TR = 64 * WPR;
  __shared__ float red[2][NW];
  const int wave = uni(threadIdx.x >> 6);
  const int i0 = threadIdx.x % TR;
  const int64_t t = (int64_t)blockIdx.x * RPB + wave / WPR;
  const bool live = t < a.Tn;
  const int nch = live ? a.H / 8 : 0;
  const int64_t row = t * a.H;
  const float inv_h = 1.0f / (float)a.H;
  float u[NCH][8], o[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int ch = i0 + c * TR;
#pragma unroll
    for (int i = 0; i < 8; ++i) u[c][i] = o[c][i] = 0.0f;
    if (ch < nch) {
      load8(a.h + row + ch * 8, o[c]);
      if (a.y) load8(a.y + row + ch * 8, u[c]);
    }
  }
  if (a.y) {
    float s = 0.0f;
    if (a.w2) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += u[c][i] * u[c][i];
      s = 1.0f / sqrtf(row_sum<WPR>(s, red[0], wave) * inv_h + a.eps);
      if (live && i0 == 0 && a.r2) a.r2[t] = s;
    }
    const float gt = a.gate_kind == kGateToken && live ? to_f<T>(a.gate[t]) : 1.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int ch = i0 + c * TR;
      if (ch < nch) {
        float v[8];
        if (a.w2) {
          load8(a.w2 + ch * 8, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) u[c][i] = u[c][i] * s * v[i];
        }
        if (a.gate_kind == kGateChannel || a.gate_kind == kGateFull) {
          load8(a.gate + (a.gate_kind == kGateFull ? row : 0) + ch * 8, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) u[c][i] *= v[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) o[c][i] = a.scale * o[c][i] + gt * u[c][i];
        store8_stream(a.hn + row + ch * 8, o[c]);
      }
    }
  }
  if (!a.w3) return;
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) s += o[c][i] * o[c][i];
  s = 1.0f / sqrtf(row_sum<WPR>(s, red[1], wave) * inv_h + a.eps);
  if (live && i0 == 0 && a.r3) a.r3[t] = s;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int ch = i0 + c * TR;
    if (ch < nch) {
      float v[8];
      load8(a.w3 + ch * 8, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = o[c][i] * s * v[i];
      store8_stream(a.n + row + ch * 8, v);
    }
  }
}

// Backward, with hh = hn r3, yh = y r2, u = yh w2 (u = y without w2); hn is formed again
// from h and u, as the forward had it before its rounding (hn_given: read as the forward stored it):
//   D = dhn + r3 (w3 dn - hh mean(hh w3 dn)),  dh = scale D,
//   dgate = D u,  dy = r2 (g w2 D - yh mean(yh g w2 D))  (g D without w2),
//   dw3 = sum_t dn hh,  dw2 = sum_t g D yh.
// D is linear in m3 = mean(hh w3 dn), so with P = dhn + r3 w3 dn one reduction of
// three sums gives both means: mean(u g D) = mean(u g P) - r3 m3 mean(u g hh).
// A token gate leaves the sums (g is applied behind them), which makes them its
// gradient as well; a channel gate's dgate and dw2 are both sum_t D yh times a
// vector.  So a row costs one barrier, and there are at most two column sums:
//   colA = sum_t D yh (channel or no gate; yh = y without w2) or sum_t g D yh,
//   colB = sum_t dn hh.
// A block takes rows b, b + grid, ..; its column sums stay with their threads and go to
// part[b] = (colA | colB), which k_norm_colsum adds in order.  The next row's loads are
// in flight over a row's reduction and stores.  Bound by memory: 8192 x 7168 bf16 (705 MB)
// 135 us, 5.2 TB/s (without the loads ahead 270); fp32 8192 x 4096 155 us, 5.2.  That holds up to H =
// 8192 in bf16 and 4096 in fp32, where all of a thread's columns are in registers.  Wider rows have
// 128 registers for more (16 waves to a block) and spill 57 (fp32 up to 8192) to 871 of them, 136 to
// 1600 bytes a lane, and that traffic bounds them: fp32 8192 x 7168 354 us, 4.0 TB/s; 4096 x 16384 472
// bf16 and 968 fp32, 1.7; 2048 x 32768 848 and 1531, 1.0.  Forming hn costs some 5 us of them; with the
// rounded hn the gradients were 2.5e-3 off a 64-bit form, now 1.7e-3 (relative L2).
template <typename T>
struct NormBwdArgs {
  const T *dhn, *dn;  // either may be null (zero)
  const T *h, *y, *w2, *gate, *w3;  // h: hn in its place when hn_given
  int gate_kind, hn_given;
  float scale;
  int64_t Tn;
  int H;
  const float *r2, *r3;
  T *dh, *dy, *dgate;  // dgate: token and full gates
  float* part;         // [grid][ncol][H], ncol = need_a + need_b
  int need_a, need_b;
};

// Eight elements as they lie in memory.
template <typename T>
struct Raw8 {
  static constexpr int N = 8 / Vec16<T>::N;
  u32x4 v[N];
  MOE_DEV void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = *gptr(reinterpret_cast<const u32x4*>(p + i * Vec16<T>::N));
  }
  MOE_DEV void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) unpack16(v[i], f + i * Vec16<T>::N, T());
  }
};

template <typename T, int WPR, int NCH>
__global__ __launch_bounds__(WPR > 4 ? 64 * WPR : 256) void k_norm_bwd(NormBwdArgs<T> a) {
  constexpr int NW = WPR > 4 ? WPR : 4, RPB = NW / WPR, TR = 64 * WPR;
  __shared__ float red[2][3][NW];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int i0 = threadIdx.x % TR;
  const int nch = a.H / 8;
  const float inv_h = 1.0f / (float)a.H;
  const bool chan = a.gate_kind == kGateChannel, full = a.gate_kind == kGateFull;
  const bool form = a.y && !a.hn_given;
  // the row vectors of a thread's columns, and the next row's tensors
  Raw8<T> w2[NCH], w3[NCH], gc[NCH], nd[NCH], nn[NCH], nh[NCH], ny[NCH], ng[NCH];
  float ca[NCH][8], cb[NCH][8];
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int ch = i0 + c * TR;
#pragma unroll
    for (int i = 0; i < 8; ++i) ca[c][i] = cb[c][i] = 0.0f;
    if (ch < nch) {
      if (a.w2) w2[c].load(a.w2 + ch * 8);
      if (a.w3) w3[c].load(a.w3 + ch * 8);
      if (chan) gc[c].load(a.gate + ch * 8);
    }
  }
  auto load_row = [&](int64_t t) {
    if (t >= a.Tn) return;
    const int64_t row = t * a.H;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int ch = i0 + c * TR;
      if (ch >= nch) continue;
      if (a.dhn) nd[c].load(a.dhn + row + ch * 8);
      if (a.w3) {
        nn[c].load(a.dn + row + ch * 8);
        nh[c].load(a.h + row + ch * 8);
      }
      if (a.y) ny[c].load(a.y + row + ch * 8);
      if (full) ng[c].load(a.gate + row + ch * 8);
    }
  };
  int set = 0;
  const int64_t stride = (int64_t)gridDim.x * RPB;
  const int64_t t0 = (int64_t)blockIdx.x * RPB;
  load_row(t0 + wave / WPR);
  for (int64_t tb = t0; tb < a.Tn; tb += stride, set ^= 1) {
    const int64_t t = tb + wave / WPR;
    const bool live = t < a.Tn;
    const int64_t row = t * a.H;
    const float r3 = live && a.w3 ? a.r3[t] : 0.0f;
    const float r2 = live && a.w2 ? a.r2[t] : 1.0f;
    const float gt = live && a.gate_kind == kGateToken ? to_f<T>(a.gate[t]) : 1.0f;
    float p[NCH][8], hh[NCH][8], yh[NCH][8];
    Raw8<T> g[NCH];
    float s3 = 0.0f, sp = 0.0f, sh = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int ch = i0 + c * TR;
#pragma unroll
      for (int i = 0; i < 8; ++i) p[c][i] = hh[c][i] = yh[c][i] = 0.0f;
      if (!live || ch >= nch) continue;
      float v[8], u[8];
      if (a.dhn) nd[c].get(p[c]);
      if (a.y) {
        ny[c].get(yh[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = yh[c][i] *= r2;
        if (a.w2) {
          w2[c].get(v);
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] *= v[i];
        }
        if (chan || full) {
          g[c] = full ? ng[c] : gc[c];
          g[c].get(v);
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] *= v[i];
        }
      }
      if (a.w3) {
        float d[8];
        nn[c].get(d);
        nh[c].get(hh[c]);
        w3[c].get(v);
        if (form) {
#pragma unroll
          for (int i = 0; i < 8; ++i) hh[c][i] = a.scale * hh[c][i] + gt * u[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          hh[c][i] *= r3;
          cb[c][i] += d[i] * hh[c][i];
          d[i] *= v[i];
          s3 += hh[c][i] * d[i];
          p[c][i] += r3 * d[i];
        }
      }
      if (a.y) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sp += u[i] * p[c][i];
          sh += u[i] * hh[c][i];
        }
      }
    }
    load_row(t + stride);  // in flight over this row's reduction and stores
    s3 = wave_sum(s3);
    sp = wave_sum(sp);
    sh = wave_sum(sh);
    if constexpr (WPR > 1) {
      float(*r)[NW] = red[set];
      if (lane == 0) {
        r[0][wave] = s3;
        r[1][wave] = sp;
        r[2][wave] = sh;
      }
      lds_barrier();  // not the row loads in flight
      const int w0 = wave / WPR * WPR;
      s3 = r[0][w0]; sp = r[1][w0]; sh = r[2][w0];
#pragma unroll
      for (int i = 1; i < WPR; ++i) {
        s3 += r[0][w0 + i];
        sp += r[1][w0 + i];
        sh += r[2][w0 + i];
      }
    }
    if (!live) continue;
    const float m3 = r3 * (s3 * inv_h);
    const float su = sp - m3 * sh;  // sum of u (g) D over the row
    if (a.gate_kind == kGateToken && i0 == 0) a.dgate[t] = from_f<T>(su);
    const float m2 = a.w2 ? gt * su * inv_h : 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int ch = i0 + c * TR;
      if (ch >= nch) continue;
      float o[8], v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[c][i] -= m3 * hh[c][i];
        o[i] = a.scale * p[c][i];
      }
      store8_stream(a.dh + row + ch * 8, o);
      if (!a.y) continue;
      float gv[8], wv[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        gv[i] = gt;
        wv[i] = 1.0f;
      }
      if (chan || full) g[c].get(gv);
      if (a.w2) w2[c].get(wv);
      if (full) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[c][i] * yh[c][i] * wv[i];
        store8_stream(a.dgate + row + ch * 8, v);
      }
      const bool colg = a.gate_kind >= kGateToken;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = gv[i] * p[c][i];
        ca[c][i] += (colg ? d : p[c][i]) * yh[c][i];
        o[i] = r2 * (wv[i] * d - yh[c][i] * m2);
      }
      store8_stream(a.dy + row + ch * 8, o);
    }
  }
  // the block's column sums: its rows' waves in order
  const int ncol = a.need_a + a.need_b;
  if (ncol == 0) return;
  float* dst = a.part + (int64_t)blockIdx.x * ncol * a.H;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int ch = i0 + c * TR;
      if (ch >= nch) continue;
      if (a.need_a) store8(dst + ch * 8, ca[c]);
      if (a.need_b) store8(dst + (int64_t)a.need_a * a.H + ch * 8, cb[c]);
    }
  } else {
    __shared__ float col[NW][64 * NCH * 8];
    auto fold = [&](float(&v)[NCH][8], float* out) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) col[wave][(c * 64 + lane) * 8 + i] = v[c][i];
      __syncthreads();
      if (wave / WPR != 0) return;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int ch = i0 + c * TR;
        if (ch >= nch) continue;
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          s[i] = col[wave][(c * 64 + lane) * 8 + i];
#pragma unroll
          for (int r = 1; r < RPB; ++r) s[i] += col[wave + r * WPR][(c * 64 + lane) * 8 + i];
        }
        store8(out + ch * 8, s);
      }
    };
    if (a.need_a) fold(ca, dst);
    if (a.need_b) fold(cb, dst + (int64_t)a.need_a * a.H);
  }
}

// Column sums of the nb partial rows of k_norm_bwd, and the weight gradients
// from them: dw2 = colA (g of a channel gate), dgate = colA w2 (channel gate), dw3 =
// colB.  A block owns kColsumCols columns of one sum; its thread (r, c) adds rows r, r +
// 64, .. of 8 columns, then eight threads' sums, then the eight that are left, each in
// order.  Bound by its chain of loads: 1024 rows of 776 7 us, 256 of 7168 5 (16 columns to a
// block 5 and 7, 64 columns 12 and 6).
constexpr int kColsumCols = 32;
template <typename T>
__global__ __launch_bounds__(256) void k_norm_colsum(const float* __restrict__ part, int nb, int H,
                                                     int need_a, int need_b,
                                                     const T* __restrict__ w2,
                                                     const T* __restrict__ chan_gate,
                                                     T* __restrict__ dw2, T* __restrict__ dgate,
                                                     T* __restrict__ dw3) {
  constexpr int C = kColsumCols, R = 256 / (C / 8), G = 256 / C;  // row lanes, and their groups
  __shared__ float col[R][C], grp[G][C];
  const int which = blockIdx.y;
  const int r0 = threadIdx.x / (C / 8), c8 = threadIdx.x % (C / 8) * 8;
  const int c = blockIdx.x * C + c8;
  const int64_t ld = (int64_t)(need_a + need_b) * H;
  float s[8], v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = 0.0f;
  if (c < H)
    for (int r = r0; r < nb; r += R) {
      load8(part + r * ld + (int64_t)which * H + c, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += v[i];
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) col[r0][c8 + i] = s[i];
  __syncthreads();
  const int g = threadIdx.x / C, n = threadIdx.x % C;
  float t = 0.0f;
#pragma unroll
  for (int r = 0; r < R / G; ++r) t += col[g * (R / G) + r][n];
  grp[g][n] = t;
  __syncthreads();
  const int cc = blockIdx.x * C + n;
  if (g > 0 || cc >= H) return;
  t = 0.0f;
#pragma unroll
  for (int r = 0; r < G; ++r) t += grp[r][n];
  if (which == need_a) {
    dw3[cc] = from_f<T>(t);
    return;
  }
  if (dw2) dw2[cc] = from_f<T>(chan_gate ? t * to_f<T>(chan_gate[cc]) : t);
  if (dgate) dgate[cc] = from_f<T>(w2 ? t * to_f<T>(w2[cc]) : t);
}

}  // namespace moe
