// HIP kernels of microscaled 4-bit numbers (gfx950 / CDNA4): quantisation and back, and expert products
// over 4-bit weights.
//
// The format is the OCP microscaling formats' MXFP4: 32 elements along a row share a scale 2^s, an E8M0 byte
// s + 127 (255: NaN); an element is an E2M1 number, 0 0.5 1 1.5 2 3 4 6 with a sign in bit 3.  Element 2 i of a
// row is the low half of its byte i.  A row of K elements (K a multiple of 32) is K / 2 bytes of codes and K / 32
// bytes of scales, both row-major.
//
//   z[r] = x[r] W_e^T + b_e,  y[r] = act(z[r]) + res[r]   for r in expert e's rows,
//   dz = dy act'(z),  dx = dz W_e,  db_e = sum_r dz[r],  dres = dy
// with W_e [N, K] in 4 bits and x in bf16, or in 4 bits too (no gradients then: a rounding has none).
#pragma once
#include "linear.hpp"

namespace moe {

constexpr int kMxBlock = 32;  // elements under one scale

// An E8M0 byte as the conversions take it: they read a float's exponent alone, for which 0 is 2^-127
// and 255 a NaN (which makes every element one).
MOE_DEV float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight elements (a dword of codes) as bf16: exact (2 bits of mantissa, and bf16 has E8M0's range); what is 2^128 or more, as in
// fp32, becomes infinite, but no quantisation makes a scale above 2^125.
MOE_DEV u32x4 mx_bf16x8(uint32_t c, float s) {
  u32x4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3));
  return r;
}

// ------------------------------------------------------------------ quantisation
// s = floor(log2 of the block's largest magnitude) - 2, so that it becomes 4 .. 8 2^s and what is above 6 2^s
// becomes that; elements are rounded to the nearest code, ties to the even one (v_cvt_scalef32_pk_fp4).  A
// block with an infinity or a NaN has scale 255: all of it is NaN.  A lane takes eight elements, four neighbouring
// lanes a block.  Bound by its bytes: 65536 x 4096 bf16 (680 MB) 107 us, 6.4 TB/s; 46 million fp32 elements (209 MB, which the
// caches hold) 29.5 us, 7.1 TB/s, and as long back.
template <typename T>
__global__ __launch_bounds__(256) void k_mx_quantize(const T* __restrict__ x, int64_t nvec,
                                                     uint32_t* __restrict__ codes,
                                                     uint8_t* __restrict__ scales) {
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (v >= nvec) return;  // whole blocks of four lanes
  float f[8];
  load8(x + v * 8, f);
  int m = 0;  // magnitudes order as integers, infinity and NaN above all numbers
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_int(f[i]) & 0x7fffffff);
  m = max(m, lane_xor<1>(m));
  m = max(m, lane_xor<2>(m));
  const bool none = m >= 0x7f800000;
  const int byte = none ? 255 : max((m >> 23) - 2, 0);
  const float s = mx_scale(byte);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], s, 3);
  codes[v] = none ? 0u : c;
  if ((threadIdx.x & 3) == 0) scales[v >> 2] = (uint8_t)byte;
}

// A lane writes 16 bytes, next to its neighbour's: eight bf16 of a dword of codes, or four floats of half of one (with eight
// floats to a lane 184 MB of them took 54 to 72 us).
MOE_DEV u32x4 mx_vector(const uint32_t* codes, int64_t v, float s, bf16_t) { return mx_bf16x8(codes[v], s); }
MOE_DEV u32x4 mx_vector(const uint32_t* codes, int64_t v, float s, float) {
  const uint32_t c = reinterpret_cast<const uint16_t*>(codes)[v];
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
  return u32x4{__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(b[0]), __float_as_uint(b[1])};
}
template <typename T>
__global__ __launch_bounds__(256) void k_mx_dequantize(const uint32_t* __restrict__ codes,
                                                       const uint8_t* __restrict__ scales, int64_t nvec,
                                                       T* __restrict__ y) {
  constexpr int V = Vec16<T>::N;
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (v >= nvec) return;
  st16_stream(y + v * V, mx_vector(codes, v, mx_scale(scales[v / (kMxBlock / V)]), T()));
}

// ------------------------------------------------------------------ tiled products
// The weights of a launch: group g's matrix at codes + g N K / 2, scales + g N K / 32.
struct MxWeights {
  const uint8_t *codes, *scales;
  int N, K;
};

// Rows of a launch: groups by offsets [G + 1], or (null) M rows of one.
struct MxRows {
  const int* offsets;
  int G, M;
};

// Block blk's part of n tiles of BM rows, dealt over the XCDs as xcd_slot does.  An XCD's 32 CUs take 32 tiles of 256 rows at
// once; where the tiles behind its last full 32 are few, each is cut into two or four parts of as many rows, for the
// CUs that would stand by.
MOE_DEV int mx_parts(int tail) { return tail <= 8 ? 4 : tail <= 16 ? 2 : 1; }
template <int BM>
MOE_DEV bool mx_slot(int blk, int n, int& id, int& part, int& parts) {
  part = 0;
  parts = 1;
  if constexpr (BM != 256) return xcd_slot(blk, n, id);
  const int x = blk & 7, j = blk >> 3, q = n >> 3, r = n & 7;
  const int mine = q + (x < r ? 1 : 0), full = mine & ~31, tail = mine - full;
  id = x * q + min(x, r) + j;
  if (j < full) return true;
  parts = mx_parts(tail);
  const int t = j - full;
  if (t >= tail * parts) return false;
  id += t / parts - t;
  part = t % parts;
  return true;
}

// Row tiles of BM rows of a launch's groups, numbered group by group as resolve_rows has them, but from the offsets alone:
// lane l counts those of groups l G / 64 .., a prefix sum over the lanes gives their number and the lane that holds a tile's
// group, so a grouped call needs no launch before it (a kernel that writes prefixes takes 6 us, and finding a group in them
// log2(G) loads one after another).  Offsets are clamped to 0 .. M and each group's end to its start: whatever they hold, a
// tile's rows exist.
template <int BM>
struct MxTileScan {
  MxRows r;
  int per, n, incl, total;
  MOE_DEV explicit MxTileScan(const MxRows& rows) : r(rows), per((rows.G + 63) >> 6), n(0) {
    const int l = threadIdx.x & 63;
    for (int i = 0; i < per; ++i) {
      int a, b;
      if (l * per + i < r.G) n += range(l * per + i, a, b);
    }
    incl = wave_incl_scan(n);
    total = __builtin_amdgcn_readlane(incl, 63);
  }
  MOE_DEV int range(int e, int& a, int& b) const {  // its tiles
    a = min(max(r.offsets[e], 0), r.M);
    b = min(max(r.offsets[e + 1], a), r.M);
    return (b - a + BM - 1) / BM;
  }
  // Walks lane l's groups until f(group, its first tile, its tiles, first row, end) is true.
  template <class F>
  MOE_DEV void walk(int l, F&& f) const {
    int first = __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(n, l);
    for (int i = 0; i < per && l * per + i < r.G; ++i) {
      int a, b;
      const int c = uni(range(l * per + i, a, b));
      if (f(l * per + i, first, c, uni(a), uni(b))) return;
      first += c;
    }
  }
  MOE_DEV int lane_of(int tile) const { return __ffsll((unsigned long long)__ballot(incl > tile)) - 1; }  // tile < total
};

// The tile of block blk of a launch with N output columns: group, first row, rows and first column, or false for a
// block past the tiles.
template <int BM, int BN>
MOE_DEV bool mx_tile(const MxRows& r, int N, int blk, int& grp, int& row0, int& mv, int& n0) {
  const int nN = (N + BN - 1) / BN;
  int id, mt, nt, part, parts;
  auto rows = [&](int first, int end) {  // the part's rows of a tile
    row0 = first + mt * BM + part * (BM / parts);
    mv = min(BM / parts, end - row0);
    n0 = nt * BN;
    return mv > 0;
  };
  if (r.offsets == nullptr) {
    const int nM = (r.M + BM - 1) / BM;
    if (!mx_slot<BM>(blk, nM * nN, id, part, parts) || !tile_order(id, nM, nN, mt, nt)) return false;
    grp = 0;
    return rows(0, r.M);
  }
  const MxTileScan<BM> scan(r);
  if (!mx_slot<BM>(blk, scan.total * nN, id, part, parts)) return false;
  const int s = uni(id / nN);
  bool found = false;
  scan.walk(scan.lane_of(s), [&](int e, int first, int c, int a, int b) {
    if (s >= first + c) return false;
    grp = e;
    found = tile_order<kRowWalk>(id - first * nN, c, nN, mt, nt) && rows(a, b);
    return true;
  });
  return found;
}

// body(tiling): a BM/4- or BM/2-row tiling when that covers the mv valid rows, else the half-width tiling when at most
// BN / 2 of the nv remaining columns are valid, else the 3BM/4-row tiling when that covers the rows, else C.
template <class C, class F>
MOE_DEV void with_mx_shape(int mv, int nv, F&& body) {
  if constexpr (has_half_rows<bf16_t, C>()) {
    if (mv <= C::BM / 4) return body(QuarterRows<C>{});
    if (mv <= C::BM / 2) return body(HalfRows<C>{});
    if (nv <= C::BN / 2) return body(HalfCols<C>{});
    if (mv <= 3 * C::BM / 4) return body(ThreeQuarterRows<C>{});
  }
  body(C{});
}
constexpr int max_of(int a, int b) { return a > b ? a : b; }
template <class C>
constexpr int mx_smem_elems() {
  int n = kernel_smem_elems<C, bf16_t, 1, 1, 1>();
  if constexpr (has_half_rows<bf16_t, C>()) {
    n = max_of(n, max_of(kernel_smem_elems<QuarterRows<C>, bf16_t, 1, 1, 1>(), kernel_smem_elems<HalfRows<C>, bf16_t, 1, 1, 1>()));
    n = max_of(n, max_of(kernel_smem_elems<HalfCols<C>, bf16_t, 1, 1, 1>(), kernel_smem_elems<ThreeQuarterRows<C>, bf16_t, 1, 1, 1>()));
  }
  return n;
}

// One operand tile of 4-bit weights, staged through registers: a piece is a block of 32 elements, 16 bytes of
// codes and a scale; a thread loads its pieces of a k-tile one k-tile ahead, and writes them as 4 x 16 bytes of bf16
// into the LDS tile, laid out as the direct loads of a bf16 operand would have left it (gemm.hpp), so the
// fragments are read the same way.  Each weight is converted once a workgroup.
// K-contiguous (KM false): R weight rows, two pieces of a 64-deep k-tile each.  K-major (KM true: the
// contraction runs over weight rows): 64 weight rows of R columns.
template <class C, int R, bool KM>
struct MxStager {
  static_assert(C::BK == 64 && (R % 32) == 0, "two blocks to a k-tile");
  static constexpr int PIECES = R * C::BK / kMxBlock;
  static constexpr int PER = (PIECES + C::THREADS - 1) / C::THREADS;
  static constexpr int CB = KM ? R / kMxBlock : C::BK / kMxBlock;  // pieces side by side
  rsrc_t rc, rs;
  int rows, blocks;  // valid rows and pieces side by side, from the tile's first (KM: rows run along the contraction)
  uint32_t ldc, lds_;  // bytes of a weight row
  u32x4 code[PER];
  uint32_t scale[PER];
  // codes, scales: the tile's first row and block; rows_valid rows and cols_valid elements from there
  MOE_DEV void init(const uint8_t* codes, const uint8_t* scales, int K, int rows_valid, int cols_valid) {
    ldc = (uint32_t)(K / 2);
    lds_ = (uint32_t)(K / kMxBlock);
    rows = rows_valid;
    blocks = cols_valid / kMxBlock;
    rc = make_rsrc(codes, (uint32_t)(rows - 1) * ldc + (uint32_t)blocks * 16);
    rs = make_rsrc(scales, (uint32_t)(rows - 1) * lds_ + (uint32_t)blocks);
  }
  MOE_DEV static void piece(int i, int& row, int& blk) {
    const int p = threadIdx.x + i * C::THREADS;
    row = p / CB;
    blk = p % CB;
  }
  // the k-tile from contraction index k0 on
  MOE_DEV void load(int k0) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int row, blk;
      piece(i, row, blk);
      const int r = KM ? k0 + row : row, b = KM ? blk : k0 / kMxBlock + blk;
      const bool in = r < rows && b < blocks && (PIECES % C::THREADS == 0 || threadIdx.x + i * C::THREADS < PIECES);
      code[i] = buf_ld16(rc, in ? (uint32_t)r * ldc + (uint32_t)b * 16 : kOobOffset, 0);
      scale[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, in ? (uint32_t)r * lds_ + (uint32_t)b : kOobOffset, 0, 0);
    }
  }
  MOE_DEV void write(bf16_t* tile) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (PIECES % C::THREADS != 0 && threadIdx.x + i * C::THREADS >= PIECES) break;
      int row, blk;
      piece(i, row, blk);
      const float s = mx_scale(scale[i]);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int slot = 4 * blk + v;
        bf16_t* to = KM ? tile + row * R + ((slot ^ tr_swz(row)) << 3)
                        : tile + row * C::BK + ((slot ^ nt_swz(row)) << 3);
        *reinterpret_cast<u32x4*>(to) = mx_bf16x8(code[i][v], s);
      }
    }
  }
};

// Behind a main loop that requests k-tiles past the last one: the zeros that these write have landed in every wave's part of
// the LDS, which the epilogue reuses (__syncthreads alone need not wait for direct loads).
MOE_DEV void direct_loads_done() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// acc += W-tile x A-tile over the contraction, A (bf16, K-contiguous) by direct-to-LDS loads as in
// mainloop_dma, W through MxStager.  Per k-tile kt: the pieces of kt + 1, loaded during kt - 1, are written
// to their stage (which was last read before the barrier that began kt), those of kt + 2 are requested, then
// the k-steps run as in mainloop_dma.  The wait before the barrier leaves at most the direct loads of later k-tiles
// outstanding, whatever the order in which the pieces' loads were issued among them.  One body serves all k-tiles (loads
// behind the last one bring zeros): with bodies of their own for the last k-tiles, hipcc keeps the sums of the scaled MFMAs
// (mainloop_mxmx) in two places and copies them at each k-tile, 100 to 400 spilled registers.
template <class C, bool KM>
MOE_DEV void mainloop_mx(f32x16 (&acc)[1][C::TN][C::TM], const OpDesc<bf16_t>& a, MxStager<C, C::BN, KM>& sb, int K,
                         bf16_t* smem) {
  using T = bf16_t;
  constexpr int TILE_A = C::BM * C::BK, TILE_B = C::BN * C::BK, STAGE = TILE_A + TILE_B;
  constexpr int NST = C::NST;
  static_assert(C::XR == 0, "no tall tiles");
  using SA = DmaStager<C, T, C::BM>;
  using SBN = DmaStager<C, T, C::BN>;
  using SBT = DmaStagerT<C, T, C::BN>;
  constexpr int IPT = SA::PER;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / C::WGN, wn = wave % C::WGN;
  const int nk = (K + C::BK - 1) / C::BK;
  if (nk <= 0) return;
  SA sa;
  sa.init(a, threadIdx.x);
  auto stage = [&](int kt) { return smem + (NST == 2 ? (kt & 1) : kt % NST) * STAGE; };
  auto issue = [&](int kt) {
#pragma unroll
    for (int i = 0; i < IPT; ++i) sa.issue_one(stage(kt), i, kt * C::BK, kt < nk);
  };
#pragma unroll
  for (int kt = 0; kt < NST - 1; ++kt) issue(kt);
  sb.load(0);
  sb.write(stage(0) + TILE_A);
  sb.load(C::BK);
  constexpr int KSTEPS = C::BK / (2 * C::V), LAST = KSTEPS - 1;
  static_assert(KSTEPS == 4, "two sets of fragments");
  const int frag_row = lane & 31, frag_kv = lane >> 5;
  u32x4 af[2][C::TM], bfr[2][C::TN];
  auto read_frags = [&](const T* sA, int ks, int set) {
    const T* sB = sA + TILE_A;
    const int kv = ks * 2 + frag_kv;
#pragma unroll
    for (int tm = 0; tm < C::TM; ++tm) af[set][tm] = SA::frag(sA, wm * C::WM + tm * 32 + frag_row, kv);
#pragma unroll
    for (int tn = 0; tn < C::TN; ++tn) {
      if constexpr (KM) bfr[set][tn] = SBT::frag(sB, wn * C::WN + tn * 32, ks * 2 * C::V);
      else bfr[set][tn] = SBN::frag(sB, wn * C::WN + tn * 32 + frag_row, kv);
    }
  };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  lds_barrier();
  issue(NST - 1);
  read_frags(smem, 0, 0);
  int kt = 0;
  do {
    sb.write(stage(kt + 1) + TILE_A);
    sb.load((kt + 2) * C::BK);
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      const int cur = ks & 1;
      if (ks < LAST) {
        read_frags(stage(kt), ks + 1, cur ^ 1);
      } else {
        asm volatile("s_waitcnt vmcnt(%0)" :: "n"((NST - 2) * IPT) : "memory");
        lds_barrier();
        read_frags(stage(kt + 1), 0, cur ^ 1);
      }
#pragma unroll
      for (int tn = 0; tn < C::TN; ++tn)
#pragma unroll
        for (int tm = 0; tm < C::TM; ++tm) mfma_frag(acc[0][tn][tm], bfr[cur][tn], af[cur][tm], T());
      if (ks == LAST) {
        issue(kt + NST);
        // as in mainloop_dma: the fragments' reads, then a direct load after each MFMA while they last
        constexpr int NM = C::TN * C::TM;
        __builtin_amdgcn_sched_group_barrier(0x100, C::TM + C::TN * (KM ? 2 : 1), 0);
#pragma unroll
        for (int i = 0; i < NM; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (i < IPT) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  } while (++kt < nk);
  direct_loads_done();
}

// Blocks from `tiles` on write the rows of no group.
template <typename T>
MOE_DEV bool mx_no_group(const MxRows& r, int tiles, const LinearEpi<T>& epi, int threads) {
  if ((int)blockIdx.x < tiles) return false;
  skinny_no_group(r.offsets, r.G, r.M, epi.N, (int64_t)blockIdx.x - tiles, (int64_t)gridDim.x - tiles, epi, threads);
  return true;
}

// y tile by tile, bf16 rows.  Bound by the main loop: 65536 rows in 128 experts, 4096 -> 1536, 840 us (982 TFLOP/s), 16384 in 16,
// 2048 -> 1408, 102 (926); a 64-deep k-tile of 256 x 256 takes 1.54 us in a long product, over bf16 weights 1.42 (a library product of
// 8192^3 runs at 1393 TFLOP/s), 1.05 of it matrix instructions.
template <class C>
__global__ __launch_bounds__(C::THREADS) void k_mx_fwd(const bf16_t* __restrict__ X, MxRows r, int tiles, MxWeights w,
                                                       LinearEpi<bf16_t> epi) {
  __shared__ __align__(16) bf16_t smem[mx_smem_elems<C>()];
  if (mx_no_group(r, tiles, epi, C::THREADS)) return;
  int grp, row0, mv, n0;
  const int N = w.N, K = w.K;
  if (!mx_tile<C::BM, C::BN>(r, N, (int)blockIdx.x, grp, row0, mv, n0)) return;
  const int64_t first = (int64_t)grp * N + n0;  // weight row
  with_mx_shape<C>(mv, N - n0, [&](auto ct) {
    using CT = decltype(ct);
    const OpDesc<bf16_t> a{X + (int64_t)row0 * K, K, mv, K};
    MxStager<CT, CT::BN, false> sb;
    sb.init(uni_ptr(w.codes + first * (K / 2)), uni_ptr(w.scales + first * (K / kMxBlock)), K, min(N - n0, CT::BN), K);
    f32x16 acc[1][CT::TN][CT::TM], none[1][CT::XTN];
    zero_acc<CT, 1>(acc);
    mainloop_mx<CT, false>(acc, a, sb, K, smem);
    static_assert(epi_lds_floats<CT, 1>() * 4 <= (int)sizeof(smem), "epilogue LDS");
    linear_epilogue<CT>(acc, none, epi, epi.bias ? epi.bias + first : nullptr, row0, mv, n0,
                        reinterpret_cast<float*>(smem));
  });
}

// dx = dz W tile by tile: the contraction runs over the weight's rows, which are read as transposed fragments.  For the products
// above 893 us (923 TFLOP/s) and 115.
template <class C>
__global__ __launch_bounds__(C::THREADS) void k_mx_dgrad(const bf16_t* __restrict__ dZ, MxRows r, int tiles, MxWeights w,
                                                         bf16_t* __restrict__ dX) {
  __shared__ __align__(16) bf16_t smem[mx_smem_elems<C>()];
  const int N = w.N, K = w.K;
  if (mx_no_group(r, tiles, LinearEpi<bf16_t>{nullptr, nullptr, dX, nullptr, kActNone, K}, C::THREADS)) return;
  int grp, row0, mv, k0;
  if (!mx_tile<C::BM, C::BN>(r, K, (int)blockIdx.x, grp, row0, mv, k0)) return;
  const int64_t first = (int64_t)grp * N;
  with_mx_shape<C>(mv, K - k0, [&](auto ct) {
    using CT = decltype(ct);
    const OpDesc<bf16_t> a{dZ + (int64_t)row0 * N, N, mv, N};
    MxStager<CT, CT::BN, true> sb;
    sb.init(uni_ptr(w.codes + first * (K / 2) + k0 / 2),
            uni_ptr(w.scales + first * (K / kMxBlock) + k0 / kMxBlock), K, N, min(K - k0, CT::BN));
    f32x16 acc[1][CT::TN][CT::TM];
    zero_acc<CT, 1>(acc);
    mainloop_mx<CT, true>(acc, a, sb, N, smem);
    for_each_row8<CT, 1>(acc, reinterpret_cast<float*>(smem), [&](int m, int n, auto& v) {
      if (m >= mv || k0 + n >= K) return;
      store8_stream(dX + ((int64_t)row0 + m) * K + k0 + n, v[0]);
    });
  });
}

// The element-wise part of a backward, as k_linear_dz and k_linear_db, their chunks found from the offsets: 12000 rows of
// 1368 in 12 groups 22 us and 4.8, where prefixes from a launch before them made 18 and 4.7 and cost 5.2 and a gap (the whole forward
// and backward 188 -> 176).  98 MB of reading dy and z and writing dz take 19 at a copy's rate; the scan, and a thread's two rows one
// behind the other, are the rest.  chunks: those that `part` holds.
static __global__ __launch_bounds__(256) void k_mx_dz(const bf16_t* __restrict__ dY, const bf16_t* __restrict__ pre, int act,
                                                      MxRows r, int N, bf16_t* __restrict__ dZ, float* __restrict__ part) {
  const int chunk = blockIdx.x;
  if (!r.offsets) return dz_chunk(dY, pre, act, chunk, chunk * kDzRows, min(kDzRows, r.M - chunk * kDzRows), N, dZ, part);
  const MxTileScan<kDzRows> scan(r);
  if (chunk >= scan.total) return;
  int r0 = 0, rows = 0;
  scan.walk(scan.lane_of(chunk), [&](int, int first, int c, int a, int b) {
    if (chunk >= first + c) return false;
    r0 = a + (chunk - first) * kDzRows;
    rows = min(kDzRows, b - r0);
    return true;
  });
  dz_chunk(dY, pre, act, chunk, r0, rows, N, dZ, part);
}
static __global__ __launch_bounds__(256) void k_mx_db(const float* __restrict__ part, MxRows r, int chunks, int N,
                                                      bf16_t* __restrict__ db) {
  const int grp = blockIdx.y;
  int p0 = 0, p1 = chunks;
  if (r.offsets) {
    const MxTileScan<kDzRows> scan(r);
    scan.walk(grp / scan.per, [&](int e, int first, int c, int, int) {
      p0 = min(first, chunks);
      p1 = min(first + c, chunks);
      return e == grp;
    });
  }
  db_columns(part, grp, p0, p1, N, db);
}

// ------------------------------------------------------------------ tiled products, both sides in 4 bits
// A 16-byte vector is 32 elements, so a k-tile of 64 bf16's bytes is 256 elements and the tilings, direct
// loads, swizzles and fragments of gemm.hpp serve as they are, over rows of K / 4 two-byte units.
// v_mfma_scale_f32_32x32x64_f8f6f4 takes such a vector of each operand and a scale for each.  Half h of a
// wave reads vector 4 h + ks in k-step ks of a k-tile instead of 2 ks + h: its four scales of a row are then one dword,
// of which step ks takes byte ks.
MOE_DEV void mfma_mx(f32x16& acc, u32x4 bt, u32x4 at, uint32_t sb, uint32_t sa, int ks) {
  typedef int i32x8 __attribute__((ext_vector_type(8)));
  const i32x8 b = {(int)bt.x, (int)bt.y, (int)bt.z, (int)bt.w, 0, 0, 0, 0};
  const i32x8 a = {(int)at.x, (int)at.y, (int)at.z, (int)at.w, 0, 0, 0, 0};
  switch (ks) {  // a constant
    case 0: acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc, 4, 4, 0, (int)sb, 0, (int)sa); break;
    case 1: acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc, 4, 4, 1, (int)sb, 1, (int)sa); break;
    case 2: acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc, 4, 4, 2, (int)sb, 2, (int)sa); break;
    default: acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc, 4, 4, 3, (int)sb, 3, (int)sa); break;
  }
}

// The scales of a tile's rows (BM of x, then BN of the weight), through registers: a thread loads 16 of each of its
// rows at once, those of two k-tiles (rows of K / 32 bytes have any alignment, and a k-tile's few bytes of a cache line
// would fetch each line many times), and writes a k-tile's, eight, to LDS.  No branch is between a load and its
// use, or it would be waited for at once: a load that would leave the tensor (its last 15 bytes) is moved back into it and
// shifted, and what is not the row's is masked.  A wave's 64 rows are all of one operand's, so its base is scalar.
// Both tensors hold 16 bytes at least.
template <class C>
struct MxScaleStager {
  static constexpr int ROWS = C::BM + C::BN;
  static constexpr int PER = (ROWS + C::THREADS - 1) / C::THREADS;
  static_assert(C::BM % 64 == 0 && C::BN % 64 == 0, "a wave's rows are of one operand");
  static_assert(C::BK == 8 * C::V, "eight blocks to a k-tile's row");
  const __attribute__((address_space(1))) uint8_t* base[PER];
  uint32_t last[PER];   // the last 16 bytes of the tensor, from base
  uint32_t row[PER];    // the thread's row, from base
  int bytes, valid;     // of a row; bit i: row i exists
  u32x4 s[PER];
  int at;               // where s begins in a row
  // xs, ws: the tensors; the tile's rows from x0 (mv of them) and w0 (nv)
  MOE_DEV void init(const uint8_t* xs, const uint8_t* ws, int64_t x0, int64_t w0, int64_t xrows, int64_t wrows, int mv, int nv,
                    int K) {
    bytes = K / kMxBlock;
    valid = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = uni((threadIdx.x & ~63) + i * C::THREADS), lane = threadIdx.x & 63;
      const bool a = r < C::BM;
      // a wave past the tile's rows stays at its first
      const int64_t first = a ? (r < mv ? x0 + r : x0) : (r - C::BM < nv ? w0 + r - C::BM : w0);
      const int left = a ? mv - r : nv - (r - C::BM);
      base[i] = gptr(uni_ptr((a ? xs : ws) + first * bytes));
      last[i] = (uint32_t)min(((a ? xrows : wrows) - first) * bytes - 16, (int64_t)INT_MAX);
      if (r < ROWS && lane < left) valid |= 1 << i;
      row[i] = (uint32_t)(lane * bytes);
    }
  }
  MOE_DEV void load(int from) {
    at = from;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      typedef u32x4 any_u32x4 __attribute__((aligned(1)));
      s[i] = *(const __attribute__((address_space(1))) any_u32x4*)(base[i] + (int64_t)min((int)(row[i] + at), (int)last[i]));
    }
  }
  // the scales of k-tile kt, the load's first half or (kt odd) its second
  MOE_DEV void write(uint32_t* tile, int kt) const {
    const int j = kt & 1, left = bytes - at - 8 * j;  // bytes of the row from here
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = threadIdx.x + i * C::THREADS;
      if (ROWS % C::THREADS != 0 && r >= ROWS) break;
      const int d = max((int)(row[i] + at) - (int)last[i], 0);  // bytes moved back
      u32x4 v = s[i];
      if (__builtin_expect(__any(d > 0), 0)) {
        if (d & 8) v = u32x4{v.z, v.w, 0, 0};
        if (d & 4) v = u32x4{v.y, v.z, v.w, 0};
        const int b = 8 * (d & 3);
        v = u32x4{(uint32_t)((((uint64_t)v.y << 32) | v.x) >> b), (uint32_t)((((uint64_t)v.z << 32) | v.y) >> b),
                  (uint32_t)((((uint64_t)v.w << 32) | v.z) >> b), v.w >> b};
        if (d >= 16) v = u32x4{0, 0, 0, 0};
      }
      const bool in = valid >> i & 1;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t q = w ? (j ? v.w : v.y) : (j ? v.z : v.x);
        const int n = left - 4 * w;
        q &= n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
        tile[2 * r + w] = in ? q : 0u;
      }
    }
  }
};

// As mainloop_dma, with scales.  A k-tile of 256 x 256 x 256 takes some 2.1 us: 1.13 of matrix instructions at their rate from registers
// (7.6 PFLOP/s), 1.4 to 1.7 with the fragments' reads and no direct loads, the rest for those (64 KB into LDS), which are waited
// for in every k-tile (below).  65536 rows in 128
// experts, 4096 -> 1536, 343 us (2.4 PFLOP/s): with the next k-tile requested only behind the last k-step 392; k-tiles half as deep in
// four stages 393 -> 439.  OUT, the results' type, only sets the instantiations of two kernels apart: hipcc's host
// pass takes the second use of one as an error.
template <class C, typename OUT>
MOE_DEV void mainloop_mxmx(f32x16 (&acc)[1][C::TN][C::TM], const OpDesc<bf16_t>& a, const OpDesc<bf16_t>& b,
                           MxScaleStager<C>& ss, int K4, bf16_t* smem, uint32_t* scales) {
  using T = bf16_t;
  constexpr int TILE_A = C::BM * C::BK, TILE_B = C::BN * C::BK, STAGE = TILE_A + TILE_B;
  constexpr int NST = C::NST, ROWS = MxScaleStager<C>::ROWS;
  static_assert(C::XR == 0, "no tall tiles");
  using SA = DmaStager<C, T, C::BM>;
  using SB = DmaStager<C, T, C::BN>;
  constexpr int IPT = SA::PER + SB::PER;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / C::WGN, wn = wave % C::WGN;
  const int nk = (K4 + C::BK - 1) / C::BK;
  if (nk <= 0) return;
  SA sa;
  SB sb;
  sa.init(a, threadIdx.x);
  sb.init(b, threadIdx.x);
  auto stage = [&](int kt) { return smem + (NST == 2 ? (kt & 1) : kt % NST) * STAGE; };
  auto scales_of = [&](int kt) { return scales + (kt & 1) * ROWS * 2; };
  auto issue = [&](int kt, int i) {
    if (i < SA::PER) sa.issue_one(stage(kt), i, kt * C::BK, kt < nk);
    else sb.issue_one(stage(kt) + TILE_A, i - SA::PER, kt * C::BK, kt < nk);
  };
#pragma unroll
  for (int kt = 0; kt < NST - 1; ++kt)
#pragma unroll
    for (int i = 0; i < IPT; ++i) issue(kt, i);
  ss.load(0);
  ss.write(scales_of(0), 0);
  constexpr int KSTEPS = C::BK / (2 * C::V), M = KSTEPS - 1;
  static_assert(KSTEPS == 4, "a lane's scales of a row: a dword");
  const int frag_row = lane & 31, half = lane >> 5;
  // one set of fragments of the weight: each is read again for the next k-step behind its last MFMA (two sets of both
  // operands spill beside the scales)
  u32x4 af[2][C::TM], bfr[C::TN];
  uint32_t as[C::TM], bs[C::TN];
  auto read_scales = [&](int kt) {
    const uint32_t* t = scales_of(kt) + half;
#pragma unroll
    for (int tm = 0; tm < C::TM; ++tm) as[tm] = t[2 * (wm * C::WM + tm * 32 + frag_row)];
#pragma unroll
    for (int tn = 0; tn < C::TN; ++tn) bs[tn] = t[2 * (C::BM + wn * C::WN + tn * 32 + frag_row)];
  };
  auto read_a = [&](const T* st, int ks, int set) {
#pragma unroll
    for (int tm = 0; tm < C::TM; ++tm) af[set][tm] = SA::frag(st, wm * C::WM + tm * 32 + frag_row, KSTEPS * half + ks);
  };
  auto read_b = [&](const T* st, int ks, int tn) {
    bfr[tn] = SB::frag(st + TILE_A, wn * C::WN + tn * 32 + frag_row, KSTEPS * half + ks);
  };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  lds_barrier();
#pragma unroll
  for (int i = 0; i < IPT; ++i) issue(NST - 1, i);
  read_a(smem, 0, 0);
#pragma unroll
  for (int tn = 0; tn < C::TN; ++tn) read_b(smem, 0, tn);
  read_scales(0);
  int kt = 0;
  do {
    // the next k-tile's scales, of a load that ended before this k-tile or began with the one before it
    ss.write(scales_of(kt + 1), kt + 1);
    if ((kt & 1) == 0) ss.load((kt + 2) * (C::BK / C::V));
    auto products = [&](int ks, int tn) {
#pragma unroll
      for (int tm = 0; tm < C::TM; ++tm) mfma_mx(acc[0][tn][tm], bfr[tn], af[ks & 1][tm], bs[tn], as[tm], ks);
    };
#pragma unroll
    for (int ks = 0; ks < M; ++ks) {
      read_a(stage(kt), ks + 1, (ks + 1) & 1);
#pragma unroll
      for (int tn = 0; tn < C::TN; ++tn) {
        products(ks, tn);
        read_b(stage(kt), ks + 1, tn);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // Last k-step, whose fragments are read.  Behind a first barrier no wave reads this k-tile's stage again, and
    // its refill is issued over the first half of the step's products; behind a second one the next k-tile has landed,
    // whose refill was issued a k-tile ago.  The counted wait would leave the refill in flight, but with the scales in an
    // LDS array of their own hipcc puts a vmcnt(0) before the next k-tile's first fragment: the refill is waited for in
    // full half a k-step behind its issue, and further stages hide nothing.
    constexpr int H = (C::TN + 1) / 2;
    lds_barrier();
#pragma unroll
    for (int tn = 0; tn < H; ++tn) {
      products(M, tn);
#pragma unroll
      for (int i = tn * IPT / H; i < (tn + 1) * IPT / H; ++i) issue(kt + NST, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"((NST - 1) * IPT) : "memory");
    lds_barrier();
    read_a(stage(kt + 1), 0, 0);
#pragma unroll
    for (int tn = 0; tn < H; ++tn) read_b(stage(kt + 1), 0, tn);
#pragma unroll
    for (int tn = H; tn < C::TN; ++tn) {
      products(M, tn);
      read_b(stage(kt + 1), 0, tn);
      __builtin_amdgcn_sched_barrier(0);
    }
    read_scales(kt + 1);
  } while (++kt < nk);
  direct_loads_done();
}

template <class C, typename T>
__global__ __launch_bounds__(C::THREADS, 2) void k_mxmx_fwd(const uint8_t* __restrict__ X, const uint8_t* __restrict__ XS,
                                                         MxRows r, int tiles, MxWeights w, LinearEpi<T> epi) {
  __shared__ __align__(16) bf16_t smem[mx_smem_elems<C>()];
  __shared__ uint32_t scales[2 * (C::BM + C::BN) * 2];
  if (mx_no_group(r, tiles, epi, C::THREADS)) return;
  int grp, row0, mv, n0;
  const int N = w.N, K = w.K, K4 = K / 4;
  if (!mx_tile<C::BM, C::BN>(r, N, (int)blockIdx.x, grp, row0, mv, n0)) return;
  const int64_t first = (int64_t)grp * N + n0;
  with_mx_shape<C>(mv, N - n0, [&](auto ct) {
    using CT = decltype(ct);
    static_assert(CT::BM <= C::BM && CT::BN <= C::BN, "scales' LDS");
    const OpDesc<bf16_t> a{reinterpret_cast<const bf16_t*>(X + (int64_t)row0 * (K / 2)), K4, mv, K4};
    const OpDesc<bf16_t> b{reinterpret_cast<const bf16_t*>(w.codes + first * (K / 2)), K4, N - n0, K4};
    MxScaleStager<CT> ss;
    ss.init(XS, w.scales, row0, first, r.M, (int64_t)r.G * N, mv, N - n0, K);
    f32x16 acc[1][CT::TN][CT::TM], none[1][CT::XTN];
    zero_acc<CT, 1>(acc);
    mainloop_mxmx<CT, T>(acc, a, b, ss, K4, smem, scales);
    static_assert(epi_lds_floats<CT, 1>() * 4 <= (int)sizeof(smem), "epilogue LDS");
    linear_epilogue<CT>(acc, none, epi, epi.bias ? epi.bias + first : nullptr, row0, mv, n0,
                        reinterpret_cast<float*>(smem));
  });
}

// ------------------------------------------------------------------ few rows
// As in k_linear_skinny a launch with few rows to an expert is the stream of the weights that it touches: a wave
// multiplies RW blocks of 16 weight rows with 16 rows of the expert straight from memory (an expert's further rows are
// other workgroups', which find the weight in the caches; 64 rows to a workgroup took 40 to 90 registers more and 10 to 60 % longer),
// KS waves of a workgroup share the weight rows and take every KS-th k-chunk of 512 elements (1024: as many registers
// too many, 20 to 100 % longer).  Lane l supplies block l / 16 + 4 q of weight row l % 16 in load q, so four lanes read
// 64 contiguous bytes.  The four lanes of a row load the scales of four chunks of it, 16 bytes each, and every
// chunk's are handed round (ds_bpermute): with each lane loading its chunk's 16 the cache lines of scales were fetched again for each
// chunk, 96 us instead of 86 below (a load for each byte: 10 % more).
// bf16 rows: the block becomes four 8-element vectors, multiplied with the four of the token row by 16 x 16 x 32 MFMAs; the row's
// next four are requested before (3 %).  4-bit rows: one 16 x 16 x 128 scaled MFMA.
// Bound by HBM where the weights outgrow the caches: 512 rows in 128 experts of 1536 x 4096 (428 MB) 86 us over bf16 rows (5.0 TB/s;
// fewer rows to a wave or registers for more waves of them: 91 to 148) and 70 over 4-bit ones (6.1; with the nontemporal hint on the
// weights a tenth more in both); 64 rows in them 38 and 29.  Bound by a launch and one chain of loads otherwise: one row of 4096 x
// 4096 4.6 and 4.0.

constexpr int kMxSkinnyRows = 16;
constexpr int kMxChunkLoads = 4;  // of 128 elements
// Scales of a wave's next four chunks: lane 16 c + rl holds the 16 of chunk c of its row, from p on; `left` of them are in the row.
template <typename V>
MOE_DEV V ld_any(const uint8_t* p) {  // of any alignment
  typedef V any_v __attribute__((aligned(1)));
  return *(const __attribute__((address_space(1))) any_v*)p;
}
MOE_DEV u32x4 mx_row_scales(const uint8_t* p, int left) {
  u32x4 v{0, 0, 0, 0};
  if (left >= 16) {
    v = ld_any<u32x4>(p);
  } else if (left > 0) {  // 8, 4, 2 and 1 of them
    const uint64_t a = left & 8 ? ld_any<uint64_t>(p) : 0;
    const uint32_t b = left & 4 ? ld_any<uint32_t>(p + (left & 8)) : 0;
    const uint32_t c = left & 2 ? ld_any<uint16_t>(p + (left & 12)) : 0;
    const uint32_t d = left & 1 ? gptr(p)[left & 14] : 0;
    const uint64_t rest = b | (uint64_t)(c | d << 8 * (left & 2)) << 8 * (left & 4);
    const uint64_t lo = left & 8 ? a : rest, hi = left & 8 ? rest : 0;
    v = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
  return v;
}
// Chunk c's, as the lanes of block l / 16 of each load take them: byte l / 16 of its dword, in the lowest byte.
MOE_DEV void mx_chunk_scales(const u32x4& held, int c, uint32_t (&s)[kMxChunkLoads]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int q = 0; q < kMxChunkLoads; ++q)
    s[q] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (16 * c + (lane & 15)), (int)held[q]) >> (8 * (lane >> 4));
}

template <bool X4, typename T, int KS, int RW>
__global__ __launch_bounds__(256) void k_mx_skinny(const void* __restrict__ X, const uint8_t* __restrict__ XS,
                                                   const int* __restrict__ offsets, int E, int M, int nslot,
                                                   MxWeights w, LinearEpi<T> epi) {
  constexpr int RB = 4 / KS, ROWS = 16 * RW, Q = kMxChunkLoads, KC = 128 * Q;
  typedef int i32x8 __attribute__((ext_vector_type(8)));
  __shared__ f32x4 red[(KS - 1) * RB * RW * 64];
  const int N = w.N, K = w.K;
  const int nNb = (N + ROWS * RB - 1) / (ROWS * RB);
  const int slot = uni(blockIdx.x / nNb), nb = uni(blockIdx.x % nNb);
  if (slot >= nslot) {
    skinny_no_group(offsets, E, M, N, (int64_t)blockIdx.x - (int64_t)nslot * nNb,
                    (int64_t)gridDim.x - (int64_t)nslot * nNb, epi);
    return;
  }
  int grp = 0, r0 = slot * kMxSkinnyRows, rows = min(kMxSkinnyRows, M - r0);
  if (offsets && !skinny_slot<kMxSkinnyRows>(offsets, E, M, slot, grp, r0, rows)) return;  // workgroup-uniform
  grp = uni(grp); r0 = uni(r0); rows = uni(rows);
  const int wave = uni(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int rb = wave / KS, ks = wave % KS;
  const int n0 = (nb * RB + rb) * ROWS;
  const int nrows = uni(min(ROWS, N - n0));
  const int g = lane >> 4, rl = lane & 15;
  const int bytes = K / 2, blocks = K / kMxBlock;
  f32x4 acc[RW];
#pragma unroll
  for (int i = 0; i < RW; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (nrows > 0) {
    const int xb = X4 ? bytes : 2 * K;  // bytes of a token row
    const rsrc_t rx = make_rsrc(uni_ptr((const uint8_t*)X + (int64_t)r0 * xb), (uint32_t)uni(rows * xb));
    const int64_t first = (int64_t)grp * N + n0;
    const rsrc_t rw = make_rsrc(uni_ptr(w.codes + first * bytes), (uint32_t)uni(nrows * bytes));
    const uint8_t* wscales = uni_ptr(w.scales + first * blocks);
    uint32_t vw[RW];
#pragma unroll
    for (int i = 0; i < RW; ++i) vw[i] = 16 * i + rl < nrows ? (uint32_t)((16 * i + rl) * bytes + 16 * g) : kOobOffset;
    const uint32_t vx = rl < rows ? (uint32_t)(rl * xb + (X4 ? 16 : 64) * g) : kOobOffset;
    u32x4 ws_held[RW], xs_held;
    auto chunk = [&](int kc, int at, auto full_c) {  // at: of the four whose scales are held
      constexpr bool FULL = decltype(full_c)::value;
      const int b0 = kc * 4 * Q, left = blocks - b0;  // blocks
      u32x4 wa[RW][Q];
      uint32_t ws[RW][Q];
#pragma unroll
      for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const bool in = FULL || 4 * q + g < left;
          wa[i][q] = buf_ld16(rw, in ? vw[i] + 64 * q : kOobOffset, (uint32_t)b0 * 16);
        }
#pragma unroll
      for (int i = 0; i < RW; ++i) mx_chunk_scales(ws_held[i], at, ws[i]);
      if constexpr (X4) {
        u32x4 xa[Q];
        uint32_t xs[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const bool in = FULL || 4 * q + g < left;
          xa[q] = buf_ld16(rx, in ? vx + 64 * q : kOobOffset, (uint32_t)b0 * 16);
        }
        mx_chunk_scales(xs_held, at, xs);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const i32x8 av = {(int)xa[q].x, (int)xa[q].y, (int)xa[q].z, (int)xa[q].w, 0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            const u32x4 v = wa[i][q];
            const i32x8 bv = {(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
            acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, acc[i], 4, 4, 0, (int)xs[q], 0, (int)ws[i][q]);
          }
        }
      } else {
        u32x4 xa[2][4];  // the rows of one load of the weight, and of the next, requested before that is multiplied
        auto load_x = [&](int q) {
          const bool in = FULL || 4 * q + g < left;
#pragma unroll
          for (int v = 0; v < 4; ++v) xa[q & 1][v] = buf_ld16(rx, in ? vx + 256 * q + 16 * v : kOobOffset, (uint32_t)b0 * 64);
          __builtin_amdgcn_sched_barrier(0);
        };
        load_x(0);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          if (q + 1 < Q) load_x(q + 1);
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            const float s = mx_scale(ws[i][q] & 255u);
#pragma unroll
            for (int v = 0; v < 4; ++v) mfma16(acc[i], xa[q & 1][v], mx_bf16x8(wa[i][q][v], s));
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    int kc = ks, at = 0;
    auto hold = [&] {
      const int b = (kc + g * KS) * 4 * Q, left = blocks - b;  // of the chunk whose scales this lane holds
#pragma unroll
      for (int i = 0; i < RW; ++i)  // rows past the weight's hold its first row's scales (their codes are zeros)
        ws_held[i] = mx_row_scales(wscales + (int64_t)(16 * i + rl < nrows ? 16 * i + rl : 0) * blocks + b, left);
      if constexpr (X4) xs_held = mx_row_scales(XS + ((int64_t)r0 + (rl < rows ? rl : 0)) * blocks + b, left);
    };
    hold();
#pragma unroll 1
    for (; (kc + 1) * KC <= K; kc += KS) {
      if (at == 4) {
        at = 0;
        hold();
      }
      chunk(kc, at++, std::true_type());
    }
    if (kc * KC < K) {
      if (at == 4) {
        at = 0;
        hold();
      }
      chunk(kc, at, std::false_type());
    }
  }
  if (ks > 0) {
#pragma unroll
    for (int i = 0; i < RW; ++i) red[(((ks - 1) * RB + rb) * RW + i) * 64 + lane] = acc[i];
  }
  __syncthreads();
  if (ks > 0) return;
#pragma unroll
  for (int q = 1; q < KS; ++q)
#pragma unroll
    for (int i = 0; i < RW; ++i) acc[i] += red[(((q - 1) * RB + rb) * RW + i) * 64 + lane];
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const f32x4 one[1] = {acc[i]};
    if (16 * i + rl < nrows) skinny_store<T, 1>(epi, one, 1, r0, rows, n0 + 16 * i + rl, grp);
  }
}

}  // namespace moe
