// A stand-in for the HIP runtime that runs kernels on the CPU, one workgroup at a time, for checks
// of their addresses: every thread is a coroutine that yields at barriers and at operations
// across a wave.  Loads and stores go to host memory, so AddressSanitizer sees each of them, LDS
// arrays are static, buffer loads are checked against their resource and against what they
// reach.  Matrix instructions change nothing: no address depends on a product.
#pragma once
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <algorithm>
#include <climits>
#include <cmath>
#include <functional>
#include <type_traits>

#define __global__
#define __device__
#define __host__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __align__(n) __attribute__((aligned(n)))
#define __shared__ static
#define __restrict__
#define address_space(n) unused
#define amdgpu_waves_per_eu(n) unused

struct dim3 {
  unsigned x, y, z;
  dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {}
};
extern dim3 threadIdx, blockIdx, blockDim, gridDim;

typedef int hipError_t;
typedef void* hipStream_t;
enum { hipSuccess = 0, hipErrorOutOfMemory = 2, hipErrorInvalidConfiguration = 9 };
inline const char* hipGetErrorString(hipError_t) { return "emulated"; }
inline hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
inline hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError();

namespace emu {
void barrier();
// The values of a wave's lanes (0 for lanes that have ended), once each live lane has given its own.
const uint64_t* exchange(uint64_t v, uint64_t* live = nullptr);
void run(const char* name, dim3 grid, dim3 block, size_t lds, const std::function<void()>& f);
void* dynamic_lds();
[[noreturn]] void die(const char* what, long long a = 0, long long b = 0);
void touch(const void* p, size_t n, bool write);  // dies unless [p, p + n) may be accessed
void count_store(const void* p);
inline int lane() { return threadIdx.x & 63; }

struct Rsrc {
  const char* base;
  uint32_t bytes;
};
// A byte is in range when its offset from the base is below the resource's size; what is in range has to
// be memory.  The scalar offset stays within the resource, or the comparison would wrap.
inline const void* buffer_at(const Rsrc& r, uint32_t voff, uint32_t soff, unsigned n) {
  if (soff > r.bytes) die("scalar offset beyond the resource", soff, r.bytes);
  const uint32_t left = r.bytes - soff;
  if (voff >= left) return nullptr;
  const char* p = r.base + (uint64_t)voff + soff;
  touch(p, std::min<uint64_t>(n, left - voff), false);
  return voff + (uint64_t)n <= left ? p : nullptr;
}
template <class V> V load(const Rsrc& r, uint32_t voff, uint32_t soff) {
  V v;
  memset(&v, 0, sizeof v);
  if (const void* p = buffer_at(r, voff, soff, sizeof v)) memcpy(&v, p, sizeof v);
  return v;
}
inline void load_lds(const Rsrc& r, void* lds, unsigned n, uint32_t voff, uint32_t soff) {
  char* to = (char*)lds + lane() * n;
  touch(to, n, true);
  buffer_at(r, voff, soff, n);
}
template <class P, class V> void nt_store(V v, P* p) {
  count_store((const void*)p);
  *p = v;
}
template <class T> uint64_t bits(T v) {
  uint64_t b = 0;
  memcpy(&b, &v, sizeof v);
  return b;
}
template <class T> T from(uint64_t b) {
  T v;
  memcpy(&v, &b, sizeof v);
  return v;
}
template <class T> T of_lane(T v, int from_lane) { return from<T>(exchange(bits(v))[from_lane & 63]); }
// Of the patterns that the kernels use: shifts right by n in a row of 16, and rows' last lanes
// broadcast to the rows above; bound_ctrl and masked rows keep `old`.
inline int dpp(int old, int v, int ctrl, int row_mask, int bank_mask, bool bound) {
  const uint64_t* all = exchange(bits(v));
  const int l = lane(), row = l >> 4, at = l & 15;
  int src = -1;
  if (ctrl >= 0x111 && ctrl <= 0x11f) src = at >= (ctrl & 15) ? l - (ctrl & 15) : -1;
  else if (ctrl >= 0x101 && ctrl <= 0x10f) src = at + (ctrl & 15) < 16 ? l + (ctrl & 15) : -1;
  else if (ctrl >= 0x121 && ctrl <= 0x12f) src = (l & ~15) | ((at - (ctrl & 15)) & 15);
  else if (ctrl == 0x142) src = row > 0 ? row * 16 - 1 : -1;
  else if (ctrl == 0x143) src = l >= 32 ? 31 : -1;
  else if (ctrl < 0x100) src = (l & ~3) | ((ctrl >> (2 * (l & 3))) & 3);
  else die("an unknown lane pattern", ctrl);
  if (!((row_mask >> row) & 1) || !((bank_mask >> ((l & 15) >> 2)) & 1)) return old;
  return src >= 0 ? from<int>(all[src]) : bound ? 0 : old;
}
struct Pair {
  unsigned v[2];
  unsigned operator[](int i) const { return v[i]; }
};
template <int D> Pair swap_halves(unsigned a, unsigned b) {
  // lanes with bit D clear keep a and take the partner's a into b; the others the other way about
  const unsigned pa = from<unsigned>(exchange(bits(a))[lane() ^ D]), pb = from<unsigned>(exchange(bits(b))[lane() ^ D]);
  return lane() & D ? Pair{{pb, b}} : Pair{{a, pa}};
}
}  // namespace emu

#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) \
  emu::run(#kernel, grid, block, lds, [=] { kernel(__VA_ARGS__); })

#define __syncthreads() emu::barrier()
#define __amdgpu_buffer_rsrc_t emu::Rsrc
#define __builtin_amdgcn_make_buffer_rsrc(p, stride, n, flags) (emu::Rsrc{(const char*)(p), (uint32_t)(n)})
#define __builtin_amdgcn_raw_buffer_load_b128(r, v, s, aux) emu::load<u32x4>(r, v, s)
#define __builtin_amdgcn_raw_buffer_load_b32(r, v, s, aux) emu::load<uint32_t>(r, v, s)
#define __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, n, v, s, inst, aux) emu::load_lds(r, (void*)(lds), n, v, s)
#define __builtin_amdgcn_ds_read_tr16_b64_v4i16(p) (*(p))
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, x, y, z) (c)
#define __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, x, y, z) (c)
#define __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, x, y, z) (c)
#define __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, x, y, z) (c)
#define __builtin_amdgcn_fence(...) ((void)0)
#define __builtin_amdgcn_wave_barrier() ((void)emu::exchange(0))
#define __builtin_amdgcn_sched_barrier(n) ((void)0)
#define __builtin_amdgcn_sched_group_barrier(a, b, c) ((void)0)
#define __builtin_amdgcn_rcpf(x) (1.0f / (x))
#define __builtin_amdgcn_readfirstlane(v) (v)  // the kernels give it wave-uniform values
#define __builtin_amdgcn_readlane(v, l) emu::of_lane((int)(v), l)
#define __builtin_amdgcn_update_dpp(o, v, c, r, b, bc) emu::dpp(o, v, c, r, b, bc)
#define __builtin_amdgcn_permlane32_swap(a, b, x, y) emu::swap_halves<32>(a, b)
#define __builtin_amdgcn_permlane16_swap(a, b, x, y) emu::swap_halves<16>(a, b)
#define __builtin_nontemporal_store(v, p) emu::nt_store(v, p)
#define __builtin_nontemporal_load(p) (*(p))

inline uint64_t __ballot(bool on) {
  uint64_t live, m = 0;
  const uint64_t* all = emu::exchange(on, &live);
  for (int i = 0; i < 64; ++i) m |= (all[i] & (live >> i) & 1) << i;
  return m;
}
template <class T> T __shfl(T v, int l, int = 64) { return emu::of_lane(v, l); }
template <class T> T __shfl_up(T v, int d, int = 64) {
  return emu::of_lane(v, emu::lane() >= d ? emu::lane() - d : emu::lane());
}
inline int __popcll(uint64_t v) { return __builtin_popcountll(v); }
inline int __popc(uint32_t v) { return __builtin_popcount(v); }
inline int __clz(int v) { return v ? __builtin_clz(v) : 32; }
inline int __ffsll(unsigned long long v) { return __builtin_ffsll(v); }
inline float __uint_as_float(uint32_t v) { return emu::from<float>(v); }
inline float __int_as_float(int v) { return emu::from<float>((uint32_t)v); }
inline uint32_t __float_as_uint(float v) { return emu::bits(v); }
inline int __float_as_int(float v) { return (int)emu::bits(v); }
using std::isnan;
using std::isinf;
inline float __expf(float v) { return expf(v); }
template <class T> T atomicAdd(T* p, T v) {
  T o = *p;
  *p = o + v;
  return o;
}
template <class T> T atomicOr(T* p, T v) {
  T o = *p;
  *p = o | v;
  return o;
}
template <class A, class B> typename std::common_type<A, B>::type min(A a, B b) {
  typedef typename std::common_type<A, B>::type C;
  return (C)b < (C)a ? (C)b : (C)a;
}
template <class A, class B> typename std::common_type<A, B>::type max(A a, B b) {
  typedef typename std::common_type<A, B>::type C;
  return (C)a < (C)b ? (C)b : (C)a;
}
