// C ABI of the router's losses.  Declared in include/moe_hip.h.  The calls keep no state.
#include <cfloat>

#include "entry.hpp"
#include "router.hpp"

using namespace moe;

namespace {

moe_status check_router(int dtype, int64_t T, int E, int k, int index_bytes, int score, float tau, bool offsets, int64_t S) {
  moe_status st = check_dtype(dtype);
  if (st != MOE_OK) return st;
  if (T < 0 || T >= (int64_t(1) << 31)) return fail(MOE_ERR_INVALID, "num_tokens is outside 0..2^31-1");
  if (k < 1 || k > 16) return fail(MOE_ERR_INVALID, "experts_per_tok %d is outside 1..16", k);
  if (E < 1 || E > 1024) return fail(MOE_ERR_INVALID, "num_experts %d is outside 1..1024", E);
  if (T * k >= int64_t(1) << 31)
    return fail(MOE_ERR_UNSUPPORTED, "num_tokens x experts_per_tok reaches 2^31");
  if (index_bytes != 4 && index_bytes != 8)
    return fail(MOE_ERR_INVALID, "index_bytes %d is neither 4 nor 8", index_bytes);
  if (score != kScoreSoftmax && score != kScoreSigmoid) return fail(MOE_ERR_INVALID, "unknown score %d", score);
  // the kernels multiply by log2(e) / tau
  if (!(tau >= FLT_MIN) || !std::isfinite(tau))
    return fail(MOE_ERR_INVALID, "temperature must be positive (at least 2^-126) and finite");
  if (offsets ? S < 0 : S != 1)
    return fail(MOE_ERR_INVALID, offsets ? "num_sequences is negative" : "num_sequences without offsets is not 1");
  if (S >= int64_t(1) << 22) return fail(MOE_ERR_UNSUPPORTED, "num_sequences reaches 2^22");
  return MOE_OK;
}

// Calls f(shape) of the narrowest wave shape that holds E columns.  A width inside a step costs up to a sixth more an
// element than at its end: 65536 rows of 160, 192 and 256 bf16 sigmoid scores 17, 22 and 25 us forward and 23, 31 and 34 back,
// of 256, 384 and 512 25, 40 and 45, and 34, 51 and 56 (fp32 softmax 15, 22 and 25, and 28, 38 and 48).
template <class F>
void with_router_shape(int E, F&& f) {
  if (E % 4 == 0) {
    if (E <= 16) f(RouterShape<4, 4, 1>());
    else if (E <= 32) f(RouterShape<4, 4, 2>());
    else if (E <= 64) f(RouterShape<4, 4, 4>());
    else if (E <= 96) f(RouterShape<4, 8, 3>());
    else if (E <= 128) f(RouterShape<4, 8, 4>());
    else if (E <= 160) f(RouterShape<4, 8, 5>());
    else if (E <= 256) f(RouterShape<4, 16, 4>());
    else if (E <= 512) f(RouterShape<4, 32, 4>());
    else f(RouterShape<4, 64, 4>());
  } else {
    if (E <= 16) f(RouterShape<1, 16, 1>());
    else if (E <= 64) f(RouterShape<1, 16, 4>());
    else if (E <= 256) f(RouterShape<1, 64, 4>());
    else f(RouterShape<1, 64, 16>());
  }
}

constexpr int kRouterMaxBlocks = 256;
struct RouterPlan {
  int64_t rpb;
  int blocks;
  size_t part_q, part_c, part_z, part_n, total;
};
RouterPlan router_plan(int64_t T, int E, int64_t S) {
  RouterPlan p{};
  int step = 1;  // rows of a block's step
  with_router_shape(E, [&](auto c) { step = kRouterBlock / 64 * decltype(c)::RPW; });
  const int64_t steps = std::max<int64_t>(1, (T + step - 1) / step);
  p.rpb = step * ((steps + kRouterMaxBlocks - 1) / kRouterMaxBlocks);
  p.blocks = (int)std::max<int64_t>(1, (T + p.rpb - 1) / p.rpb);
  const size_t slots = (size_t)(p.blocks + S);
  Carve c;
  p.part_q = c.take(slots * E * 4);
  p.part_c = c.take(slots * E * 4);
  p.part_z = c.take(slots * 4);
  p.part_n = c.take(slots * 4);
  p.total = c.off;
  return p;
}

template <typename T, typename I>
RouterRows<T, I> router_rows(const void* logits, const void* idx, const int* offsets, int64_t Tn, int E, int k, int64_t S,
                             int score, float tau) {
  return {(const T*)logits, (const I*)idx, offsets, Tn, E, k, (int)S, score, 1.0f / tau};
}

// Calls f(logits' type, index type).
template <class F>
void with_router_types(int dtype, int index_bytes, F&& f) {
  if (dtype == MOE_DTYPE_BF16) {
    if (index_bytes == 4) f(bf16_t(), int32_t());
    else f(bf16_t(), int64_t());
  } else {
    if (index_bytes == 4) f(float(), int32_t());
    else f(float(), int64_t());
  }
}

}  // namespace

extern "C" {

size_t moe_router_losses_workspace_bytes(int64_t T, int32_t E, int64_t S) {
  if (check_router(MOE_DTYPE_F32, T, E, 1, 4, kScoreSoftmax, 1.0f, true, S) != MOE_OK) return 0;
  return router_plan(T, E, S).total;
}

moe_status moe_router_losses(int32_t device, void* stream, int32_t dtype, int64_t T, int32_t E, int32_t k,
                             int32_t index_bytes, const void* logits, const void* topk_idx, int32_t score,
                             float temperature, float switch_coef, float sqprob_coef, const int32_t* offsets, int64_t S,
                             float* balance, float* z, int32_t* counts, float* slope, float* inv_real,
                             void* workspace) {
  moe_status st = check_router(dtype, T, E, k, index_bytes, score, temperature, offsets != nullptr, S);
  if (st != MOE_OK || S == 0) return st;
  if ((st = check_ints({balance, z, counts})) != MOE_OK || (st = check_pointers({workspace})) != MOE_OK) return st;
  if (T > 0 && ((st = check_pointers({logits})) != MOE_OK || (st = check_ints({topk_idx}, index_bytes)) != MOE_OK))
    return st;
  if (offsets && (st = check_ints({offsets})) != MOE_OK) return st;
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  hipStream_t s = (hipStream_t)stream;
  const RouterPlan p = router_plan(T, E, S);
  char* ws = (char*)workspace;
  float *pq = (float*)(ws + p.part_q), *pz = (float*)(ws + p.part_z);
  int *pc = (int*)(ws + p.part_c), *pn = (int*)(ws + p.part_n);
  with_router_types(dtype, index_bytes, [&](auto t, auto i) {
    using D = decltype(t);
    using I = decltype(i);
    with_router_shape(E, [&](auto c) {
      hipLaunchKernelGGL((k_router_losses<decltype(c), D, I>), dim3(p.blocks), dim3(kRouterBlock), 0, s,
                         (router_rows<D, I>(logits, topk_idx, offsets, T, E, k, S, score, temperature)), p.rpb, pq, pc,
                         pz, pn);
    });
  });
  if (E % 4 == 0)
    hipLaunchKernelGGL(k_router_reduce<4>, dim3((unsigned)S), dim3(1024), 0, s, pq, pc, pz, pn, offsets, T, p.rpb, E, k,
                       switch_coef, sqprob_coef, balance, z, counts, slope, inv_real);
  else
    hipLaunchKernelGGL(k_router_reduce<1>, dim3((unsigned)S), dim3(1024), 0, s, pq, pc, pz, pn, offsets, T, p.rpb, E, k,
                       switch_coef, sqprob_coef, balance, z, counts, slope, inv_real);
  LAUNCH_CHECK();
  return MOE_OK;
}

moe_status moe_router_losses_backward(int32_t device, void* stream, int32_t dtype, int64_t T, int32_t E, int32_t k,
                                      int32_t index_bytes, const void* logits, const void* topk_idx, int32_t score,
                                      float temperature, const int32_t* offsets, int64_t S, const float* slope,
                                      const float* inv_real, const float* d_balance, const float* d_z, void* d_logits) {
  moe_status st = check_router(dtype, T, E, k, index_bytes, score, temperature, offsets != nullptr, S);
  if (st != MOE_OK || T == 0) return st;
  if ((st = check_pointers({logits, d_logits})) != MOE_OK || (st = check_ints({topk_idx}, index_bytes)) != MOE_OK)
    return st;
  if (S > 0 && (st = check_ints({slope, inv_real})) != MOE_OK) return st;
  if (offsets && (st = check_ints({offsets})) != MOE_OK) return st;
  DeviceScope dev(device);
  HIP_TRY(dev.enter());
  hipStream_t s = (hipStream_t)stream;
  with_router_types(dtype, index_bytes, [&](auto t, auto i) {
    using D = decltype(t);
    using I = decltype(i);
    with_router_shape(E, [&](auto c) {
      using C = decltype(c);
      // rows of a block: some steps where there are enough of them for every CU; within 2^20 blocks
      const int64_t step = (kRouterBwdBlock / 64) * C::RPW, steps = T / step;
      const int64_t rpb = step * std::max(std::min<int64_t>(4, steps / 1024 + 1), (steps >> 20) + 1);
      hipLaunchKernelGGL((k_router_losses_bwd<C, D, I>), dim3((unsigned)((T + rpb - 1) / rpb)), dim3(kRouterBwdBlock), 0,
                         s, (router_rows<D, I>(logits, topk_idx, offsets, T, E, k, S, score, temperature)), rpb, slope,
                         inv_real, d_balance, d_z, (D*)d_logits);
    });
  });
  LAUNCH_CHECK();
  return MOE_OK;
}

}  // extern "C"
