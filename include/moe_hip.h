/*
 * moe_hip.h -- C ABI of the MI355X (gfx950) Mixture-of-Experts layer.
 *
 * Drop-in boundary for oxidizr's MoE layer.  In the reference the layer is
 * `struct MoeLayer<R> { moe: boostr::nn::moe::layer::MoeLayer<R> }`
 * (src/model.rs:1632-1634), whose `forward` (src/model.rs:1834-1885) returns
 * (out, aux_loss, z_loss) and whose backward is the boostr autograd graph
 * walked by `backward_wrt` (src/trainer.rs:1097).  A Rust wrapper keeps that
 * struct, its constructors and config keys, and calls these entry points
 * through a thin FFI crate (rust/moe-hip-sys).
 *
 * Conventions
 *  - Every tensor argument is a DEVICE pointer, 16-byte aligned, row-major
 *    and contiguous, in the plan's dtype unless stated.  Linear weights are
 *    [out, in] and applied as y = x W^T (src/model.rs:1422-1445).
 *  - Per-expert weights are HOST arrays of E device pointers, because oxidizr
 *    keeps every expert projection as its own tensor (src/model.rs:1661-1672).
 *  - The caller owns all memory: `saved` (state kept from forward to
 *    backward) and `workspace` (scratch) are caller-allocated device buffers
 *    of moe_saved_bytes / moe_workspace_bytes.  The library allocates only at
 *    plan creation.
 *  - Work is enqueued on `stream` (a hipStream_t); calls do not synchronise
 *    the host.  Calls on one plan must be ordered on one stream.
 *  - Entry points never abort: they return a moe_status and leave a message
 *    for moe_last_error() (thread-local).
 *  - Results are bit-reproducible run to run: no floating-point atomics,
 *    every reduction has a fixed order.
 */
#ifndef MOE_HIP_H
#define MOE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  MOE_OK = 0,
  MOE_ERR_INVALID = 1,      /* bad argument or configuration */
  MOE_ERR_OOM = 2,          /* device allocation failed (plan creation) */
  MOE_ERR_HIP = 3,          /* HIP runtime error */
  MOE_ERR_UNSUPPORTED = 4   /* valid request this build does not implement */
} moe_status;

typedef enum { MOE_DTYPE_F32 = 0, MOE_DTYPE_BF16 = 1 } moe_dtype;

/* Layer configuration.  Keys follow oxidizr's ModelConfig / TrainerConfig
 * (src/config.rs:125-131, src/config_convert.rs:380-404); the boostr router
 * constants that the reference does not pin are explicit fields. */
typedef struct {
  int32_t hidden;               /* H  = hidden_size                                */
  int32_t num_experts;          /* E  = moe.num_experts (1..1024)                  */
  int32_t experts_per_tok;      /* k  = moe.experts_per_tok (1..min(E,16))         */
  int32_t intermediate;         /* I  = moe.intermediate_size (multiple of 8)      */
  int32_t shared_intermediate;  /* S  = total shared-expert width; 0 = none
                                   (shared_expert_enabled = false)                */
  int32_t dtype;                /* moe_dtype of x, weights, outputs, gradients     */
  int32_t norm_topk_prob;       /* 1: renormalise the k routing weights to sum 1   */
  int32_t has_router_bias;      /* 1: router Linear has a bias [E] (fp32)          */
  float router_temperature;     /* tau: probs = softmax(logits / tau)  (boostr
                                   MOE_ROUTER_TEMPERATURE, src/model.rs:1901)      */
  float shared_expert_scale;    /* s: out += s * shared(x) (src/model.rs:1923)     */
  float aux_switch_coef;        /* aux = E*(c_sw*sum_e f_e P_e + c_sq*sum_e P_e^2)  */
  float aux_sqprob_coef;        /*   (SwitchPlusSquaredProb, src/model.rs:1905)     */
  int32_t recompute_activations;/* 1: `saved` keeps the routing state only and
                                   moe_backward recomputes the expert activations
                                   first (trainer.activation_checkpointing covering
                                   this layer, src/config/activation_checkpointing.rs
                                   :25-35, src/model/recompute/segment.rs:58-170)  */
  int32_t fused_block;          /* 1: the plan runs the block's whole MoE sub-block
                                   through moe_block_forward / moe_block_backward:
                                   post_attention_layernorm (RMSNorm) before the
                                   layer and the residual add after it
                                   (src/model.rs:2792-2800, :2822-2826)           */
  float rms_norm_eps;           /* RMSNorm eps (cfg.rms_norm_eps); fused_block only */
} moe_config;

/* Fills cfg with the documented defaults: tau = 1, s = 1, c_sw = c_sq = 1,
 * no renormalisation, no router bias, bf16, activations kept. */
void moe_config_default(moe_config* cfg, int32_t hidden, int32_t num_experts,
                        int32_t experts_per_tok, int32_t intermediate,
                        int32_t shared_intermediate);

typedef struct moe_plan moe_plan;

/* Replaces MoeLayer::new / with_ids validation (src/model.rs:1640-1772,
 * required_moe_dims :1927-1958).  Binds the plan to `device`. */
moe_status moe_plan_create(const moe_config* cfg, int device, moe_plan** plan);
moe_status moe_plan_destroy(moe_plan* plan);

/* Whether a call over num_tokens tokens is supported by a plan of this
 * configuration, without a device: MOE_OK, MOE_ERR_INVALID (bad config or
 * negative count) or MOE_ERR_UNSUPPORTED (above 2^24 tokens, or an operand of
 * num_tokens x max(H, I, S, E rounded up to 8) elements reaching 2^31 bytes:
 * buffer loads take 32-bit offsets; split such a batch).  The forward and
 * backward entry points make the same check.  No reference counterpart (the
 * limit of this implementation; callers that batch tokens query it). */
moe_status moe_check_tokens(const moe_config* cfg, int64_t num_tokens);

/* Device-free self-check of this implementation's workspace plan for a call
 * over num_tokens tokens: every scratch region a launch uses, sized from the
 * launch's own grid and split arithmetic, fits the region moe_workspace_bytes
 * plans for it, and the regions of the forward (and of the backward) do not
 * overlap.  MOE_OK, or the moe_check_tokens errors, or MOE_ERR_INVALID naming
 * the region that does not fit.  No reference counterpart (a test of this
 * implementation's sizing, callable without a GPU). */
moe_status moe_workspace_check(const moe_config* cfg, int64_t num_tokens);

/* Bytes of the caller-owned buffers for a call over num_tokens tokens. */
size_t moe_saved_bytes(const moe_plan* plan, int64_t num_tokens);
size_t moe_workspace_bytes(const moe_plan* plan, int64_t num_tokens);

typedef struct {
  const void* router;              /* [E, H]   router.gate.weight                 */
  const float* router_bias;        /* [E] fp32 or NULL                             */
  const void* const* gate;         /* E x [I, H]  experts.{e}.gate_proj.weight    */
  const void* const* up;           /* E x [I, H]  experts.{e}.up_proj.weight      */
  const void* const* down;         /* E x [H, I]  experts.{e}.down_proj.weight    */
  const void* shared_gate;         /* [S, H] or NULL  shared_expert.gate_proj     */
  const void* shared_up;           /* [S, H] or NULL  shared_expert.up_proj       */
  const void* shared_down;         /* [H, S] or NULL  shared_expert.down_proj     */
} moe_weights;

typedef struct {
  void* router;                    /* [E, H]                                      */
  float* router_bias;              /* [E] fp32, or NULL (skip)                     */
  void* const* gate;               /* E x [I, H]; expert e written iff has_grad[e] */
  void* const* up;                 /* E x [I, H]                                  */
  void* const* down;               /* E x [H, I]                                  */
  void* shared_gate;               /* [S, H] or NULL                              */
  void* shared_up;                 /* [S, H] or NULL                              */
  void* shared_down;               /* [H, S] or NULL                              */
} moe_grads;

/* Forward over x [T, H] (the reference flattens [B, S, H] to [T, H],
 * src/model.rs:1878).  Writes out [T, H], and the fp32 scalars *aux_loss and
 * *z_loss (device pointers; MoeOutput::aux_loss / z_loss, src/model.rs:1884).
 * `saved` receives routing and activations for moe_backward; it must stay
 * untouched until then.  saved == NULL makes a forward-only call (the
 * need_grad = 0 case: eval under no_grad, src/eval/run.rs:74): no state
 * outlives the call, the routing and activations live in `workspace`, and the
 * gate / up pre-activations that only a backward reads are not computed into
 * memory.  Replaces MoeLayer::forward (src/model.rs:1834). */
moe_status moe_forward(moe_plan* plan, void* stream, int64_t num_tokens, const void* x,
                       const moe_weights* w, void* out, float* aux_loss, float* z_loss,
                       void* saved, void* workspace);

/* Forward-only call (as moe_forward with saved == NULL) that allocates
 * nothing: its scratch is a static device array of the library, 64 MiB per
 * GPU (held until the process ends), instead of a caller workspace, and it
 * creates no events (per-stage profiling is skipped for it).  Returns
 * MOE_ERR_UNSUPPORTED when num_tokens needs more scratch than that (the
 * forward regions of moe_workspace_bytes; decode-sized batches fit).  Every
 * call on one GPU shares that GPU's array, so calls that overlap on one GPU
 * (other streams, other plans, other threads) race; order them.  Under HIP
 * graph capture, call it once eagerly first with the same weight pointer
 * tables: a table change while the stream captures is refused with
 * MOE_ERR_UNSUPPORTED (the upload could not be replayed safely).  A captured
 * call reads the plan's device pointer tables when it replays, so replay it
 * only while the plan's last call used the same tables.  No counterpart in
 * the reference: for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops). */
moe_status moe_forward_noalloc(moe_plan* plan, void* stream, int64_t num_tokens, const void* x,
                               const moe_weights* w, void* out, float* aux_loss, float* z_loss);

/* Backward of the forward that filled `saved` (same x, weights, num_tokens).
 * d_out [T, H]; d_aux, d_z: device fp32 scalars dL/d(aux_loss), dL/d(z_loss)
 * (the trainer's alpha/n and gamma/n, src/trainer.rs:399-421), or NULL for 0.
 * Writes dx [T, H] and every weight gradient (overwriting, not accumulating).
 * has_grad (device uint8 [E], may be NULL) receives 1 for experts that saw at
 * least one token; experts with has_grad 0 have no gradient entry
 * (src/trainer.rs:556-566) and their buffers are left untouched.  With
 * num_tokens = 0 has_grad and the dense gradients (router, router bias, shared
 * expert) are set to zero.  Weight and gradient pointer tables are uploaded
 * when they change, without synchronising the stream.
 * Replaces the boostr GradFn chain walked by backward_wrt (src/trainer.rs:1097). */
moe_status moe_backward(moe_plan* plan, void* stream, int64_t num_tokens, const void* d_out,
                        const float* d_aux, const float* d_z, const void* x,
                        const moe_weights* w, const void* saved, void* workspace, void* dx,
                        const moe_grads* g, uint8_t* has_grad);

/* The MoE sub-block of a decoder block, for plans created with fused_block = 1
 * (src/model.rs:2792-2800 MLA arm, :2822-2826 legacy arm: residual = h;
 * x = post_attention_layernorm(h); (y, aux, z) = ffn(x); out = y + residual).
 * h [T, H]; norm_weight [H] (dtype) is post_attention_layernorm.weight;
 * RMSNorm(h) = h / sqrt(mean(h^2) + rms_norm_eps) * norm_weight with fp32
 * statistics.  The residual add is fused into the combine: out is rounded once.
 * `saved` as for moe_forward (NULL: forward only). */
moe_status moe_block_forward(moe_plan* plan, void* stream, int64_t num_tokens, const void* h,
                             const void* norm_weight, const moe_weights* w, void* out,
                             float* aux_loss, float* z_loss, void* saved, void* workspace);

/* Backward of moe_block_forward: dh [T, H] = d_out (the residual's path) +
 * the RMSNorm backward of the layer's input gradient; d_norm_weight [H]
 * (dtype, overwritten) = sum_t dx_t * h_t * rstd_t, reduced in a fixed order.
 * The layer's weight gradients and has_grad as for moe_backward. */
moe_status moe_block_backward(moe_plan* plan, void* stream, int64_t num_tokens,
                              const void* d_out, const float* d_aux, const float* d_z,
                              const void* h, const void* norm_weight, const moe_weights* w,
                              const void* saved, void* workspace, void* dh,
                              void* d_norm_weight, const moe_grads* g, uint8_t* has_grad);

/* Routing and dispatch only, from given fp32 logits [T, E] (no reference
 * counterpart; lets a caller check top-k and the permutation bit-exactly on
 * identical logits).  Fills the routing fields of `saved`. */
moe_status moe_route_from_logits(moe_plan* plan, void* stream, int64_t num_tokens,
                                 const float* logits, void* saved, void* workspace);

/* Byte offset and size of one field inside `saved` (for tests and callers
 * that want the routing decisions). */
typedef enum {
  MOE_SAVED_LOGITS = 0,   /* fp32 [T, E] */
  MOE_SAVED_PROBS,        /* fp32 [T, E] */
  MOE_SAVED_LSE,          /* fp32 [T] */
  MOE_SAVED_TOPK_IDX,     /* int32 [T, k], slot 0 = largest logit, ties -> lower index */
  MOE_SAVED_TOPK_W,       /* fp32 [T, k] */
  MOE_SAVED_COUNTS,       /* int32 [E] */
  MOE_SAVED_OFFSETS,      /* int32 [E + 1] */
  MOE_SAVED_PERM,         /* int32 [T*k]: expert-major position -> t*k + j */
  MOE_SAVED_INV_PERM,     /* int32 [T*k]: t*k + j -> position */
  MOE_SAVED_MEAN_PROB,    /* fp32 [E]: P_e = mean_t probs[t, e] */
  MOE_SAVED_X_PERM,       /* 0 bytes: the expert GEMMs read each assignment's token
                             row of x through the permutation (no permuted copy) */
  MOE_SAVED_GATE_ACT,     /* dtype [T*k, I]: x W_g^T */
  MOE_SAVED_UP_ACT,       /* dtype [T*k, I]: x W_u^T */
  MOE_SAVED_SWIGLU,       /* dtype [T*k, I]: silu(gate) * up */
  MOE_SAVED_EXPERT_OUT,   /* dtype [T*k, H]: per-assignment expert output; 0 bytes in
                             a training forward's `saved` (the backward does not
                             read it), present in the forward-only state */
  MOE_SAVED_RSTD,         /* fp32 [T]: 1 / RMS of h (fused_block plans only) */
  MOE_SAVED_NORM_X,       /* dtype [T, H]: RMSNorm(h), the layer input (fused_block only) */
  MOE_SAVED_NUM_FIELDS
} moe_saved_field;
moe_status moe_saved_field_range(const moe_plan* plan, int64_t num_tokens, int32_t field,
                                 size_t* offset, size_t* bytes);

/* Per-stage device timing with HIP events recorded on the call's stream
 * around each stage whose bit (1 << moe_stage) is set in stage_mask; -1 times
 * every stage, 0 (the default) none.  A stage whose work rides another's launch
 * records nothing.  Above 64 tokens: the losses (in the combine), and where the
 * router GEMM's launches also route (at most 64 experts, or 256 with hidden
 * >= 3584) the routing.  Up to 64 tokens: the dispatch and the losses
 * (in the routing), and in a bf16 forward the shared expert (beside the router
 * GEMM and the routing). */
typedef enum {
  MOE_STAGE_ROUTER_GEMM = 0, MOE_STAGE_ROUTE, MOE_STAGE_DISPATCH, MOE_STAGE_GATHER,
  MOE_STAGE_GATEUP_FWD, MOE_STAGE_DOWN_FWD, MOE_STAGE_SHARED_FWD, MOE_STAGE_COMBINE_FWD,
  MOE_STAGE_LOSSES, MOE_STAGE_COMBINE_BWD, MOE_STAGE_DOWN_DGRAD, MOE_STAGE_DOWN_WGRAD,
  MOE_STAGE_GATEUP_DGRAD, MOE_STAGE_GATEUP_WGRAD, MOE_STAGE_SHARED_BWD, MOE_STAGE_ROUTER_BWD,
  MOE_STAGE_DX, MOE_STAGE_RECOMPUTE, MOE_STAGE_NORM_FWD, MOE_STAGE_NORM_BWD, MOE_NUM_STAGES
} moe_stage;
const char* moe_stage_name(int32_t stage);
moe_status moe_plan_set_profiling(moe_plan* plan, int32_t stage_mask);
/* The shared expert runs on a second stream of the plan, and the backward's
 * routed weight gradients on a third (each forked from and joined back into
 * the call's stream inside every call), so that independent GEMMs fill each
 * other's partial rounds of work.  on = 0 runs everything on the call's
 * stream instead (serial order, for per-kernel measurements); on = 2 uses the
 * second stream only; on = 1 is the default.  The forward of at most 64 bf16
 * tokens runs on the call's stream alone.  Results are bitwise the same
 * every way.  No reference counterpart (scheduling knob of this
 * implementation). */
moe_status moe_plan_set_shared_overlap(moe_plan* plan, int32_t on);
/* Synchronises the pending events, then returns the accumulated milliseconds
 * and launch counts per stage since the last reset (arrays of MOE_NUM_STAGES). */
moe_status moe_plan_stage_times(moe_plan* plan, float* ms, int32_t* calls, int32_t reset);

/* ---- Operators beside the layer
 *
 * The pieces of a Mixture-of-Experts layer whose experts are not the plan's
 * SwiGLU (adapted experts, src/model.rs:1416-1446, other activations, biases,
 * norms on both sides of the block), as calls of their own: no plan, no state.
 * `device` is the device of every pointer and of `stream`; the caller's current
 * device is left as it was.  dtype: a moe_dtype of the activations, weights and
 * gradients.  Alignment, ownership, streams, errors and reproducibility as above,
 * but integer arrays need only their own alignment (they may be slices); a workspace is
 * used only while the call's kernels run. */

/* Stable counting sort of the T k assignments by expert: expert ascending, then
 * t k + j ascending.  topk_idx [T, k]: int32 (index_bytes 4) or int64 (8); an index
 * outside [0, E) is an assignment without an expert (padding) and is sorted behind
 * every expert, in t k + j's order.  The same expert may occur several times in a token.  counts [E],
 * offsets [E + 1] (offsets[E] = assignments that have an expert), perm [T k]
 * (position -> t k + j), inv_perm [T k] (t k + j -> position).  1 <= E <= 1024, 1 <= k
 * <= 16, T k < 2^31.  The workspace may be NULL where
 * moe_sort_workspace_bytes is 0. */
size_t moe_sort_workspace_bytes(int64_t num_tokens, int32_t experts_per_tok, int32_t num_experts);
moe_status moe_sort_tokens(int32_t device, void* stream, int64_t num_tokens,
                           int32_t experts_per_tok, int32_t num_experts, int32_t index_bytes,
                           const void* topk_idx, int32_t* counts, int32_t* offsets, int32_t* perm,
                           int32_t* inv_perm, void* workspace);

/* x_perm[inv_perm[t, j]] = x[t]; rows at or beyond *num_kept (a device int: the
 * sort's offsets + E) are zeros.  x [T, H], x_perm [T k, H], H a multiple of 8.  The
 * backward of x is moe_unpermute of the rows' gradient without weights. */
moe_status moe_permute(int32_t device, void* stream, int32_t dtype, int64_t num_tokens,
                       int32_t experts_per_tok, int32_t hidden, const int32_t* inv_perm,
                       const int32_t* num_kept, const void* x, void* x_perm);

/* out[t] = sum_j weights[t, j] y[inv_perm[t, j]] over the assignments that have an
 * expert, j ascending, in fp32, rounded once.  weights [T, k] fp32, or NULL: 1. */
moe_status moe_unpermute(int32_t device, void* stream, int32_t dtype, int64_t num_tokens,
                         int32_t experts_per_tok, int32_t hidden, const int32_t* inv_perm,
                         const int32_t* num_kept, const void* y, const float* weights, void* out);

/* Backward of moe_unpermute: d_y[inv_perm[t, j]] = weights[t, j] d_out[t] (zeros for an
 * assignment without an expert) and, when d_weights [T, k] is not NULL, d_weights[t, j] =
 * <d_out[t], y[inv_perm[t, j]]> (0 without an expert), in fp32. */
moe_status moe_unpermute_backward(int32_t device, void* stream, int32_t dtype, int64_t num_tokens,
                                  int32_t experts_per_tok, int32_t hidden,
                                  const int32_t* inv_perm, const int32_t* num_kept,
                                  const void* d_out, const void* y, const float* weights,
                                  void* d_y, float* d_weights);

/* Activations of moe_linear_forward: gelu with the error function, gelu_tanh with
 * its tanh approximation. */
typedef enum {
  MOE_ACT_NONE = 0, MOE_ACT_RELU, MOE_ACT_SILU, MOE_ACT_GELU, MOE_ACT_GELU_TANH
} moe_activation;

/* y[r] = act(x[r] W_g^T + b_g) + residual[r] for the rows offsets[g] <= r < offsets[g + 1]
 * of each group g.  x [M, K], weight [G, N, K], bias [G, N] or NULL, residual [M, N] or
 * NULL, y [M, N]; K = in_features and N = out_features are multiples of 8.  Rows before
 * the first group's and behind the last one's get y = residual (or 0).  offsets NULL: one weight [N, K] for every
 * row (num_groups 1).  pre_act [M, N] (or NULL) receives the pre-activation for a
 * backward.  Offsets ascend within 0..M (a range of a longer array will do, for
 * a range of its groups); with others no access leaves the
 * tensors, but which rows a group has, and whether every row of y is written, is not
 * defined.  Refused with MOE_ERR_UNSUPPORTED: a width above 2^20, a weight matrix of 2^31
 * bytes, more than 2^26 rows, operands of 2^34 bytes (2^31 where d_weight is asked for), and
 * more tiles than a launch holds (a thousand groups of a million columns).  moe_linear_workspace_bytes
 * is 0 for a refused call, backward: for one that asks for dx and d_weight. */
size_t moe_linear_workspace_bytes(int32_t dtype, int64_t num_rows, int32_t in_features,
                                  int32_t out_features, int32_t num_groups, int32_t grouped,
                                  int32_t activation, int32_t backward);
moe_status moe_linear_forward(int32_t device, void* stream, int32_t dtype, int64_t num_rows,
                              int32_t in_features, int32_t out_features, int32_t num_groups,
                              const int32_t* offsets, const void* x, const void* weight,
                              const void* bias, const void* residual, int32_t activation, void* y,
                              void* pre_act, void* workspace);
/* dx [M, K] (0 for rows of no group), d_weight [G, N, K] and d_bias [G, N] (0 for a
 * group without rows), each written unless NULL.  The residual's gradient is d_y. */
moe_status moe_linear_backward(int32_t device, void* stream, int32_t dtype, int64_t num_rows,
                               int32_t in_features, int32_t out_features, int32_t num_groups,
                               const int32_t* offsets, const void* d_y, const void* x,
                               const void* weight, const void* pre_act, int32_t activation,
                               void* dx, void* d_weight, void* d_bias, void* workspace);

/* The norms before and after a block, its gate and its residual, in one pass:
 *   u = RMSNorm(y) post_weight (u = y without post_weight),
 *   h_out = residual_scale h + gate u,  n_out = RMSNorm(h_out) next_weight,
 * with RMSNorm(v) = v / sqrt(mean(v^2) + eps), fp32 statistics, one rounding of h_out and
 * one of n_out (which is formed from the unrounded h_out).  All [T, H]; weights [H]; H a
 * multiple of 8 up to 32768.  gate: [H], [T] or [T, H] by gate_kind.  Without next_weight no
 * n_out is written.  Without y the call is a plain RMSNorm of h (no post_weight, no
 * gate, residual_scale 1): n_out = RMSNorm(h) next_weight, h_out is not written.
 * rstd_post, rstd_next [T] fp32: kept for a backward, or NULL. */
typedef enum {
  MOE_GATE_NONE = 0, MOE_GATE_CHANNEL, MOE_GATE_TOKEN, MOE_GATE_FULL
} moe_gate_kind;
moe_status moe_residual_norm(int32_t device, void* stream, int32_t dtype, int64_t num_tokens,
                             int32_t hidden, const void* h, const void* y,
                             const void* post_weight, const void* gate, int32_t gate_kind,
                             const void* next_weight, float residual_scale, float eps,
                             void* h_out, void* n_out, float* rstd_post, float* rstd_next);
/* Backward: d_h, d_y [T, H] and the gradients of post_weight, gate and next_weight, each in
 * its tensor's shape, for what the forward was given.  d_h_out may be NULL (0) where
 * d_n_out is given.  h_out is the forward's (without y: h).  _from_input takes the forward's h
 * instead and forms h_out from it again as it was before its rounding (from which the forward
 * formed n_out): the gradients are then those of the values that the forward used. */
size_t moe_residual_norm_workspace_bytes(int64_t num_tokens, int32_t hidden);
moe_status moe_residual_norm_backward(int32_t device, void* stream, int32_t dtype,
                                      int64_t num_tokens, int32_t hidden, const void* d_h_out,
                                      const void* d_n_out, const void* h_out, const void* y,
                                      const void* post_weight, const void* gate,
                                      int32_t gate_kind, const void* next_weight,
                                      float residual_scale, const float* rstd_post,
                                      const float* rstd_next, void* d_h, void* d_y,
                                      void* d_post_weight, void* d_gate, void* d_next_weight,
                                      void* workspace);
moe_status moe_residual_norm_backward_from_input(int32_t device, void* stream, int32_t dtype,
                                      int64_t num_tokens, int32_t hidden, const void* d_h_out,
                                      const void* d_n_out, const void* h, const void* y,
                                      const void* post_weight, const void* gate,
                                      int32_t gate_kind, const void* next_weight,
                                      float residual_scale, const float* rstd_post,
                                      const float* rstd_next, void* d_h, void* d_y,
                                      void* d_post_weight, void* d_gate, void* d_next_weight,
                                      void* workspace);

const char* moe_last_error(void);
const char* moe_version(void);

#ifdef __cplusplus
}
#endif
#endif /* MOE_HIP_H */
