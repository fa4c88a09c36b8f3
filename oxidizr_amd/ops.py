"""Operators beside the MoE layer, for layers whose experts are not the plan's SwiGLU: adapted
experts (src/model.rs:1416-1446), biases, other activations, norms on both sides of the block.

    order = sort_tokens(topk_idx, num_experts)            # assignments sorted by expert
    rows = permute_tokens(x, order)                       # [T, H] -> [T k, H], expert by expert
    a = expert_linear(rows, w1, b1, offsets=order.offsets, activation="gelu")
    b = expert_linear(a, w2, b2, offsets=order.offsets)
    y = unpermute_tokens(b, order, weights)               # back to [T, H], weighted
    h, n = residual_norm(h, y, post_weight, gate=g, next_weight=w)

The router's losses over the same routing, and experts whose frozen weights are held in 4 bits (adapters are
trained over such, prompts and decoding served from them):

    losses = router_losses(logits, topk_idx)              # balance, z, counts
    q1 = quantize_mxfp4(w1)                               # once
    a = mx_linear(rows, q1, b1, offsets=order.offsets, activation="gelu")
    a = mx_linear(quantize_mxfp4(rows), q1, b1, offsets=order.offsets, activation="gelu")  # both sides in 4 bits

Every function takes float32 or bfloat16 CUDA tensors (one dtype to a call; routing weights are
float32), runs on the current stream of their device, sums in fp32 in a fixed order and is
differentiable once, backward; a forward-mode derivative and a trace (torch.jit.trace, make_fx) are
refused.  Tensors that are not contiguous or not 16-byte aligned are copied first.
Wrong arguments raise ModelError, what the library refuses MoeError.  The arithmetic runs in
libmoe_hip.so; PyTorch provides memory, streams and the autograd nodes.
"""
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .moe import ModelError, _derivable, _dtype_code, _refuse_trace

ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")  # moe_activation's order
_GATE_NONE, _GATE_CHANNEL, _GATE_TOKEN, _GATE_FULL = range(4)
MAX_EXPERTS_PER_TOK = 16
MAX_EXPERTS = 1024


class TokenOrder(NamedTuple):
    """The T k assignments of a routing sorted by expert (int32 tensors)."""
    counts: torch.Tensor    # [E] assignments of each expert
    offsets: torch.Tensor   # [E + 1] their exclusive prefix; offsets[E]: assignments with an expert
    perm: torch.Tensor      # [T k] position -> t * k + j
    inv_perm: torch.Tensor  # [T, k] t * k + j -> position


def _ready(t):
    """t (or None) as the library reads it: contiguous and 16-byte aligned."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _once(backward):
    """once_differentiable, at no cost where no second derivative can follow."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _on_device(first, *others):
    """The device index of a call's tensors (the first is always there)."""
    _refuse_trace()
    dev = first.get_device()
    if dev < 0:
        raise ModelError(f"expected CUDA tensors, got one on {first.device}")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ModelError(f"tensors on different devices: {first.device} and {t.device}")
    return dev


def _call(fn, device, *args):
    # the current stream's handle without the Stream object around it (1.5 us of a call)
    _lib.check(fn(device, torch._C._cuda_getCurrentRawStream(device), *args))


def _workspace(nbytes, like):
    """Scratch of one call, from the caching allocator: its stream hands the memory out again only
    behind the call's kernels, and a captured call keeps its own in the graph's pool."""
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


# ---------------------------------------------------------------- tokens sorted by expert and back

def sort_tokens(topk_idx, num_experts: int) -> TokenOrder:
    """Stable sort of topk_idx [T, k] (int32 or int64) by expert, then by t * k + j. An index outside
    [0, num_experts) has no expert (a padding token) and comes behind every expert."""
    if topk_idx.dim() != 2:
        raise ModelError(f"topk_idx must be [T, k], got {list(topk_idx.shape)}")
    if topk_idx.dtype not in (torch.int32, torch.int64):
        raise ModelError(f"topk_idx must be int32 or int64, got {topk_idx.dtype}")
    T, k = topk_idx.shape
    if not 1 <= k <= MAX_EXPERTS_PER_TOK:
        raise ModelError(f"experts per token must be 1..{MAX_EXPERTS_PER_TOK}, got {k}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ModelError(f"num_experts must be 1..{MAX_EXPERTS}, got {num_experts}")
    dev = _on_device(topk_idx)
    idx = topk_idx.contiguous()
    L = _lib.load()
    # one allocation for all four; .data gives perm and counts version counters of their own, apart from that
    # of inv and offsets, which gradients read: writing to the former before a backward is no error
    out = torch.empty(2 * num_experts + 1 + 2 * T * k, dtype=torch.int32, device=idx.device)
    perm, inv, offsets, counts = out.split((T * k, T * k, num_experts + 1, num_experts))
    perm, counts = perm.data, counts.data
    ws = _workspace(L.moe_sort_workspace_bytes(T, k, num_experts), idx)
    _call(L.moe_sort_tokens, dev, T, k, num_experts, idx.element_size(), idx.data_ptr(), counts.data_ptr(),
          offsets.data_ptr(), perm.data_ptr(), inv.data_ptr(), _ptr(ws))
    return TokenOrder(counts, offsets, perm, inv.view(T, k))


def _check_hidden(H):
    if H < 8 or H % 8:
        raise ModelError(f"the hidden size must be a positive multiple of 8, got {H}")


def _kept(offsets):
    """Address of the number of assignments that have an expert."""
    return offsets.data_ptr() + 4 * (offsets.numel() - 1)


class _Slots:
    """What the row kernels read of a TokenOrder."""
    __slots__ = ("inv", "offsets", "T", "k", "kept")

    def __init__(self, order):
        if not isinstance(order, TokenOrder):
            raise ModelError("order must be a TokenOrder (sort_tokens)")
        offsets, inv = order.offsets, order.inv_perm
        if inv.dim() != 2:
            raise ModelError("order.inv_perm must be [T, k]")
        if inv.dtype != torch.int32 or offsets.dtype != torch.int32:
            raise ModelError(f"a TokenOrder holds int32 tensors, got {inv.dtype} and {offsets.dtype}")
        self.T, self.k = inv.shape
        if not 1 <= self.k <= MAX_EXPERTS_PER_TOK:
            raise ModelError(f"experts per token must be 1..{MAX_EXPERTS_PER_TOK}, got {self.k}")
        E = offsets.numel() - 1
        if offsets.dim() != 1 or E < 1:
            raise ModelError("order.offsets must be [E + 1]")
        self.inv, self.offsets = inv.contiguous(), offsets.contiguous()
        self.kept = _kept(self.offsets)


def _permute(x, slots):
    H = x.shape[1]
    out = x.new_empty(slots.T * slots.k, H)
    _call(_lib.load().moe_permute, x.get_device(), _dtype_code(x.dtype), slots.T, slots.k, H,
          slots.inv.data_ptr(), slots.kept, x.data_ptr(), out.data_ptr())
    return out


def _unpermute(y, slots, weights):
    H = y.shape[1]
    out = y.new_empty(slots.T, H)
    _call(_lib.load().moe_unpermute, y.get_device(), _dtype_code(y.dtype), slots.T, slots.k, H,
          slots.inv.data_ptr(), slots.kept, y.data_ptr(), _ptr(weights), out.data_ptr())
    return out


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slots):
        # saved, so that autograd sees whether the order was written to before the backward
        ctx.save_for_backward(slots.offsets, slots.inv)
        return _permute(_ready(x), slots)

    @staticmethod
    @_once
    def backward(ctx, dxp):
        offsets, inv = ctx.saved_tensors
        dxp = _ready(dxp)
        (T, k), H = inv.shape, dxp.shape[1]
        dx = dxp.new_empty(T, H)
        _call(_lib.load().moe_unpermute, dxp.get_device(), _dtype_code(dxp.dtype), T, k, H, inv.data_ptr(),
              _kept(offsets), dxp.data_ptr(), None, dx.data_ptr())
        return dx, None


def permute_tokens(x, order: TokenOrder):
    """Rows of x [T, H] in the order's positions: out[inv_perm[t, j]] = x[t] [T k, H]; the rows behind
    the last expert's (assignments without one) are zeros."""
    slots = _Slots(order)
    if x.dim() != 2 or x.shape[0] != slots.T:
        raise ModelError(f"x must be [{slots.T}, H], got {list(x.shape)}")
    _check_hidden(x.shape[1])
    _dtype_code(x.dtype)
    _on_device(x, slots.inv, slots.offsets)
    if _derivable(x):
        return _Permute.apply(x, slots)
    return _permute(_ready(x), slots)


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, slots):
        y = _ready(y)
        weights = _ready(weights)
        need_dw = weights is not None and ctx.needs_input_grad[1]
        # the rows are read again only for the gradient of the weights
        ctx.save_for_backward(y if need_dw else None, weights, slots.offsets, slots.inv)
        return _unpermute(y, slots, weights)

    @staticmethod
    @_once
    def backward(ctx, dout):
        y, weights, offsets, inv = ctx.saved_tensors
        dout = _ready(dout)
        (T, k), H = inv.shape, dout.shape[1]
        dy = dout.new_empty(T * k, H)
        dw = torch.empty_like(weights) if y is not None else None
        _call(_lib.load().moe_unpermute_backward, dout.get_device(), _dtype_code(dout.dtype), T, k, H,
              inv.data_ptr(), _kept(offsets), dout.data_ptr(), _ptr(y), _ptr(weights), dy.data_ptr(),
              _ptr(dw))
        return dy, dw, None


def unpermute_tokens(y, order: TokenOrder, weights: Optional[torch.Tensor] = None):
    """out[t] = sum_j weights[t, j] * y[inv_perm[t, j]] [T, H] over the assignments that have an expert,
    j ascending; weights [T, k] float32, or None for a plain sum."""
    slots = _Slots(order)
    T, k = slots.T, slots.k
    if y.dim() != 2 or y.shape[0] != T * k:
        raise ModelError(f"y must be [{T * k}, H], got {list(y.shape)}")
    _check_hidden(y.shape[1])
    _dtype_code(y.dtype)
    if weights is not None and (weights.dtype != torch.float32 or weights.shape != (T, k)):
        raise ModelError(f"weights must be float32 [{T}, {k}], got {weights.dtype} {list(weights.shape)}")
    _on_device(y, slots.inv, slots.offsets, weights)
    if _derivable(y, weights):
        return _Unpermute.apply(y, weights, slots)
    return _unpermute(_ready(y), slots, _ready(weights))


# ---------------------------------------------------------------- expert products

class _LinearShape(NamedTuple):
    M: int
    K: int
    N: int
    groups: int
    grouped: bool
    act: int


def _linear(x, weight, bias, offsets, residual, s, keep):
    L = _lib.load()
    code = _dtype_code(x.dtype)
    y = x.new_empty(s.M, s.N)
    pre = torch.empty_like(y) if keep else None
    ws = _workspace(L.moe_linear_workspace_bytes(code, s.M, s.K, s.N, s.groups, s.grouped, s.act, 0), x)
    _call(L.moe_linear_forward, x.get_device(), code, s.M, s.K, s.N, s.groups, _ptr(offsets), _ptr(x),
          _ptr(weight), _ptr(bias), _ptr(residual), s.act, _ptr(y), _ptr(pre), _ptr(ws))
    return y, pre


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, offsets, s):
        x, weight = _ready(x), _ready(weight)
        bias = _ready(bias)
        residual = _ready(residual)
        products = any(ctx.needs_input_grad[:3])  # any gradient that reads the pre-activation
        if products:
            # here, where a refused backward can still be told (and calls cost less than in autograd's thread)
            L = _lib.load()
            ctx.ws_bytes = L.moe_linear_workspace_bytes(_dtype_code(x.dtype), s.M, s.K, s.N, s.groups, s.grouped,
                                                        s.act, 1)
            if ctx.ws_bytes == 0 and s.M > 0:
                raise _lib.MoeError(_lib.MOE_ERR_UNSUPPORTED, L.moe_last_error().decode())
        y, pre = _linear(x, weight, bias, offsets, residual, s, products and s.act != 0)
        ctx.save_for_backward(x, weight, pre, offsets)
        ctx.s = s
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, pre, offsets = ctx.saved_tensors
        s, (need_x, need_w, need_b, need_r) = ctx.s, ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            up = _ready(dy)
            L = _lib.load()
            code = _dtype_code(up.dtype)
            dx = torch.empty_like(x) if need_x else None
            dw = torch.empty_like(weight) if need_w else None
            db = up.new_empty((s.groups, s.N) if s.grouped else (s.N,)) if need_b else None
            ws = _workspace(ctx.ws_bytes, up)
            _call(L.moe_linear_backward, up.get_device(), code, s.M, s.K, s.N, s.groups, _ptr(offsets),
                  _ptr(up), _ptr(x), _ptr(weight), _ptr(pre), s.act, _ptr(dx), _ptr(dw), _ptr(db),
                  _ptr(ws))
        return dx, dw, db, dy if need_r else None, None, None


def expert_linear(x, weight, bias=None, *, offsets=None, activation: str = "none", residual=None):
    """activation(x W^T + bias) + residual, [M, N].

    With offsets (int32 [E + 1], ascending, as sort_tokens gives them, or a range of those with as
    many weights) rows offsets[e] .. offsets[e + 1] of x [M, K] take weight[e] of weight [E, N, K] and
    bias[e] of bias [E, N]; rows of no expert are the residual's, or zeros. Without offsets weight is
    [N, K] and bias [N]. K and N are multiples of 8. Where weight requires a gradient, x and y hold less than
    2^31 bytes.
    activation: one of ACTIVATIONS ("gelu" with the error function, "gelu_tanh" approximated)."""
    if activation not in ACTIVATIONS:
        raise ModelError(f"activation must be one of {ACTIVATIONS}, got {activation!r}")
    if x.dim() != 2:
        raise ModelError(f"x must be [M, K], got {list(x.shape)}")
    M, K = x.shape
    grouped = offsets is not None
    if not (weight.dim() == (3 if grouped else 2) and weight.shape[-1] == K):
        raise ModelError(f"weight must be {'[E, N' if grouped else '[N'}, {K}], got {list(weight.shape)}")
    groups, N = (weight.shape[0], weight.shape[1]) if grouped else (1, weight.shape[0])
    if not (K >= 8 and K % 8 == 0 and N >= 8 and N % 8 == 0):
        raise ModelError(f"input and output widths must be positive multiples of 8, got {K} and {N}")
    if grouped:
        if not 1 <= groups <= MAX_EXPERTS:
            raise ModelError(f"num_experts must be 1..{MAX_EXPERTS}, got {groups}")
        if not (offsets.dtype == torch.int32 and offsets.shape == (groups + 1,)):
            raise ModelError(f"offsets must be int32 [{groups + 1}], got {offsets.dtype} {list(offsets.shape)}")
    if bias is not None:
        want = (groups, N) if grouped else (N,)
        if bias.shape != want:
            raise ModelError(f"bias must be {list(want)}, got {list(bias.shape)}")
    if residual is not None:
        if not (residual.shape == (M, N)):
            raise ModelError(f"residual must be [{M}, {N}], got {list(residual.shape)}")
    _dtype_code(x.dtype)
    for t in (weight, bias, residual):
        if not (t is None or t.dtype == x.dtype):
            raise ModelError("x, weight, bias and residual must have one dtype")
    # the operands of the weight's gradient reach over all rows
    if M * max(K, N) * x.element_size() >= 1 << 31 and torch.is_grad_enabled() and weight.requires_grad:
        raise ModelError(f"{M} rows of {max(K, N)} reach 2^31 bytes, more than the weight's gradient takes: "
                         "split the batch")
    _on_device(x, weight, bias, residual, offsets)
    s = _LinearShape(M, K, N, groups, grouped, ACTIVATIONS.index(activation))
    offsets = offsets.contiguous() if grouped else None
    if _derivable(x, weight, bias, residual):
        return _ExpertLinear.apply(x, weight, bias, residual, offsets, s)
    return _linear(_ready(x), _ready(weight), _ready(bias), offsets,
                   _ready(residual), s, False)[0]


# ---------------------------------------------------------------- norms around a block

class _NormShape(NamedTuple):
    T: int
    H: int
    gate_kind: int
    scale: float
    eps: float


def _norm(h, y, post_weight, gate, next_weight, s, keep):
    out = torch.empty_like(h) if y is not None else None
    n = torch.empty_like(h) if next_weight is not None else None
    r2 = h.new_empty(s.T, dtype=torch.float32) if keep and post_weight is not None else None
    r3 = h.new_empty(s.T, dtype=torch.float32) if keep and next_weight is not None else None
    _call(_lib.load().moe_residual_norm, h.get_device(), _dtype_code(h.dtype), s.T, s.H, _ptr(h), _ptr(y),
          _ptr(post_weight), _ptr(gate), s.gate_kind, _ptr(next_weight), s.scale, s.eps, _ptr(out), _ptr(n),
          _ptr(r2), _ptr(r3))
    return out, n, r2, r3


class _ResidualNorm(torch.autograd.Function):
    """(h_out, n) of a block's output y, or n alone without y (a plain RMSNorm of h)."""

    @staticmethod
    def forward(ctx, h, y, post_weight, gate, next_weight, s):
        ctx.set_materialize_grads(False)
        h, y, gate = _ready(h), _ready(y), _ready(gate)
        post_weight, next_weight = _ready(post_weight), _ready(next_weight)
        out, n, r2, r3 = _norm(h, y, post_weight, gate, next_weight, s, True)
        # h alone: what the second norm is taken of is formed from it again, unrounded
        ctx.save_for_backward(h if n is not None else None, y, post_weight, gate, next_weight, r2, r3)
        ctx.s = s
        # the backward runs in autograd's thread, where every call costs several times as much
        ctx.ws_bytes = _lib.load().moe_residual_norm_workspace_bytes(s.T, s.H)
        return (out, n) if y is not None and n is not None else out if n is None else n

    @staticmethod
    @_once
    def backward(ctx, *up):
        h, y, post_weight, gate, next_weight, r2, r3 = ctx.saved_tensors
        s = ctx.s
        d_out = up[0] if y is not None else None
        d_n = up[-1] if next_weight is not None else None
        d_out, d_n = _ready(d_out), _ready(d_n)
        like = d_out if d_out is not None else d_n
        if like is None:
            return (None,) * 6
        d_next = None
        if next_weight is not None:
            # without a gradient of n the second norm has none
            d_next = torch.zeros_like(next_weight) if d_n is None else torch.empty_like(next_weight)
        used = next_weight if d_n is not None else None
        d_h = torch.empty_like(like)
        d_y = None if y is None else torch.empty_like(like)
        d_post = None if post_weight is None else torch.empty_like(post_weight)
        d_gate = None if gate is None else torch.empty_like(gate)
        ws = _workspace(ctx.ws_bytes, like)
        _call(_lib.load().moe_residual_norm_backward_from_input, like.get_device(), _dtype_code(like.dtype),
              s.T, s.H, _ptr(d_out), _ptr(d_n), _ptr(h), _ptr(y), _ptr(post_weight), _ptr(gate), s.gate_kind,
              _ptr(used), s.scale, _ptr(r2), _ptr(r3), _ptr(d_h), _ptr(d_y), _ptr(d_post), _ptr(d_gate),
              _ptr(d_next) if used is not None else None, _ptr(ws))
        return d_h, d_y, d_post, d_gate, d_next, None


def _gate_kind(gate, h):
    if gate is None:
        return _GATE_NONE
    if gate.shape == h.shape:
        return _GATE_FULL
    if gate.shape == h.shape[-1:]:
        return _GATE_CHANNEL
    if gate.shape != h.shape[:-1] + (1,):
        raise ModelError(
            f"gate must be {list(h.shape[-1:])}, {list(h.shape[:-1]) + [1]} or {list(h.shape)}, "
            f"got {list(gate.shape)}")
    return _GATE_TOKEN


def _check_norm(h, *weights):
    if h.dim() < 2:
        raise ModelError(f"expected [..., T, H], got {list(h.shape)}")
    H = h.shape[-1]
    _check_hidden(H)
    _dtype_code(h.dtype)
    for w in weights:
        if not (w is None or w.shape == (H,)):
            raise ModelError(f"a norm's weight must be [{H}]")
        if not (w is None or w.dtype == h.dtype):
            raise ModelError("activations and norm weights must have one dtype")
    return H


def rms_norm(x, weight, eps: float = 1e-6):
    """x / sqrt(mean(x^2) + eps) * weight over the last dimension."""
    if weight is None:
        raise ModelError("rms_norm needs a weight")
    H = _check_norm(x, weight)
    _on_device(x, weight)
    s = _NormShape(x.numel() // H, H, _GATE_NONE, 1.0, eps)
    if _derivable(x, weight):
        return _ResidualNorm.apply(x, None, None, None, weight, s)
    return _norm(_ready(x), None, None, None, _ready(weight), s, False)[1]


def residual_norm(h, y, post_weight=None, *, gate=None, next_weight=None, residual_scale: float = 1.0,
                  eps: float = 1e-6):
    """A block's output y added to its input h, with the norms on both sides, in one pass:

        h_out = residual_scale * h + gate * RMSNorm(y) * post_weight   (y itself without post_weight)
        n     = RMSNorm(h_out) * next_weight                           (the next block's input)

    h, y [..., H]; post_weight, next_weight [H]; gate [H], [..., 1] or [..., H]. Returns h_out, or
    (h_out, n) with a next_weight."""
    H = _check_norm(h, post_weight, next_weight)
    if y.shape != h.shape:
        raise ModelError(f"y must be {list(h.shape)}, got {list(y.shape)}")
    if not (y.dtype == h.dtype and (gate is None or gate.dtype == h.dtype)):
        raise ModelError("h, y and gate must have one dtype")
    kind = _gate_kind(gate, h)
    _on_device(h, y, post_weight, gate, next_weight)
    s = _NormShape(h.numel() // H, H, kind, float(residual_scale), eps)
    if _derivable(h, y, post_weight, gate, next_weight):
        return _ResidualNorm.apply(h, y, post_weight, gate, next_weight, s)
    out, n, _, _ = _norm(_ready(h), _ready(y), _ready(post_weight), _ready(gate), _ready(next_weight), s, False)
    return out if n is None else (out, n)


# ---------------------------------------------------------------- losses of a router

SCORES = ("softmax", "sigmoid")  # moe_score's order
MAX_SEQUENCES = (1 << 22) - 1


class RouterLosses(NamedTuple):
    """Losses of a routing (float32) and its counts (int32); a leading S with offsets."""
    balance: torch.Tensor  # [] or [S]
    z: torch.Tensor        # [] or [S]
    counts: torch.Tensor   # [E] or [S, E] assignments of each expert


class _RouterShape(NamedTuple):
    T: int
    E: int
    k: int
    S: int
    score: int
    temperature: float
    switch_coef: float
    sqprob_coef: float
    shape: tuple  # of a loss


def _router(logits, idx, offsets, s, keep):
    L = _lib.load()
    balance, z = logits.new_empty(s.shape, dtype=torch.float32), logits.new_empty(s.shape, dtype=torch.float32)
    counts = logits.new_empty(s.shape + (s.E,), dtype=torch.int32)
    # one allocation for what a backward reads: slope and inv_real
    kept, at = None, (None, None)
    if keep:
        kept = logits.new_empty(s.S * (s.E + 1), dtype=torch.float32)
        at = _kept_of_router(kept, s)
    ws = _workspace(L.moe_router_losses_workspace_bytes(s.T, s.E, s.S), logits)
    _call(L.moe_router_losses, logits.get_device(), _dtype_code(logits.dtype), s.T, s.E, s.k, idx.element_size(),
          logits.data_ptr(), idx.data_ptr(), s.score, s.temperature, s.switch_coef, s.sqprob_coef, _ptr(offsets), s.S,
          balance.data_ptr(), z.data_ptr(), counts.data_ptr(), *at, _ptr(ws))
    return balance, z, counts, kept


def _kept_of_router(kept, s):
    at = kept.data_ptr()
    return at, at + 4 * s.S * s.E


class _RouterLosses(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, idx, offsets, s):
        ctx.set_materialize_grads(False)
        logits = _ready(logits)
        balance, z, counts, kept = _router(logits, idx, offsets, s, True)
        ctx.save_for_backward(logits, idx, offsets, kept)
        ctx.s = s
        ctx.mark_non_differentiable(counts)
        return balance, z, counts

    @staticmethod
    @_once
    def backward(ctx, d_balance, d_z, _):
        logits, idx, offsets, kept = ctx.saved_tensors
        s = ctx.s
        if d_balance is None and d_z is None:
            return (None,) * 4
        d_balance = None if d_balance is None else d_balance.contiguous()
        d_z = None if d_z is None else d_z.contiguous()
        d_logits = torch.empty_like(logits)
        _call(_lib.load().moe_router_losses_backward, logits.get_device(), _dtype_code(logits.dtype), s.T, s.E, s.k,
              idx.element_size(), logits.data_ptr(), idx.data_ptr(), s.score, s.temperature, _ptr(offsets), s.S,
              *_kept_of_router(kept, s), _ptr(d_balance), _ptr(d_z), d_logits.data_ptr())
        return d_logits, None, None, None


def router_losses(logits, topk_idx, *, score: str = "softmax", temperature: float = 1.0, switch_coef: float = 1.0,
                  sqprob_coef: float = 1.0, offsets=None) -> RouterLosses:
    """The load-balance and z losses of a routing, and each expert's assignments:

        x = logits / temperature,  q = softmax(x), or sigmoid(x) / sum sigmoid(x)
        balance = E sum_e (switch_coef f_e P_e + sqprob_coef P_e^2),  P_e = mean_t q_te,  f_e = M_e / (k n)
        z = mean_t logsumexp(x_t)^2

    over the n tokens that have an expert; tokens all of whose topk_idx [T, k] (int32 or int64) lie outside [0, E) are
    padding, whatever their logits [T, E] hold. With offsets (int32 [S + 1], ascending row offsets of sequences) each sequence
    has losses and counts of its own; rows of none count nowhere. A sequence without tokens has losses 0. Differentiable in
    logits; the counts M_e are not."""
    if logits.dim() != 2:
        raise ModelError(f"logits must be [T, E], got {list(logits.shape)}")
    T, E = logits.shape
    if topk_idx.dim() != 2 or topk_idx.shape[0] != T:
        raise ModelError(f"topk_idx must be [{T}, k], got {list(topk_idx.shape)}")
    if topk_idx.dtype not in (torch.int32, torch.int64):
        raise ModelError(f"topk_idx must be int32 or int64, got {topk_idx.dtype}")
    k = topk_idx.shape[1]
    if not 1 <= k <= MAX_EXPERTS_PER_TOK:
        raise ModelError(f"experts per token must be 1..{MAX_EXPERTS_PER_TOK}, got {k}")
    if not 1 <= E <= MAX_EXPERTS:
        raise ModelError(f"num_experts must be 1..{MAX_EXPERTS}, got {E}")
    if score not in SCORES:
        raise ModelError(f"score must be one of {SCORES}, got {score!r}")
    # as a float32, and its inverse
    if not 2.0 ** -126 <= temperature < 2.0 ** 128:
        raise ModelError(f"temperature must be positive (at least 2^-126) and finite, got {temperature}")
    S = 1
    if offsets is not None:
        if offsets.dim() != 1 or offsets.dtype != torch.int32 or offsets.numel() < 1:
            raise ModelError(f"offsets must be int32 [S + 1], got {offsets.dtype} {list(offsets.shape)}")
        S = offsets.numel() - 1
        if S > MAX_SEQUENCES:
            raise ModelError(f"at most {MAX_SEQUENCES} sequences, got {S}")
    _dtype_code(logits.dtype)
    _on_device(logits, topk_idx, offsets)
    s = _RouterShape(T, E, k, S, SCORES.index(score), float(temperature), float(switch_coef), float(sqprob_coef),
                     () if offsets is None else (S,))
    idx = topk_idx.contiguous()
    offsets = None if offsets is None else offsets.contiguous()
    if _derivable(logits):
        return RouterLosses(*_RouterLosses.apply(logits, idx, offsets, s))
    return RouterLosses(*_router(_ready(logits), idx, offsets, s, False)[:3])


# ---------------------------------------------------------------- microscaled 4-bit numbers

MX_BLOCK = 32


class MxTensor(NamedTuple):
    """A tensor [..., K] of OCP MXFP4 numbers: E2M1 elements, 32 along the last dimension under one
    power of two. An element's four bits are its sign and one of 0 0.5 1 1.5 2 3 4 6; element 2 i is the low
    half of byte i. A scale byte is the exponent plus 127 (255: NaN)."""
    codes: torch.Tensor   # uint8 [..., K / 2]
    scales: torch.Tensor  # uint8 [..., K / 32]


def quantize_mxfp4(x) -> MxTensor:
    """x [..., K] (float32 or bfloat16, K a multiple of 32) in 4 bits: a block's exponent is that of its largest
    magnitude less 2, an element the nearest number (ties to the even code; what is above the largest becomes it). A block that
    holds an infinity or a NaN becomes NaN. The result has no gradient."""
    if x.dim() < 1 or x.shape[-1] < MX_BLOCK or x.shape[-1] % MX_BLOCK:
        raise ModelError(f"expected [..., K] with K a positive multiple of {MX_BLOCK}, got {list(x.shape)}")
    code = _dtype_code(x.dtype)
    dev = _on_device(x)
    x = _ready(x.detach())
    lead, K = x.shape[:-1], x.shape[-1]
    codes = x.new_empty(lead + (K // 2,), dtype=torch.uint8)
    scales = x.new_empty(lead + (K // MX_BLOCK,), dtype=torch.uint8)
    _call(_lib.load().moe_mx_quantize, dev, code, scales.numel(), x.data_ptr(), codes.data_ptr(), scales.data_ptr())
    return MxTensor(codes, scales)


def _check_mx(q, what):
    if not isinstance(q, MxTensor):
        raise ModelError(f"{what} must be an MxTensor (quantize_mxfp4)")
    c, s = q
    if c.dtype != torch.uint8 or s.dtype != torch.uint8:
        raise ModelError(f"an MxTensor holds uint8 tensors, got {c.dtype} and {s.dtype}")
    if not (c.dim() >= 1 and c.dim() == s.dim() and c.shape[:-1] == s.shape[:-1] and s.shape[-1] >= 1 and
            c.shape[-1] == MX_BLOCK // 2 * s.shape[-1]):
        raise ModelError(f"{what}: codes {list(c.shape)} and scales {list(s.shape)} do not go together "
                         f"([..., K / 2] and [..., K / {MX_BLOCK}])")


def dequantize_mxfp4(q: MxTensor, dtype=torch.bfloat16):
    """The numbers [..., K] that q stands for, in dtype (float32 or bfloat16): exact, and infinite from 2^128 on (elements of 2
    and more under the scale byte 254, of 4 and more under 253, which quantize_mxfp4 never makes)."""
    _check_mx(q, "q")
    code = _dtype_code(dtype)
    dev = _on_device(*q)
    codes, scales = _ready(q.codes), q.scales.contiguous()
    y = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=dtype, device=codes.device)
    _call(_lib.load().moe_mx_dequantize, dev, code, scales.numel(), codes.data_ptr(), scales.data_ptr(), y.data_ptr())
    return y


class _MxShape(NamedTuple):
    M: int
    K: int
    N: int
    groups: int
    grouped: bool
    act: int
    rows: int          # moe_mx_rows
    dtype: torch.dtype


def _mx(x, x_scales, codes, scales, bias, offsets, residual, s, keep):
    y = torch.empty(s.M, s.N, dtype=s.dtype, device=x.device)
    pre = torch.empty_like(y) if keep else None
    _call(_lib.load().moe_mx_linear_forward, x.get_device(), s.rows, _dtype_code(s.dtype), s.M, s.K, s.N, s.groups,
          _ptr(offsets), x.data_ptr(), _ptr(x_scales), codes.data_ptr(), scales.data_ptr(), _ptr(bias), _ptr(residual),
          s.act, y.data_ptr(), _ptr(pre))
    return y, pre


class _MxLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, x_scales, bias, residual, codes, scales, offsets, s):
        x, bias, residual = _ready(x), _ready(bias), _ready(residual)
        products = ctx.needs_input_grad[0] or ctx.needs_input_grad[2]
        if products:
            # here, where a refused backward can still be told
            L = _lib.load()
            ctx.ws_bytes = L.moe_mx_linear_workspace_bytes(s.M, s.K, s.N, s.groups, s.grouped, s.act)
            if ctx.ws_bytes == 0 and s.M > 0:
                raise _lib.MoeError(_lib.MOE_ERR_UNSUPPORTED, L.moe_last_error().decode())
        y, pre = _mx(x, x_scales, codes, scales, bias, offsets, residual, s, products and s.act != 0)
        ctx.save_for_backward(codes, scales, pre, offsets)
        ctx.s = s
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        codes, scales, pre, offsets = ctx.saved_tensors
        s, need_x, need_b, need_r = ctx.s, ctx.needs_input_grad[0], ctx.needs_input_grad[2], ctx.needs_input_grad[3]
        dx = db = None
        if need_x or need_b:
            up = _ready(dy)
            dx = up.new_empty(s.M, s.K) if need_x else None
            db = up.new_empty((s.groups, s.N) if s.grouped else (s.N,)) if need_b else None
            ws = _workspace(ctx.ws_bytes, up)
            _call(_lib.load().moe_mx_linear_backward, up.get_device(), s.M, s.K, s.N, s.groups, _ptr(offsets),
                  _ptr(up), codes.data_ptr(), scales.data_ptr(), _ptr(pre), s.act, _ptr(dx), _ptr(db), _ptr(ws))
        return dx, None, db, dy if need_r else None, None, None, None, None


def mx_linear(x, weight: MxTensor, bias=None, *, offsets=None, activation: str = "none", residual=None, dtype=None):
    """activation(x W^T + bias) + residual, [M, N], as expert_linear, over 4-bit weights: an MxTensor [E, N, K], or
    [N, K] without offsets. N is a multiple of 8, K of 32.

    x [M, K] is bfloat16, as are bias, residual and the result, and the products are bf16 ones of the exact weights:
    differentiable in x, bias and residual. Or x is an MxTensor [M, K]: products of 4-bit numbers, in bfloat16 or float32
    (dtype; bias and residual too), with a gradient of the residual alone. Sums are fp32."""
    if activation not in ACTIVATIONS:
        raise ModelError(f"activation must be one of {ACTIVATIONS}, got {activation!r}")
    _check_mx(weight, "weight")
    four = isinstance(x, MxTensor)
    if four:
        _check_mx(x, "x")
        rows, x_scales = x
        dtype = torch.bfloat16 if dtype is None else dtype
        _dtype_code(dtype)
    else:
        rows, x_scales = x, None
        if x.dtype != torch.bfloat16:
            raise ModelError(f"x must be bfloat16 or an MxTensor, got {x.dtype}")
        if dtype is not None and dtype != torch.bfloat16:
            raise ModelError(f"bfloat16 rows have bfloat16 results, got {dtype}")
        dtype = torch.bfloat16
    if rows.dim() != 2:
        raise ModelError(f"x must be [M, K], got {list(rows.shape)}")
    M, K = rows.shape[0], rows.shape[1] * (2 if four else 1)
    codes, scales = weight
    grouped = offsets is not None
    if not (codes.dim() == (3 if grouped else 2) and 2 * codes.shape[-1] == K):
        raise ModelError(f"weight must be {'[E, N' if grouped else '[N'}, {K}], got "
                         f"{list(codes.shape[:-1]) + [2 * codes.shape[-1]]}")
    groups, N = (codes.shape[0], codes.shape[1]) if grouped else (1, codes.shape[0])
    if not (N >= 8 and N % 8 == 0):
        raise ModelError(f"the output width must be a positive multiple of 8, got {N}")
    if grouped:
        if not 1 <= groups <= MAX_EXPERTS:
            raise ModelError(f"num_experts must be 1..{MAX_EXPERTS}, got {groups}")
        if not (offsets.dtype == torch.int32 and offsets.shape == (groups + 1,)):
            raise ModelError(f"offsets must be int32 [{groups + 1}], got {offsets.dtype} {list(offsets.shape)}")
    if bias is not None:
        want = (groups, N) if grouped else (N,)
        if bias.shape != want:
            raise ModelError(f"bias must be {list(want)}, got {list(bias.shape)}")
    if residual is not None and residual.shape != (M, N):
        raise ModelError(f"residual must be [{M}, {N}], got {list(residual.shape)}")
    for t in (bias, residual):
        if not (t is None or t.dtype == dtype):
            raise ModelError(f"bias and residual must be {dtype}, as the result")
    if four and bias is not None and torch.is_grad_enabled() and bias.requires_grad:
        raise ModelError("rows in 4 bits have no gradient of a bias: detach it")
    _on_device(rows, codes, scales, x_scales, bias, offsets, residual)
    s = _MxShape(M, K, N, groups, grouped, ACTIVATIONS.index(activation),
                 _lib.MOE_MX_ROWS_FOUR_BIT if four else _lib.MOE_MX_ROWS_BF16, dtype)
    offsets = offsets.contiguous() if grouped else None
    codes, scales = _ready(codes), scales.contiguous()
    x_scales = x_scales.contiguous() if four else None
    if _derivable(rows, bias, residual):
        return _MxLinear.apply(rows, x_scales, bias, residual, codes, scales, offsets, s)
    return _mx(_ready(rows), x_scales, codes, scales, _ready(bias), offsets, _ready(residual), s, False)[0]
