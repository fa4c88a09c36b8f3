"""Refusals of oxidizr_amd.ops and of their C entries, workspace sizes, and the reference forms
themselves, without a GPU."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from oxidizr_amd import _lib, ops
from oxidizr_amd.moe import ModelError
from tests import ops_ref as ref

F32, BF16 = _lib.MOE_DTYPE_F32, _lib.MOE_DTYPE_BF16
P = 1 << 20  # an aligned address that a refused call never touches


def fails(match, fn, *args, **kw):
    with pytest.raises(ModelError, match=match):
        fn(*args, **kw)


def order(T=4, k=2, E=3, dtype=torch.int32):
    return ops.TokenOrder(torch.zeros(E, dtype=dtype), torch.zeros(E + 1, dtype=dtype),
                          torch.zeros(T * k, dtype=dtype), torch.zeros(T, k, dtype=dtype))


def test_sort_refusals():
    fails("topk_idx must be", ops.sort_tokens, torch.zeros(4, dtype=torch.int32), 3)
    fails("int32 or int64", ops.sort_tokens, torch.zeros(4, 2), 3)
    fails("experts per token", ops.sort_tokens, torch.zeros(4, 17, dtype=torch.int32), 32)
    fails("experts per token", ops.sort_tokens, torch.zeros(4, 0, dtype=torch.int32), 32)
    for E in (0, 1025):
        fails("num_experts", ops.sort_tokens, torch.zeros(4, 2, dtype=torch.int32), E)
    fails("CUDA", ops.sort_tokens, torch.zeros(4, 2, dtype=torch.int32), 3)


def test_row_refusals():
    x = torch.zeros(4, 16)
    fails("TokenOrder", ops.permute_tokens, x, tuple(order()))
    fails("int32", ops.permute_tokens, x, order(dtype=torch.int64))
    fails("x must be", ops.permute_tokens, torch.zeros(5, 16), order())
    fails("multiple of 8", ops.permute_tokens, torch.zeros(4, 12), order())
    fails("unsupported", ops.permute_tokens, x.half(), order())
    fails("CUDA", ops.permute_tokens, x, order())
    fails("y must be", ops.unpermute_tokens, torch.zeros(7, 16), order())
    y = torch.zeros(8, 16)
    fails("weights must be", ops.unpermute_tokens, y, order(), torch.zeros(4, 3))
    fails("weights must be", ops.unpermute_tokens, y, order(), torch.zeros(4, 2, dtype=torch.bfloat16))
    fails("CUDA", ops.unpermute_tokens, y, order(), torch.zeros(4, 2))


def test_linear_refusals():
    x, w, off = torch.zeros(4, 16), torch.zeros(3, 8, 16), torch.zeros(4, dtype=torch.int32)
    lin = ops.expert_linear
    fails("activation", lin, x, w, offsets=off, activation="tanh")
    fails("x must be", lin, x[0], w, offsets=off)
    fails("weight must be", lin, x, w)                       # grouped weight without offsets
    fails("weight must be", lin, x, w[0], offsets=off)
    fails("weight must be", lin, x, torch.zeros(3, 8, 24), offsets=off)
    fails("multiples of 8", lin, x, torch.zeros(3, 12, 16), offsets=off)
    fails("multiples of 8", lin, torch.zeros(4, 20), torch.zeros(8, 20))
    fails("offsets must be", lin, x, w, offsets=off.long())
    fails("offsets must be", lin, x, w, offsets=off[:3])
    fails("num_experts", lin, x, torch.zeros(1025, 8, 16), offsets=torch.zeros(1026, dtype=torch.int32))
    fails("bias must be", lin, x, w, torch.zeros(8), offsets=off)
    fails("residual must be", lin, x, w, offsets=off, residual=torch.zeros(4, 16))
    fails("one dtype", lin, x, w.bfloat16(), offsets=off)
    fails("unsupported", lin, x.double(), w.double(), offsets=off)
    fails("CUDA", lin, x, w, offsets=off)


def test_norm_refusals():
    h, w = torch.zeros(4, 16), torch.ones(16)
    fails("multiple of 8", ops.rms_norm, torch.zeros(4, 12), torch.ones(12))
    fails("weight must be", ops.rms_norm, h, torch.ones(8))
    fails("one dtype", ops.rms_norm, h, w.bfloat16())
    fails("expected", ops.rms_norm, h[0], w)
    fails("y must be", ops.residual_norm, h, h[:2])
    fails("one dtype", ops.residual_norm, h, h.bfloat16())
    for gate in (torch.ones(4), torch.ones(1, 16), torch.ones(2, 1)):
        fails("gate must be", ops.residual_norm, h, h, gate=gate)
    fails("CUDA", ops.residual_norm, h, h, w)


def status(st, match):
    assert st != 0
    assert match in _lib.load().moe_last_error().decode(), _lib.load().moe_last_error()
    return st


def test_c_entries_refuse_before_any_device_call():
    L = _lib.load()

    def sort(T=4, k=2, E=3, nbytes=4, idx=P, counts=P, ws=P):
        return L.moe_sort_tokens(0, None, T, k, E, nbytes, idx, counts, P, P, P, ws)
    assert status(sort(T=-1), "num_tokens") == 1
    assert status(sort(k=17), "experts_per_tok") == 1
    assert status(sort(E=1025), "num_experts") == 1
    assert status(sort(T=2 ** 30), "2^31") == 4
    assert status(sort(nbytes=2), "index_bytes") == 1
    assert status(sort(idx=None), "NULL") == 1
    assert status(sort(counts=P + 2), "aligned") == 1
    assert status(sort(nbytes=8, idx=P + 4), "aligned") == 1
    assert status(sort(T=10 ** 6, ws=P + 8), "16-byte") == 1
    assert status(sort(T=10 ** 6, ws=None), "NULL") == 1

    def rows(fn, T=4, k=2, H=16, dtype=F32, x=P, kept=P, extra=(P,)):
        return fn(0, None, dtype, T, k, H, P, kept, x, *extra)
    for fn, extra in ((L.moe_permute, (P,)), (L.moe_unpermute, (None, P)),
                      (L.moe_unpermute_backward, (P, None, P, None))):
        assert status(rows(fn, H=12, extra=extra), "multiple of 8") == 1
        assert status(rows(fn, k=0, extra=extra), "experts_per_tok") == 1
        assert status(rows(fn, dtype=7, extra=extra), "dtype") == 1
        assert status(rows(fn, x=None, extra=extra), "NULL") == 1
        assert status(rows(fn, x=P + 8, extra=extra), "16-byte") == 1
        assert status(rows(fn, kept=None, extra=extra), "NULL") == 1
        assert rows(fn, T=0, extra=extra) == 0
    assert status(rows(L.moe_unpermute_backward, extra=(None, None, P, P)), "d_weights needs y") == 1

    def fwd(M=4, K=16, N=8, E=3, off=P, act=0, x=P, ws=P, dtype=F32):
        return L.moe_linear_forward(0, None, dtype, M, K, N, E, off, x, P, None, None, act, P, None, ws)

    def bwd(M=4, K=16, N=8, E=3, off=P, act=0, dy=P, pre=None, ws=P, dtype=F32):
        return L.moe_linear_backward(0, None, dtype, M, K, N, E, off, dy, P, P, pre, act, P, P, P, ws)
    for fn in (fwd, bwd):
        assert status(fn(M=-1), "num_rows") == 1
        assert status(fn(K=12), "multiples of 8") == 1
        assert status(fn(N=4), "multiples of 8") == 1
        assert status(fn(E=0), "num_groups") == 1
        assert status(fn(E=1025), "num_groups") == 1
        assert status(fn(off=None), "num_groups") == 1  # three groups without offsets
        assert status(fn(act=5), "activation") == 1
        assert status(fn(K=2 ** 15, N=2 ** 15), "weight matrix") == 4
        assert status(fn(K=8, N=2 ** 20 + 8), "above 1048576") == 4
        assert status(fn(M=2 ** 27), "rows") == 4
        assert status(fn(ws=P + 8), "16-byte") == 1
    assert status(bwd(M=2 ** 21, K=1024, dtype=BF16), "2^31") == 4
    assert status(fwd(ws=None), "NULL") == 1
    assert status(fwd(x=None), "NULL") == 1
    assert fwd(M=0) == 0

    def norm(T=4, H=16, h=P, y=P, w2=P, gate=None, kind=0, w3=P, scale=1.0, out=P, n=P, dtype=F32):
        return L.moe_residual_norm(0, None, dtype, T, H, h, y, w2, gate, kind, w3, scale, 1e-6, out, n, None, None)
    assert status(norm(H=12), "multiple of 8") == 1
    assert status(norm(H=32776), "above 32768") == 4
    assert status(norm(kind=4), "gate kind") == 1
    assert status(norm(kind=1), "do not go together") == 1
    assert status(norm(gate=P), "do not go together") == 1
    assert status(norm(y=None), "needs the block's output") == 1
    assert status(norm(y=None, w2=None, w3=None), "nothing to compute") == 1
    assert status(norm(y=None, w2=None, scale=0.5), "residual_scale") == 1
    assert status(norm(out=None), "NULL") == 1
    assert status(norm(n=None), "NULL") == 1
    assert status(norm(h=P + 4), "16-byte") == 1
    assert norm(T=0) == 0


def test_workspace_sizes():
    L = _lib.load()
    assert L.moe_sort_workspace_bytes(1024, 2, 1024) == 0          # one block
    assert L.moe_sort_workspace_bytes(8192, 8, 256) >= 32 * 257 * 4
    assert L.moe_sort_workspace_bytes(2 ** 24, 8, 64) == 512 * 65 * 4
    assert L.moe_sort_workspace_bytes(-1, 8, 64) == 0
    one = L.moe_linear_workspace_bytes(BF16, 4096, 512, 256, 1, 0, 0, 0)
    assert one == 0                                                # dense forward
    none = L.moe_linear_workspace_bytes(BF16, 4096, 512, 256, 8, 1, 0, 1)
    act = L.moe_linear_workspace_bytes(BF16, 4096, 512, 256, 8, 1, 1, 1)
    assert act - none == 4096 * 256 * 2                            # dz of an activation
    assert none >= (4096 // 64 + 8) * 256 * 4                      # the bias gradient's parts
    assert L.moe_linear_workspace_bytes(BF16, 4096, 500, 256, 8, 1, 0, 1) == 0
    assert L.moe_residual_norm_workspace_bytes(10 ** 6, 2048) == 1024 * 2 * 2048 * 4
    assert L.moe_residual_norm_workspace_bytes(3, 2048) == 3 * 2 * 2048 * 4


def test_reference_gradients_are_autograds():
    g = torch.Generator().manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64).requires_grad_()
    for act in ops.ACTIVATIONS:
        x, w, b, r = normal(9, 16), normal(3, 8, 16), normal(3, 8), normal(9, 8)
        off, dy = torch.tensor([0, 2, 2, 8]), normal(9, 8).detach()
        want = ref.linear(*(t.detach() for t in (x, w, b)), off, act, r.detach(), dy, torch.float32)
        f = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu,
             "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[act]
        y = torch.cat([f(x[off[e]:off[e + 1]] @ w[e].t() + b[e]) for e in range(3)] +
                      [torch.zeros(1, 8, dtype=torch.float64)]) + r
        got = torch.autograd.grad(y, [x, w, b, r], dy)
        for n, t in zip(("y", "dx", "dw", "db", "dr"), (y,) + got):
            assert torch.allclose(t, want[n][0], atol=1e-12), (act, n)
    h, y, w2, w3 = normal(5, 16), normal(5, 16), normal(16), normal(16)
    dh, dn = normal(5, 16).detach(), normal(5, 16).detach()
    for gate in (normal(16), normal(5, 1), normal(5, 16)):
        want = ref.norm(*(t.detach() for t in (h, y, w2, gate, w3)), 0.75, 1e-5, dh, dn, torch.float32)
        out = 0.75 * h + gate * torch.nn.functional.rms_norm(y, (16,), w2, 1e-5)
        n = torch.nn.functional.rms_norm(out, (16,), w3, 1e-5)
        got = torch.autograd.grad((out, n), [h, y, w2, gate, w3], (dh, dn))
        for name, t in zip(("h", "n", "dh", "dy", "dw2", "dgate", "dw3"), (out, n) + got):
            assert torch.allclose(t, want[name][0], atol=1e-10), name


def test_a_bound_that_is_passed_is_seen():
    a = torch.ones(4)
    ref.assert_close(a, a.double() * (1 + 2.0 ** -25), torch.zeros(4), "a")
    with pytest.raises(AssertionError):
        ref.assert_close(a, a.double() * (1 + 2.0 ** -22), torch.zeros(4, dtype=torch.float64), "a")


def test_a_linear_whose_backward_would_be_refused_is_refused_at_once():
    x = torch.zeros(1, 1024).expand(1 << 19, 1024)
    w = torch.zeros(8, 1024, requires_grad=True)
    fails("reach 2\\^31 bytes", ops.expert_linear, x, w)
    with torch.no_grad():
        fails("CUDA", ops.expert_linear, x, w)  # a forward alone takes them


def test_rms_norm_needs_a_weight():
    fails("needs a weight", ops.rms_norm, torch.zeros(2, 64), None)


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_workspace_of_a_linear_without_rows():
    # in a process of its own: a division by zero would end it
    code = """
from oxidizr_amd import _lib
L = _lib.load()
for dtype in (_lib.MOE_DTYPE_F32, _lib.MOE_DTYPE_BF16):
    for K, N in ((8, 8), (64, 64), (2048, 1408), (8, 1 << 20)):
        for act in range(5):
            for backward in (0, 1):
                assert L.moe_linear_workspace_bytes(dtype, 0, K, N, 1, 0, act, backward) == 0
                for E in (1, 3, 1024):
                    assert L.moe_linear_workspace_bytes(dtype, 0, K, N, E, 1, act, backward) > 0
print("done")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "done" in r.stdout, (r.returncode, r.stderr[-500:])


def test_norm_backward_entries_refuse_before_any_device_call():
    L = _lib.load()
    for entry in (L.moe_residual_norm_backward, L.moe_residual_norm_backward_from_input):
        def bwd(T=4, H=16, d_out=P, d_n=P, h=P, y=P, w2=P, gate=None, kind=0, w3=P, r2=P, r3=P, dw2=P, dgate=None,
                dw3=P, ws=P, dtype=F32):
            return entry(0, None, dtype, T, H, d_out, d_n, h, y, w2, gate, kind, w3, 1.0, r2, r3, P, P, dw2, dgate,
                         dw3, ws)
        assert status(bwd(H=12), "multiple of 8") == 1
        assert status(bwd(dtype=7), "dtype") == 1
        assert status(bwd(kind=2), "do not go together") == 1
        assert status(bwd(kind=2, gate=P), "NULL") == 1
        for missing in ("h", "r2", "r3", "d_n", "dw2", "dw3", "ws"):
            assert status(bwd(**{missing: None}), "NULL") == 1
        assert status(bwd(h=P + 8), "16-byte") == 1


# ---- forward-mode derivatives and traces: nothing may come back without them

def calls(t, order_=None):
    """One call of each operator on tensors made by t(shape), by name."""
    o = order_ or order()
    return {
        "permute": lambda x: ops.permute_tokens(x, o),
        "unpermute": lambda x: ops.unpermute_tokens(torch.cat([x, x]), o, t(4, 2)),
        "weights": lambda x: ops.unpermute_tokens(t(8, 16), o, x[:, :2].contiguous()),
        "linear": lambda x: ops.expert_linear(x, t(8, 16)),
        "residual": lambda x: ops.expert_linear(t(4, 16), t(16, 16), residual=x),
        "rms_norm": lambda x: ops.rms_norm(x, t(16)),
        "norm weight": lambda x: ops.rms_norm(t(4, 16), x[0].contiguous()),
        "residual_norm": lambda x: ops.residual_norm(t(4, 16), x, t(16)),
    }


@pytest.mark.parametrize("name", sorted(calls(None)))
def test_forward_mode_is_refused(name, monkeypatch):
    monkeypatch.setattr(ops, "_on_device", lambda *a: 0)
    monkeypatch.setattr(ops, "_call", lambda *a: None)  # the library is not reached
    call = calls(torch.ones)[name]
    with torch.autograd.forward_ad.dual_level():
        x = torch.autograd.forward_ad.make_dual(torch.ones(4, 16), torch.ones(4, 16))
        assert not x.requires_grad
        with pytest.raises(NotImplementedError, match="forward mode"):
            call(x)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
            call(x)
        call(torch.ones(4, 16))  # without a derivative there is nothing to lose


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", sorted(calls(None)))
def test_traces_are_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    call = calls(torch.ones)[name]
    x = torch.ones(4, 16)
    for leaf in (x, x.clone().requires_grad_()):
        fails("traced", torch.jit.trace, call, leaf, check_trace=False)
        for pre in (False, True):
            fails("traced", make_fx(call, pre_dispatch=pre), leaf)
    fails("CUDA", call, x)  # and outside a trace the call is looked at as before


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_sorting_is_not_traced():
    from torch.fx.experimental.proxy_tensor import make_fx
    idx = torch.zeros(4, 2, dtype=torch.int32)
    fails("traced", torch.jit.trace, lambda i: ops.sort_tokens(i, 3).perm, idx, check_trace=False)
    fails("traced", make_fx(lambda i: ops.sort_tokens(i, 3).perm), idx)


def test_other_modes_are_no_trace():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Count(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with Count():
        fails("CUDA", ops.rms_norm, torch.ones(4, 16), torch.ones(16))


def test_only_the_weights_gradient_is_refused_past_2_31_bytes():
    x = torch.zeros(1, 1024).expand(1 << 19, 1024)
    w, b = torch.zeros(8, 1024), torch.zeros(8, requires_grad=True)
    r = torch.zeros(1 << 19, 8, requires_grad=True)
    fails("reach 2\\^31 bytes", ops.expert_linear, x, w.clone().requires_grad_())
    for kw in ({"bias": b}, {"residual": r}):
        fails("CUDA", ops.expert_linear, x, w, **kw)  # taken, as far as the device
    L, M, K = _lib.load(), 2 ** 21, 1024
    assert status(L.moe_linear_backward(0, None, BF16, M, K, 8, 3, P, P, P, P, None, 0, P, P, P, P), "2^31") == 4
    assert status(L.moe_linear_backward(0, None, BF16, M, K, 8, 3, P, None, P, P, None, 0, P, None, P, P), "NULL") == 1


def test_linears_of_more_tiles_than_a_launch_are_refused_at_once():
    L, N = _lib.load(), 1 << 20
    fwd, bwd = L.moe_linear_forward, L.moe_linear_backward

    def forward(dtype, M, K, N, E):
        return fwd(0, None, dtype, M, K, N, E, P, P, P, None, None, 0, P, None, P)

    def backward(dtype, M, K, N, E, dx=P, dw=P):
        return bwd(0, None, dtype, M, K, N, E, P, P, P, P, None, 0, dx, dw, None, P)
    # fp32: 16384 column tiles of 64, and as many weight tiles to an expert
    assert status(forward(F32, 2000, 8, N, 1024), "too many rows or tiles") == 4
    assert L.moe_linear_workspace_bytes(F32, 2000, 8, N, 1024, 1, 0, 0) == 0
    assert status(fwd(0, None, F32, 2000, 8, N, 1024, P, P, P, None, None, 0, P, None, None), "too many") == 4
    assert status(backward(F32, 100, 8, N, 1024), "too many rows or tiles") == 4
    assert L.moe_linear_workspace_bytes(F32, 100, 8, N, 1024, 1, 0, 1) == 0
    assert status(backward(F32, 2000, N, 8, 1024, dw=None), "too many rows or tiles") == 4
    assert L.moe_linear_workspace_bytes(F32, 100, 8, N, 1000, 1, 0, 1) > 0  # just below
