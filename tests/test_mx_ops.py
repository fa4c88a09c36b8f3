"""Refusals of router_losses, of 4-bit numbers and the products over them, and of their C entries; and the reference
forms themselves, without a GPU."""
import pytest
import torch

from oxidizr_amd import _lib, ops
from oxidizr_amd.moe import ModelError
from tests import mx_ref

F32, BF16 = _lib.MOE_DTYPE_F32, _lib.MOE_DTYPE_BF16
ROWS_BF16, ROWS_FOUR = _lib.MOE_MX_ROWS_BF16, _lib.MOE_MX_ROWS_FOUR_BIT
P = 1 << 20  # an aligned address that a refused call never touches


def fails(match, fn, *args, **kw):
    with pytest.raises(ModelError, match=match):
        fn(*args, **kw)


def four(*shape):
    return ops.MxTensor(torch.zeros(*shape[:-1], shape[-1] // 2, dtype=torch.uint8),
                        torch.zeros(*shape[:-1], shape[-1] // 32, dtype=torch.uint8))


def test_router_refusals():
    x, i = torch.zeros(4, 6), torch.zeros(4, 2, dtype=torch.int32)
    f = ops.router_losses
    fails("logits must be", f, x[0], i)
    fails("topk_idx must be", f, x, i[:3])
    fails("topk_idx must be", f, x, i[:, 0])
    fails("int32 or int64", f, x, i.float())
    fails("experts per token", f, x, torch.zeros(4, 17, dtype=torch.int32))
    fails("num_experts", f, torch.zeros(4, 1025), i)
    fails("num_experts", f, torch.zeros(4, 0), i)
    fails("score", f, x, i, score="tanh")
    for tau in (0.0, -1.0, float("inf"), float("nan")):
        fails("temperature", f, x, i, temperature=tau)
    fails("offsets must be", f, x, i, offsets=torch.zeros(3, dtype=torch.int64))
    fails("offsets must be", f, x, i, offsets=torch.zeros(0, dtype=torch.int32))
    fails("offsets must be", f, x, i, offsets=torch.zeros(2, 2, dtype=torch.int32))
    fails("sequences", f, x, i, offsets=torch.zeros(1, dtype=torch.int32).expand(2 ** 22 + 1))
    fails("unsupported", f, x.double(), i)
    fails("CUDA", f, x, i)


def test_quantize_refusals():
    fails("multiple of 32", ops.quantize_mxfp4, torch.zeros(4, 40))
    fails("multiple of 32", ops.quantize_mxfp4, torch.zeros(4, 0))
    fails("multiple of 32", ops.quantize_mxfp4, torch.zeros(()))
    fails("unsupported", ops.quantize_mxfp4, torch.zeros(4, 32).half())
    fails("CUDA", ops.quantize_mxfp4, torch.zeros(4, 32))
    q = four(4, 64)
    fails("must be an MxTensor", ops.dequantize_mxfp4, tuple(q))
    fails("uint8", ops.dequantize_mxfp4, ops.MxTensor(q.codes.int(), q.scales))
    for bad in (ops.MxTensor(q.codes, q.scales[:3]), ops.MxTensor(q.codes[:, :31], q.scales), ops.MxTensor(q.codes[0], q.scales),
                ops.MxTensor(q.codes[:, :0], q.scales[:, :0])):
        fails("do not go together", ops.dequantize_mxfp4, bad)
    fails("unsupported", ops.dequantize_mxfp4, q, dtype=torch.half)
    fails("CUDA", ops.dequantize_mxfp4, q)


def test_linear_refusals():
    x, w, off = torch.zeros(4, 64, dtype=torch.bfloat16), four(3, 8, 64), torch.zeros(4, dtype=torch.int32)
    f = ops.mx_linear
    fails("activation", f, x, w, offsets=off, activation="tanh")
    fails("must be an MxTensor", f, x, tuple(w), offsets=off)
    fails("do not go together", f, x, ops.MxTensor(w.codes, w.scales[:2]), offsets=off)
    fails("bfloat16 or an MxTensor", f, x.float(), w, offsets=off)
    fails("bfloat16 results", f, x, w, offsets=off, dtype=torch.float32)
    fails("unsupported", f, four(4, 64), w, offsets=off, dtype=torch.half)
    fails("x must be", f, x[0], w, offsets=off)
    fails("x must be", f, four(2, 4, 64), w, offsets=off)
    fails("weight must be", f, x, w)
    fails("weight must be", f, x, four(8, 64), offsets=off)
    fails("weight must be", f, x, four(3, 8, 96), offsets=off)
    fails("weight must be", f, four(4, 32), w, offsets=off)
    fails("multiple of 8", f, x, four(3, 12, 64), offsets=off)
    fails("offsets must be", f, x, w, offsets=off.long())
    fails("offsets must be", f, x, w, offsets=off[:3])
    fails("num_experts", f, x, four(1025, 8, 64), offsets=torch.zeros(1026, dtype=torch.int32))
    fails("bias must be", f, x, w, torch.zeros(8, dtype=torch.bfloat16), offsets=off)
    fails("residual must be", f, x, w, offsets=off, residual=torch.zeros(4, 16, dtype=torch.bfloat16))
    fails("as the result", f, x, w, torch.zeros(3, 8), offsets=off)
    fails("as the result", f, four(4, 64), w, torch.zeros(3, 8), offsets=off)
    fails("no gradient of a bias", f, four(4, 64), w, torch.zeros(3, 8, dtype=torch.bfloat16, requires_grad=True), offsets=off)
    fails("CUDA", f, x, w, offsets=off)
    fails("CUDA", f, four(4, 64), w, offsets=off)


def status(st, match):
    assert st != 0
    assert match in _lib.load().moe_last_error().decode(), _lib.load().moe_last_error()
    return st


def test_c_entries_refuse_before_any_device_call():
    L = _lib.load()

    def losses(T=4, E=6, k=2, nbytes=4, dtype=F32, x=P, idx=P, score=0, tau=1.0, off=None, S=1, out=P, ws=P):
        return L.moe_router_losses(0, None, dtype, T, E, k, nbytes, x, idx, score, tau, 1.0, 1.0, off, S, out, P, P, None,
                                   None, ws)

    def losses_bwd(T=4, E=6, k=2, nbytes=4, dtype=F32, x=P, idx=P, score=0, tau=1.0, off=None, S=1, out=P):
        return L.moe_router_losses_backward(0, None, dtype, T, E, k, nbytes, x, idx, score, tau, off, S, P, P, P, P, out)
    for f in (losses, losses_bwd):
        assert status(f(T=-1), "num_tokens") == 1
        assert status(f(T=2 ** 31), "num_tokens") == 1
        assert status(f(T=2 ** 30, k=2), "2^31") == 4
        assert status(f(E=0), "num_experts") == 1
        assert status(f(E=1025), "num_experts") == 1
        assert status(f(k=17), "experts_per_tok") == 1
        assert status(f(nbytes=2), "index_bytes") == 1
        assert status(f(dtype=5), "dtype") == 1
        assert status(f(score=2), "score") == 1
        for tau in (0.0, -1.0, float("inf"), float("nan")):
            assert status(f(tau=tau), "temperature") == 1
        assert status(f(S=2), "num_sequences") == 1
        assert status(f(off=P, S=-1), "num_sequences") == 1
        assert status(f(off=P, S=2 ** 22), "2^22") == 4
        assert status(f(off=P + 2), "aligned") == 1
        assert status(f(x=None), "NULL") == 1
        assert status(f(x=P + 8), "16-byte") == 1
        assert status(f(idx=P + 2), "aligned") == 1
        assert status(f(nbytes=8, idx=P + 4), "aligned") == 1
        assert status(f(out=None), "NULL") == 1
    assert status(losses(ws=None), "NULL") == 1
    assert losses(off=P, S=0) == 0
    assert losses_bwd(T=0) == 0

    for f in (L.moe_mx_quantize, L.moe_mx_dequantize):
        for args, match, code in (((7, 4, P, P, P), "dtype", 1), ((F32, -1, P, P, P), "num_blocks", 1),
                                  ((F32, 2 ** 29, P, P, P), "2^29", 4), ((F32, 4, None, P, P), "NULL", 1),
                                  ((F32, 4, P + 8, P, P), "16-byte", 1)):
            assert status(f(0, None, *args), match) == code
        assert f(0, None, F32, 0, None, None, None) == 0
    assert status(L.moe_mx_quantize(0, None, F32, 4, P, P, None), "NULL") == 1
    assert status(L.moe_mx_dequantize(0, None, F32, 4, P, None, P), "NULL") == 1

    def fwd(M=4, K=64, N=8, E=3, off=P, act=0, x=P, xs=None, wc=P, wsc=P, rows=ROWS_BF16, dtype=BF16, y=P):
        return L.moe_mx_linear_forward(0, None, rows, dtype, M, K, N, E, off, x, xs, wc, wsc, None, None, act, y, None)

    def bwd(M=4, K=64, N=8, E=3, off=P, act=0, x=P, pre=None, wc=P, wsc=P, ws=P):
        return L.moe_mx_linear_backward(0, None, M, K, N, E, off, x, wc, wsc, pre, act, P, P, ws)
    for f in (fwd, bwd):
        assert status(f(M=-1), "num_rows") == 1
        for K in (0, 16, 40):
            assert status(f(K=K), "multiple of 32") == 1
        assert status(f(N=12), "multiple of 8") == 1
        assert status(f(E=0), "num_groups") == 1
        assert status(f(E=1025), "num_groups") == 1
        assert status(f(off=None), "num_groups") == 1
        assert status(f(act=5), "activation") == 1
        assert status(f(K=2 ** 15, N=2 ** 15), "2^30 elements") == 4
        assert status(f(N=2 ** 20 + 8), "above 1048576") == 4
        assert status(f(M=2 ** 27), "rows") == 4
        assert status(f(M=2 ** 26, K=256), "2^34") == 4
        assert status(f(x=None), "NULL") == 1
        assert status(f(wc=P + 8), "16-byte") == 1
        assert status(f(wsc=None), "NULL") == 1
        assert status(f(off=P + 2), "aligned") == 1
    assert status(bwd(ws=P + 8), "16-byte") == 1
    assert status(bwd(ws=None), "NULL") == 1
    assert status(fwd(y=None), "NULL") == 1
    assert fwd(M=0) == 0
    assert status(fwd(rows=2), "row format") == 1
    assert status(fwd(dtype=F32), "bf16 results") == 1
    assert status(fwd(rows=ROWS_FOUR, dtype=3), "dtype") == 1
    assert status(fwd(rows=ROWS_FOUR), "NULL") == 1           # without the rows' scales
    assert status(bwd(act=2), "pre_act") == 1


def test_workspace_sizes():
    L = _lib.load()
    ws = L.moe_mx_linear_workspace_bytes
    none, act = (ws(4096, 512, 256, 8, 1, a) for a in (0, 1))
    assert act - none == 4096 * 256 * 2 and none >= (4096 // 64 + 8) * 256 * 4
    assert ws(4096, 500, 256, 8, 1, 0) == 0
    assert ws(2 ** 27, 512, 256, 8, 1, 0) == 0
    r = L.moe_router_losses_workspace_bytes
    assert r(8192, 256, 1) >= 257 * 256 * 8 and r(0, 8, 1) > 0 and r(8, 0, 1) == 0 and r(8, 8, -1) == 0


def test_reference_quantisation():
    # by hand: borders, ties to even, saturation, signs, zeros, and the exponent of the largest
    x = torch.zeros(2, 32)
    x[0, :9] = torch.tensor([7.9, 0.25, 0.75, -1.25, 1.75, 2.5, 3.5, 5.0, -0.0])
    x[1, 0] = 2.0 ** -126
    codes, scales = mx_ref.quantize(x)
    assert scales[:, 0].tolist() == [127, 0]
    got = mx_ref.values(codes, scales)[0, :9].tolist()
    assert got == [6.0, 0.0, 1.0, -1.0, 2.0, 2.0, 4.0, 4.0, 0.0]
    assert mx_ref.values(codes, scales)[1, 0] == 2.0 ** -126
    x[1, 3] = float("nan")
    codes, scales = mx_ref.quantize(x)
    assert int(scales[1, 0]) == 255 and bool(mx_ref.values(codes, scales)[1].isnan().all())
    # no number is nearer than the one chosen
    g = torch.Generator().manual_seed(1)
    x = torch.randn(64, 32, generator=g, dtype=torch.float64)
    codes, scales = mx_ref.quantize(x)
    s = torch.exp2(scales.double() - 127)
    best = ((x.abs() / s)[..., None] - mx_ref.GRID).abs().amin(-1) * s
    assert torch.equal((mx_ref.values(codes, scales) - x).abs() <= best * (1 + 1e-15), torch.ones(64, 32, dtype=torch.bool))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_reference_losses_are_autograds(score):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(20, 7, generator=g, dtype=torch.float64).requires_grad_()
    idx = torch.randint(-1, 8, (20, 2), generator=g)
    idx[3] = -1
    off = torch.tensor([2, 9, 9, 18], dtype=torch.int32)
    up = torch.rand(2, 3, generator=g, dtype=torch.float64)
    want = mx_ref.losses(x.detach(), idx, score, 0.7, 1.5, 0.5, off, up[0], up[1])
    total = 0.0
    for s, (a, b) in enumerate(((2, 9), (9, 9), (9, 18))):
        keep = [t for t in range(a, b) if any(0 <= e < 7 for e in idx[t].tolist())]
        if not keep:
            assert float(want["balance"][0][s]) == 0 and float(want["z"][0][s]) == 0
            continue
        l = x[keep] / 0.7
        q = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l) / torch.sigmoid(l).sum(1, keepdim=True)
        m = torch.tensor([sum(int(e == j) for t in keep for e in idx[t].tolist()) for j in range(7)], dtype=torch.float64)
        assert torch.equal(want["counts"][s].double(), m)
        P, f = q.mean(0), m / (2 * len(keep))
        balance, z = 7 * (1.5 * f * P + 0.5 * P * P).sum(), torch.logsumexp(l, 1).square().mean()
        assert abs(float((want["balance"][0][s] - balance).detach())) < 1e-12
        assert abs(float((want["z"][0][s] - z).detach())) < 1e-12
        total = total + up[0, s] * balance + up[1, s] * z
    d, = torch.autograd.grad(total, x)
    assert torch.allclose(d, want["d"][0], atol=1e-13)
