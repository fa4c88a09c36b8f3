"""The router's losses and 4-bit products together with the operators around them, as a layer uses them: adapters trained over
frozen 4-bit experts, and decoding with both sides in 4 bits; captured, on streams, over ranges of experts, views and large tensors."""
import threading

import pytest
import torch

from oxidizr_amd import ops
from oxidizr_amd.moe import ModelError
from tests import mx_ref, ops_ref
from tests.test_gpu_ops import gen, normal

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def inputs(seed, T, H, I, E, R=8):
    """Frozen 4-bit experts H -> I -> H, trained biases and an adapter of rank R beside the first product."""
    g = gen(seed)
    q1, q2 = (ops.MxTensor(*mx_ref.quantize(normal(g, E, n, k, std=k ** -0.5))) for n, k in ((I, H), (H, I)))
    leaves = {"x": normal(g, T, H, dtype=BF16), "logits": normal(g, T, E), "b1": normal(g, E, I, dtype=BF16, std=0.1),
              "down": normal(g, E, R, H, dtype=BF16, std=H ** -0.5), "up": normal(g, E, I, R, dtype=BF16, std=R ** -0.5),
              "b2": normal(g, E, H, dtype=BF16, std=0.1)}
    return q1, q2, leaves


def layer(q1, q2, p, k, pad, four=False):
    E = p["logits"].shape[1]
    top, idx = torch.topk(p["logits"], k, dim=1)
    idx = torch.where(pad[:, None], -1, idx)
    losses = ops.router_losses(p["logits"], idx)
    order = ops.sort_tokens(idx, E)
    rows = ops.permute_tokens(p["x"], order)
    first = ops.quantize_mxfp4(rows) if four else rows
    a = ops.mx_linear(first, q1, p["b1"], offsets=order.offsets)
    low = ops.expert_linear(rows, p["down"], offsets=order.offsets)
    a = ops.expert_linear(low, p["up"], offsets=order.offsets, residual=a)
    second = ops.quantize_mxfp4(a) if four else a
    b = ops.mx_linear(second, q2, p["b2"], offsets=order.offsets, activation="silu")
    y = ops.unpermute_tokens(b, order, torch.softmax(top, 1))
    return y, losses


def dense(q1, q2, p, k, pad):
    """The same in float64, every expert on every token."""
    q = {n: t.detach().double().requires_grad_(t.requires_grad) for n, t in p.items()}
    w1, w2 = mx_ref.values(*q1), mx_ref.values(*q2)
    E = q["logits"].shape[1]
    idx = torch.topk(p["logits"], k, dim=1).indices
    top = q["logits"].gather(1, idx)
    real = ~pad
    a = torch.stack([q["x"] @ w1[e].t() + q["b1"][e] + q["x"] @ q["down"][e].t() @ q["up"][e].t() for e in range(E)])
    b = torch.nn.functional.silu(torch.stack([a[e] @ w2[e].t() + q["b2"][e] for e in range(E)]))
    w = torch.zeros_like(q["logits"]).scatter(1, idx, torch.softmax(top, 1)) * real[:, None]
    y = (w.t()[..., None] * b).sum(0)
    prob = torch.softmax(q["logits"], 1)[real].mean(0)
    counts = torch.bincount(idx[real].flatten(), minlength=E)
    f = counts.double() / (k * int(real.sum()))
    balance = E * (f * prob + prob * prob).sum()
    z = torch.logsumexp(q["logits"], 1)[real].square().mean()
    return y, balance, z, counts, q


def rel(got, want):
    return float((got.double() - want).norm() / want.norm())


def test_training_over_frozen_experts():
    T, H, I, E, k = 700, 288, 160, 6, 2
    q1, q2, p = inputs(1, T, H, I, E)
    pad = torch.rand(T, device="cuda", generator=gen(2)) < 0.1
    for t in p.values():
        t.requires_grad_()
    y, losses = layer(q1, q2, p, k, pad)
    dy = normal(gen(3), T, H, dtype=BF16)
    loss = (y.float() * dy.float()).sum() + 3.0 * losses.balance + 0.5 * losses.z
    got = dict(zip(p, torch.autograd.grad(loss, list(p.values()))))
    wy, wb, wz, counts, q = dense(q1, q2, p, k, pad)
    want = dict(zip(q, torch.autograd.grad((wy * dy.double()).sum() + 3.0 * wb + 0.5 * wz, list(q.values()))))
    assert torch.equal(losses.counts.long(), counts)
    assert abs(float((losses.balance - wb).detach())) < 1e-5 * float(wb.detach())
    assert abs(float((losses.z - wz).detach())) < 1e-5 * float(wz.detach())
    # at most ten roundings to bf16 lie between an input and any of these, each 2^-8 of the value at most
    assert rel(y.detach(), wy.detach()) < 10 * 2.0 ** -8
    for n in p:
        assert rel(got[n], want[n]) < 10 * 2.0 ** -8, n
    assert bool((y.detach()[pad] == 0).all()) and bool((got["x"][pad] == 0).all())


def test_decoding_in_four_bits():
    T, H, I, E, k = 16, 512, 256, 12, 3
    q1, q2, p = inputs(4, T, H, I, E)
    pad = torch.zeros(T, dtype=torch.bool, device="cuda")
    with torch.no_grad():
        y, _ = layer(q1, q2, p, k, pad, four=True)
        exact, _ = layer(q1, q2, p, k, pad)
    # a 4-bit number is off by a sixth of itself at most beyond saturation's quarter; rms over N(0, 1) is about 0.1
    assert 0.02 < rel(y, exact.double()) < 0.4
    again, _ = layer(q1, q2, p, k, pad, four=True)
    assert torch.equal(y, again)


@pytest.mark.parametrize("T", [5, 600])
@pytest.mark.parametrize("four", [False, True])
def test_replayed_graph_gives_the_eager_results(T, four):
    H, I, E, k = 288, 160, 9, 3
    q1, q2, p = inputs(T, T, H, I, E)
    pad = torch.rand(T, device="cuda", generator=gen(T)) < 0.1
    leaves = list(p.values())
    if not four:
        for t in leaves:
            t.requires_grad_()
    dy = normal(gen(7), T, H, dtype=BF16)

    def step():
        if four:
            with torch.no_grad():
                y, losses = layer(q1, q2, p, k, pad, four=True)
            return (y,) + tuple(losses)
        y, losses = layer(q1, q2, p, k, pad)
        one = torch.ones((), device="cuda")
        return ((y.detach(),) + tuple(t.detach() for t in losses) +
                torch.autograd.grad((y, losses.balance, losses.z), leaves, (dy, one, one)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        new1, new2, q = inputs(100 + seed, T, H, I, E)
        with torch.no_grad():
            for a, b in zip(leaves + list(q1) + list(q2), list(q.values()) + list(new1) + list(new2)):
                a.copy_(b)
            pad.copy_(torch.rand(T, device="cuda", generator=gen(seed)) < 0.1 * seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = step()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (seed, i)


def test_threads_with_streams_of_their_own():
    T, H, I, E, k = 400, 288, 160, 6, 2
    cases = [inputs(50 + i, T, H, I, E) for i in range(3)]
    pad = torch.zeros(T, dtype=torch.bool, device="cuda")
    dy = normal(gen(8), T, H, dtype=BF16)

    def step(c):
        q1, q2, p = c
        q = {n: t.detach().requires_grad_() for n, t in p.items()}
        y, losses = layer(q1, q2, q, k, pad)
        return [y.detach()] + list(torch.autograd.grad((y, losses.z), list(q.values()), (dy, torch.ones_like(losses.z))))
    want = [step(c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 3, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = step(cases[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("M", [40, 1500])
@pytest.mark.parametrize("four", [False, True])
def test_a_range_of_the_experts(four, M):
    E, K, N = 7, 160, 136
    g = gen(M)
    sizes = torch.multinomial(torch.ones(E), M, replacement=True, generator=torch.Generator().manual_seed(M)).bincount(minlength=E)
    offsets = torch.cat((sizes.new_zeros(1), sizes.cumsum(0))).to(torch.int32).cuda()
    w = ops.quantize_mxfp4(normal(g, E, N, K, dtype=BF16, std=K ** -0.5))
    x, b, r = normal(g, M, K, dtype=BF16), normal(g, E, N, dtype=BF16), normal(g, M, N, dtype=BF16)
    rows = ops.quantize_mxfp4(x) if four else x
    whole = ops.mx_linear(rows, w, b, offsets=offsets, residual=r)
    total = r.float() * 0
    for a, c in ((0, 2), (2, 3), (3, 7)):
        part = ops.mx_linear(rows, ops.MxTensor(w.codes[a:c], w.scales[a:c]), b[a:c], offsets=offsets[a:c + 1], residual=r)
        lo, hi = int(offsets[a]), int(offsets[c])
        assert torch.equal(part[:lo], r[:lo]) and torch.equal(part[hi:], r[hi:])
        total[lo:hi] = part[lo:hi].float()
        if not four:
            xg = x.clone().requires_grad_()
            y = ops.mx_linear(xg, ops.MxTensor(w.codes[a:c], w.scales[a:c]), offsets=offsets[a:c + 1], activation="silu")
            d, = torch.autograd.grad(y, xg, r)
            assert bool((d[:lo] == 0).all()) and bool((d[hi:] == 0).all())
    # the stream of few rows may take another number of waves for a range: sums in another order, one rounding apart
    assert bool(((total - whole.float()).abs() <= 2.0 ** -7 * whole.float().abs() + 2.0 ** -8 * r.float().abs() + 1e-3).all())


@pytest.mark.parametrize("M", [9, 600])
def test_views_and_broadcasts(M):
    g = gen(M)
    K, N = 96, 72
    w = ops.quantize_mxfp4(normal(g, N, 2 * K, dtype=BF16))
    wide = normal(g, 2 * M, K + 40, dtype=BF16)
    half = ops.MxTensor(w.codes[:, :K // 2], w.scales[:, :K // 32])           # a part of the input width
    whole = ops.MxTensor(half.codes.contiguous(), half.scales.contiguous())
    bias, one = normal(g, N + 3, dtype=BF16)[3:], normal(g, N, dtype=BF16)
    for x in (wide[::2, 8:8 + K], wide[1:M + 1, 1:1 + K], wide[:1, :K].expand(M, K), wide.t().contiguous().t()[:M, :K]):
        got = ops.mx_linear(x, half, bias, residual=one.expand(M, N))
        want = ops.mx_linear(x.contiguous(), whole, bias.clone(), residual=one.expand(M, N).contiguous())
        assert torch.equal(got, want)
    q = ops.quantize_mxfp4(wide[:M, :K])
    strided = ops.MxTensor(torch.cat((q.codes, q.codes), 1)[:, :K // 2], torch.cat((q.scales, q.scales), 1)[:, :K // 32])
    assert torch.equal(ops.mx_linear(strided, whole), ops.mx_linear(q, whole))
    x = wide[:M, :K].clone().requires_grad_()
    r = normal(g, N, dtype=BF16).requires_grad_()
    y = ops.mx_linear(x, whole, residual=r.expand(M, N))
    dx, dr = torch.autograd.grad(y.sum(), (x, r))                               # an upstream gradient of stride 0
    ones = torch.ones(M, N, dtype=torch.float64, device="cuda")
    ref = ops_ref.linear(x.detach().double(), mx_ref.values(*whole), None, None, "none", None, ones, BF16)
    ops_ref.assert_close(dx, *ref["dx"], "dx")
    assert bool((dr == M).all())


def test_a_gradient_alone():
    g = gen(21)
    x, b, r = normal(g, 70, 64, dtype=BF16), normal(g, 2, 16, dtype=BF16), normal(g, 70, 16, dtype=BF16)
    w = ops.quantize_mxfp4(normal(g, 2, 16, 64, dtype=BF16, std=0.2))
    off = torch.tensor([0, 30, 66], dtype=torch.int32, device="cuda")
    dy = normal(g, 70, 16, dtype=BF16)

    def grads(*which):
        t = {"x": x.clone(), "b": b.clone(), "r": r.clone()}
        leaves = [t[n].requires_grad_() for n in which]
        y = ops.mx_linear(t["x"], w, t["b"], offsets=off, activation="gelu", residual=t["r"])
        return dict(zip(which, torch.autograd.grad(y, leaves, dy)))
    full = grads("x", "b", "r")
    for which in (("x",), ("b",), ("r",), ("x", "r"), ("b", "r")):
        for n, t in grads(*which).items():
            assert torch.equal(t, full[n]), (which, n)
    assert bool((full["x"][66:] == 0).all()) and torch.equal(full["r"], dy)


def test_written_weights_are_told_before_a_backward():
    x = torch.zeros(4, 64, dtype=BF16, device="cuda", requires_grad=True)
    w = ops.quantize_mxfp4(torch.ones(8, 64, device="cuda"))
    y = ops.mx_linear(x, w)
    w.codes.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    logits, idx = torch.zeros(4, 8, device="cuda", requires_grad=True), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    out = ops.router_losses(logits, idx)
    out.counts.zero_()            # the caller's
    out.balance.backward()
    out = ops.router_losses(logits, idx)
    idx.fill_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.balance.backward()


def test_derivatives_that_there_are_not():
    x = torch.ones(4, 64, dtype=BF16, device="cuda", requires_grad=True)
    w = ops.quantize_mxfp4(torch.ones(8, 64, device="cuda"))
    d, = torch.autograd.grad(ops.mx_linear(x, w).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    logits, idx = torch.zeros(4, 8, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(logits, torch.ones_like(logits))
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.router_losses(dual, idx)
    for f, a in ((lambda t: ops.quantize_mxfp4(t).codes, torch.ones(4, 64, device="cuda")),
                 (lambda t: ops.router_losses(t, idx).balance, logits), (lambda t: ops.mx_linear(t, w), x.detach())):
        with pytest.raises(ModelError, match="traced"):
            torch.jit.trace(f, a)


def test_weights_past_2_to_the_31_bytes():
    # 160 experts of 4096 x 7168: 2.35 GB of codes; rows of the last experts alone
    E, N, K = 160, 4096, 7168
    g = gen(31)
    codes = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.randint(110, 118, (E, N, K // 32), dtype=torch.uint8, device="cuda", generator=g)
    w = ops.MxTensor(codes, scales)
    for M in (12, 900):
        x = normal(g, M, K, dtype=BF16)
        off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        off[E - 1], off[E] = M // 3, M
        ref = torch.cat([x[a:b].double() @ mx_ref.values(codes[e], scales[e]).t() for e, a, b in ((E - 2, 0, M // 3), (E - 1, M // 3, M))])
        mag = torch.cat([x[a:b].double().abs() @ mx_ref.values(codes[e], scales[e]).abs().t()
                         for e, a, b in ((E - 2, 0, M // 3), (E - 1, M // 3, M))])
        ops_ref.assert_close(ops.mx_linear(x, w, offsets=off), ref, (K + 1) * ops_ref.U32 * mag, "y")
        dy = normal(g, M, N, dtype=BF16)
        xg = x.requires_grad_()
        d, = torch.autograd.grad(ops.mx_linear(xg, w, offsets=off), xg, dy)
        ref = torch.cat([dy[a:b].double() @ mx_ref.values(codes[e], scales[e]) for e, a, b in ((E - 2, 0, M // 3), (E - 1, M // 3, M))])
        mag = torch.cat([dy[a:b].double().abs() @ mx_ref.values(codes[e], scales[e]).abs()
                         for e, a, b in ((E - 2, 0, M // 3), (E - 1, M // 3, M))])
        ops_ref.assert_close(d, ref, N * ops_ref.U32 * mag, "dx")


def test_rows_past_2_to_the_31_bytes():
    # 600000 rows of 2048: 2.46 GB of bf16 rows, 0.6 GB of codes; the first and last rows checked
    M, K, N = 600000, 2048, 64
    g = gen(32)
    x = normal(g, M, K, dtype=BF16)
    q = ops.quantize_mxfp4(x)
    for rows in (slice(0, 300), slice(M - 300, M)):
        codes, scales = mx_ref.quantize(x[rows])
        assert torch.equal(q.codes[rows], codes) and torch.equal(q.scales[rows], scales)
        assert torch.equal(ops.dequantize_mxfp4(q)[rows].double(), mx_ref.values(codes, scales))
    w = ops.quantize_mxfp4(normal(g, N, K, dtype=BF16, std=K ** -0.5))
    wv = mx_ref.values(*w)
    y, y4 = ops.mx_linear(x, w), ops.mx_linear(q, w)
    for rows in (slice(0, 300), slice(M - 300, M)):
        for got, a in ((y, x[rows].double()), (y4, mx_ref.values(q.codes[rows], q.scales[rows]))):
            ops_ref.assert_close(got[rows], a @ wv.t(), (K + 1) * ops_ref.U32 * (a.abs() @ wv.abs().t()), "y")
    # 4.3 million tokens of 512 experts: logits past 2^31 elements
    T, E = 4_300_000, 512
    logits = torch.empty(T, E, dtype=BF16, device="cuda").normal_(generator=g).requires_grad_()
    idx = torch.randint(0, E, (T, 1), device="cuda", generator=g, dtype=torch.int32)
    offsets = torch.tensor([0, T - 1000, T], dtype=torch.int32, device="cuda")
    out = ops.router_losses(logits, idx, offsets=offsets)
    last = logits.detach()[T - 1000:].double()
    ref = mx_ref.losses(last, idx[T - 1000:], "softmax", 1.0, 1.0, 1.0, None, torch.ones(1), torch.ones(1))
    mx_ref.assert_close(out.balance.detach()[1:], *ref["balance"], "balance")
    mx_ref.assert_close(out.z.detach()[1:], *ref["z"], "z")
    assert torch.equal(out.counts[1:], ref["counts"]) and int(out.counts.sum()) == T
    d, = torch.autograd.grad((out.balance, out.z), logits, (torch.ones(2, device="cuda"),) * 2)
    mx_ref.assert_close(d[T - 1000:], *ref["d"], "d_logits")
