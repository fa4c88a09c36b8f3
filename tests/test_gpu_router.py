"""router_losses on the GPU against the float64 form (tests/mx_ref.py)."""
import pytest
import torch

from oxidizr_amd import ops
from tests import mx_ref
from tests.test_gpu_ops import gen

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def problem(T, E, k, seed, dtype=F32, pad=0.1, std=1.0, index=torch.int32):
    g = gen(seed)
    logits = (torch.randn(T, E, device="cuda", generator=g) * std).to(dtype)
    idx = torch.randint(0, E, (T, k), device="cuda", generator=g).to(index)
    idx[torch.rand(T, k, device="cuda", generator=g) < 0.1] = E + 3       # dropped
    idx[torch.rand(T, device="cuda", generator=g) < pad] = -1
    return logits, idx


def check(logits, idx, score="softmax", tau=1.0, c_sw=1.0, c_sq=1.0, offsets=None, up=(0.01, 0.001), clean=None):
    """clean: the logits where padding holds no numbers."""
    S = 1 if offsets is None else offsets.numel() - 1
    g = gen(77)
    d_balance, d_z = (None if c is None else c * (0.5 + torch.rand(S, device="cuda", generator=g)) for c in up)
    ref = mx_ref.losses((logits if clean is None else clean).double(), idx, score, tau, c_sw, c_sq, offsets, d_balance, d_z)
    kw = dict(score=score, temperature=tau, switch_coef=c_sw, sqprob_coef=c_sq, offsets=offsets)
    plain = ops.router_losses(logits, idx, **kw)
    x = logits.clone().requires_grad_()
    out = ops.router_losses(x, idx, **kw)
    lead = () if offsets is None else (S,)
    for name in ("balance", "z", "counts"):
        got = getattr(out, name).detach()
        assert torch.equal(got, getattr(plain, name)), name
        assert got.shape == lead + ((logits.shape[1],) if name == "counts" else ())
    assert torch.equal(out.counts.view(S, -1), ref["counts"]) and out.counts.dtype == torch.int32
    for name in ("balance", "z"):
        mx_ref.assert_close(getattr(out, name).detach().view(S), *ref[name], name)
    pairs = [(t, d.view(lead)) for t, d in ((out.balance, d_balance), (out.z, d_z)) if d is not None]
    d, = torch.autograd.grad([t for t, _ in pairs], x, [v for _, v in pairs])
    assert d.dtype == logits.dtype
    mx_ref.assert_close(d, *ref["d"], "d_logits")
    return out, d


SIZES = [(1, 1, 1), (1, 16, 2), (5, 3, 1), (7, 8, 8), (33, 12, 3), (64, 33, 16), (100, 64, 6), (255, 100, 5), (257, 128, 8),
         (1000, 160, 6), (513, 256, 8), (300, 257, 4), (77, 512, 2), (129, 700, 3), (90, 1000, 16), (65, 1023, 7), (40, 1024, 8),
         (8192, 16, 2), (9001, 256, 8), (20001, 64, 6)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,E,k", SIZES)
def test_sizes(T, E, k, dtype, score):
    logits, idx = problem(T, E, k, T + E, dtype, index=torch.int64 if T % 2 else torch.int32)
    check(logits, idx, score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tau,c_sw,c_sq", [(0.5, 1.0, 0.0), (3.0, 0.0, 1.0), (1.0, 2.5, 0.25), (1.0, 0.0, 0.0), (0.7, -1.0, 2.0)])
def test_coefficients(score, tau, c_sw, c_sq):
    logits, idx = problem(300, 40, 4, 3)
    check(logits, idx, score, tau, c_sw, c_sq)
    check(logits, idx, score, tau, c_sw, c_sq, up=(None, 0.1))
    check(logits, idx, score, tau, c_sw, c_sq, up=(0.1, None))


def cut(T, seed, S, lead=0, tail=0):
    g = torch.Generator().manual_seed(seed)
    at = torch.randint(lead, T - tail + 1, (S - 1,), generator=g).sort().values
    return torch.cat((torch.tensor([lead]), at, torch.tensor([T - tail]))).to(torch.int32).cuda()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,S,lead,tail", [(40, 16, 2, 1, 0, 0), (40, 16, 2, 5, 0, 0), (300, 33, 3, 9, 11, 17), (5000, 64, 6, 7, 0, 500),
                                               (9001, 256, 8, 40, 100, 0), (6000, 12, 2, 3000, 0, 0), (50, 1000, 4, 200, 3, 3)])
def test_sequences(T, E, k, S, lead, tail, score):
    logits, idx = problem(T, E, k, S)
    offsets = cut(T, S, S, lead, tail)
    idx[int(offsets[S // 2]):int(offsets[S // 2 + 1])] = -1      # a sequence of padding alone
    clean = logits.clone()
    logits[:lead] = float("nan")                                 # rows of no sequence
    if tail:
        logits[T - tail:] = float("inf")
    out, d = check(logits, idx, score, offsets=offsets, clean=clean)
    assert bool((d[:lead] == 0).all()) and (tail == 0 or bool((d[T - tail:] == 0).all()))


def test_edges_of_blocks_and_sequences():
    # sequences that end where a block's rows do, and one row before and behind
    T = 5000
    logits, idx = problem(T, 64, 4, 1)
    for at in (16, 63, 64, 65, 128, 1024, 4096, 4999):
        check(logits, idx, offsets=torch.tensor([0, at, at, min(at + 64, T), T], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_padding_may_hold_anything(score, dtype):
    logits, idx = problem(500, 64, 4, 5, dtype, pad=0.5)
    pad = ((idx < 0) | (idx >= 64)).all(1)
    clean = logits.clone()
    for i, v in enumerate((float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min)):
        rows = pad.nonzero()[i::4, 0]
        logits[rows] = v
        logits[rows, i] = 0.0
    _, d = check(logits, idx, score, clean=clean)
    assert bool((d[pad] == 0).all())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("fill", [-float("inf"), torch.finfo(F32).min, -1e4, -200.0])
def test_masked_experts(score, fill):
    # experts switched off by very negative logits, and rows of very negative logits only
    logits, idx = problem(200, 48, 3, 6)
    logits[:, 5:20] = fill
    logits[7] = logits[7] * 0.01 - 150.0
    if fill != torch.finfo(F32).min:
        check(logits, idx, score)
    else:
        out = ops.router_losses(logits, idx, score=score)
        logits[:, 5:20] = -float("inf")
        same = ops.router_losses(logits, idx, score=score)
        assert torch.equal(out.balance, same.balance) and torch.equal(out.z, same.z)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("at", [32.0, 2.0 ** 15, -2.0 ** 15])
def test_a_softmax_does_not_depend_on_a_rows_level(at, dtype):
    # logits of few bits: x + at is exact, so each x less the largest is the same number, and so are all results but lse's
    idx = problem(300, 48, 3, 8)[1]
    step = 2.0 ** -4 if dtype == F32 else 2.0 ** (-2 if at == 32.0 else 8)
    x = torch.randint(-4, 4, (300, 48), device="cuda", generator=gen(8)).double() * step
    out = []
    for level in (0.0, at):
        logits = (x + level).to(dtype)
        assert torch.equal(logits.double(), x + level)
        logits.requires_grad_()
        balance = ops.router_losses(logits, idx).balance
        out.append((balance.detach(), torch.autograd.grad(balance, logits)[0]))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


def test_rows_masked_whole_by_the_lowest_value():
    logits, idx = problem(90, 24, 2, 9, pad=0.0)
    logits[::3] = torch.finfo(F32).min
    ref = logits.double().requires_grad_()
    real = ((idx >= 0) & (idx < 24)).any(1)
    P = torch.softmax(ref, 1)[real].mean(0)
    f = torch.bincount(idx[(idx >= 0) & (idx < 24)].long(), minlength=24) / (2 * real.sum().double())
    want, = torch.autograd.grad(24 * (f * P + P * P).sum(), ref)
    x = logits.requires_grad_()
    got, = torch.autograd.grad(ops.router_losses(x, idx).balance, x)
    # g_e and its mean over p: some 200 roundings of what is at most max |g|
    n = float(real.sum())
    assert bool(((got.double() - want).abs() <= 200 * 2.0 ** -24 * float(24 * (f + 2 * P).max()) / n).all())
    assert float(want[::3].abs().max()) > 1e-4


def test_nothing_real():
    for T in (0, 1, 70):
        logits = torch.full((T, 24), float("nan"), device="cuda").requires_grad_()
        out = ops.router_losses(logits, torch.full((T, 2), -1, dtype=torch.int64, device="cuda"))
        assert float(out.balance.detach()) == 0 and float(out.z.detach()) == 0 and int(out.counts.sum()) == 0
        d, = torch.autograd.grad((out.balance, out.z), logits, (torch.ones((), device="cuda"),) * 2)
        assert bool((d == 0).all())
    out = ops.router_losses(torch.zeros(5, 8, device="cuda"), torch.zeros(5, 1, dtype=torch.int32, device="cuda"),
                            offsets=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert out.balance.shape == (0,) and out.counts.shape == (0, 8)


def test_the_same_index_twice_counts_twice():
    logits, _ = problem(30, 8, 2, 7)
    idx = torch.full((30, 4), 3, dtype=torch.int32, device="cuda")
    out, _ = check(logits, idx)
    assert int(out.counts[3]) == 120


def test_views_and_expanded_upstreams():
    logits, idx = problem(300, 64, 6, 8)
    wide = torch.cat((logits, logits), 1)
    check(wide[:, 64:], idx)
    check(wide[:, 1:64], torch.where(idx < 63, idx, -1))
    check(logits.t().contiguous().t(), idx.t().contiguous().t())
    offsets = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    x = logits.clone().requires_grad_()
    out = ops.router_losses(x, idx, offsets=offsets)
    d, = torch.autograd.grad(out.balance.sum() + out.z.sum(), x)
    want = torch.autograd.grad((out2 := ops.router_losses(x, idx, offsets=offsets)).balance, x, torch.ones(2, device="cuda"),
                               retain_graph=True)[0] + torch.autograd.grad(out2.z, x, torch.ones(2, device="cuda"))[0]
    assert torch.allclose(d, want, rtol=1e-5, atol=1e-8)


def test_gradient_against_differences():
    logits, idx = problem(24, 12, 3, 9)
    offsets = torch.tensor([0, 9, 24], dtype=torch.int32, device="cuda")
    for score in ops.SCORES:
        def f(x):
            r = mx_ref.losses(x, idx, score, 0.8, 1.0, 0.5, offsets, None, None)
            return float(r["balance"][0].sum() * 0.3 + r["z"][0].sum() * 0.2)
        x = logits.clone().requires_grad_()
        out = ops.router_losses(x, idx, score=score, temperature=0.8, sqprob_coef=0.5, offsets=offsets)
        d, = torch.autograd.grad(0.3 * out.balance.sum() + 0.2 * out.z.sum(), x)
        for t, e in ((0, 0), (8, 5), (9, 11), (23, 3)):
            step = torch.zeros_like(logits, dtype=torch.float64)
            step[t, e] = 1e-5
            diff = (f(logits.double() + step) - f(logits.double() - step)) / 2e-5
            # differences of a smooth function in 64 bits: 1e-10 of truncation, 1e-10 of rounding; fp32 gradients
            assert abs(float(d[t, e]) - diff) < 1e-8 + 1e-4 * abs(diff)
