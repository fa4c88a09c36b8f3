"""router_losses over logits at the ends of their types' ranges."""
import pytest
import torch

from oxidizr_amd import ops
from tests import mx_ref
from tests.ops_ref import U32
from tests.test_gpu_router import problem

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("end", ["min", "max"])
@pytest.mark.parametrize("tau", [0.5, 0.03])
def test_rows_beyond_fp32_once_divided_by_the_temperature(tau, end, score, dtype):
    # whole rows of a type's lowest or largest value: their scores are even, as at any other level
    logits, idx = problem(90, 24, 2, 9, dtype, pad=0.1)
    level = getattr(torch.finfo(dtype), end)
    logits[::3] = level
    logits[1::9, 4:20] = torch.finfo(dtype).min
    # the level does not matter to a softmax; sigmoid and its slope are those of +-200 to 1e-80
    ref = logits.double()
    ref[::3] = 0.0 if score == "softmax" else 200.0 if level > 0 else -200.0
    ref[1::9, 4:20] = -float("inf")
    d_balance = torch.tensor([0.3], device="cuda")
    want = mx_ref.losses(ref, idx, score, tau, 1.0, 1.0, None, d_balance, None)
    x = logits.clone().requires_grad_()
    out = ops.router_losses(x, idx, score=score, temperature=tau)
    mx_ref.assert_close(out.balance.detach().view(1), *want["balance"], "balance")
    assert torch.equal(out.counts.view(1, -1), want["counts"])
    got, = torch.autograd.grad(out.balance, x, d_balance[0])
    mx_ref.assert_close(got, *want["d"], "d_logits")
    assert float(want["d"][0][::3].abs().max()) > (1e-5 if score == "softmax" or level < 0 else -1.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("end", ["min", "max"])
def test_gradient_of_z_where_the_log_sum_is_beyond_fp32(end, dtype):
    logits, idx = problem(60, 24, 2, 4, dtype, pad=0.1)
    logits[::3] = getattr(torch.finfo(dtype), end)
    real = ((idx >= 0) & (idx < 24)).any(1)
    up = 1e-6
    ref = logits.double() / 0.5
    # the formula, not autograd's: torch's gradient of logsumexp is exp(x - lse), 1 in each of 24 where lse rounds to x
    want = 2 * up / real.sum() * torch.logsumexp(ref, 1, keepdim=True) * torch.softmax(ref, 1) / 0.5
    x = logits.clone().requires_grad_()
    out = ops.router_losses(x, idx, temperature=0.5)
    got, = torch.autograd.grad(out.z, x, torch.tensor(up, device="cuda"))
    # h has four roundings, its product with 1 / tau and m two, the sum one, p some 5 (the sum of 24 ones is exact), the last two;
    # the slope of the balance is not asked for
    rows = real.clone()
    rows[1::3] = rows[2::3] = False
    tol = 16 * U32 + torch.finfo(dtype).eps / 2
    assert bool(rows.any()) and float(want[rows].abs().max()) < 3e38
    assert bool(((got[rows].double() - want[rows]).abs() <= tol * want[rows].abs()).all())
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("E", [24, 13, 160])
def test_infinite_logits_of_sigmoid_scores(E, dtype):
    # sigmoid(inf) = 1: the balance loss and its gradient are numbers
    logits, idx = problem(200, E, 2, 6, dtype, pad=0.1)
    logits[::4, 3] = float("inf")
    logits[1::4, 5:12] = -float("inf")
    logits[2::8, :10] = float("inf")
    ref = torch.where(logits == float("inf"), 200.0, logits.double())
    d_balance = torch.tensor([0.3], device="cuda")
    want = mx_ref.losses(ref, idx, "sigmoid", 1.0, 1.0, 1.0, None, d_balance, None)
    x = logits.clone().requires_grad_()
    out = ops.router_losses(x, idx, score="sigmoid")
    mx_ref.assert_close(out.balance.detach().view(1), *want["balance"], "balance")
    got, = torch.autograd.grad(out.balance, x, d_balance[0], retain_graph=True)
    mx_ref.assert_close(got, *want["d"], "d_logits")
    again, = torch.autograd.grad((out.balance, out.z), x, (d_balance[0], torch.zeros_like(d_balance[0])))
    assert torch.equal(got, again)
    assert float(out.z.detach()) == float("inf")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("value,z", [(float("inf"), float("inf")), (-float("inf"), float("inf")), (float("nan"), float("nan"))])
def test_z_of_a_row_that_is_not_finite(value, z, score):
    # one such row of the second sequence: z and its gradient of all other rows are as the definition has them
    logits, idx = problem(90, 24, 2, 9, pad=0.1)
    idx[50] = 3
    offsets = torch.tensor([0, 40, 90], dtype=torch.int32, device="cuda")
    up = torch.tensor([0.2, 0.4], device="cuda")
    want = mx_ref.losses(logits.double(), idx, score, 1.0, 1.0, 1.0, offsets, None, up)
    logits[50] = value if value == -float("inf") else torch.where(torch.arange(24, device="cuda") == 7, value, logits[50])
    x = logits.clone().requires_grad_()
    out = ops.router_losses(x, idx, score=score, offsets=offsets)
    got_z = out.z.detach()
    mx_ref.assert_close(got_z[:1], *(t[:1] for t in want["z"]), "z")
    assert str(float(got_z[1])) == str(z)
    got, = torch.autograd.grad(out.z, x, up)
    ref, err = want["d"]
    others = torch.arange(90, device="cuda") != 50
    mx_ref.assert_close(got[others], ref[others], err[others], "d_logits")
    if value == float("inf"):
        both = logits.clone()
        both[50, 2] = float("nan")
        assert bool(ops.router_losses(both, idx, score=score, offsets=offsets).z[1].isnan())


@pytest.mark.parametrize("runs", [[1], [3, 7, 8, 9, 10, 200], [5000, 1, 60000]])
def test_runs_of_empty_sequences(runs):
    # sequences of 7 rows with so many empty ones behind each
    logits, idx = problem(7 * (len(runs) + 1), 16, 2, 5, pad=0.2)
    ends = [0]
    for i, n in enumerate(runs):
        ends += [7 * (i + 1)] * (n + 1)
    offsets = torch.tensor(ends + [logits.shape[0]], dtype=torch.int32, device="cuda")
    full = torch.tensor([0] + [7 * (i + 1) for i in range(len(runs) + 1)], dtype=torch.int32, device="cuda")
    has = offsets[1:] > offsets[:-1]
    x = logits.clone().requires_grad_()
    out, want = (ops.router_losses(x, idx, offsets=o) for o in (offsets, full))
    for a, b in zip(out, want):
        assert torch.equal(a[has], b) and not bool(a[~has].any())
    g = torch.rand(has.shape, device="cuda")
    assert torch.equal(torch.autograd.grad(out.balance, x, g)[0], torch.autograd.grad(want.balance, x, g[has])[0])


def test_a_long_run_of_empty_sequences_does_not_hold_up_a_block():
    # 2^22 - 1 sequences, of which two have rows: beside each other, or (one block walks them) at both ends
    S, T = 2 ** 22 - 1, 64
    logits, idx = problem(T, 4, 1, 3, pad=0.0)
    beside, ends = (torch.full((S + 1,), n, dtype=torch.int32, device="cuda") for n in (T, 10))
    beside[0], beside[1], ends[0], ends[-1] = 0, 10, 0, T
    x = logits.clone().requires_grad_()
    up = torch.ones(S, device="cuda")

    def ms(offsets):
        best = []
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            out = ops.router_losses(x, idx, offsets=offsets)
            d, = torch.autograd.grad(out.balance, x, up)
            b.record()
            b.synchronize()
            best.append(a.elapsed_time(b))
        return min(best), d
    (quick, a), (walked, b) = ms(beside), ms(ends)
    assert torch.equal(a, b)
    # 0.1 us a sequence and direction when each is loaded behind the other: 0.8 s, where the rest takes some 40 ms
    assert walked < 3 * quick + 20, (quick, walked)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tau", [2.0 ** -126, 1e-30, 1e30, 3e38])
def test_temperatures_at_the_ends_of_their_range(tau, score):
    # whole numbers, and each row's largest alone: at the lowest temperatures all of its score (a sigmoid's: of each above 0),
    # at the highest none of it
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randint(-9, 8, (60, 24), device="cuda", generator=g).float()
    logits[torch.arange(60), torch.randint(0, 24, (60,), device="cuda", generator=g)] = 8.0
    idx = torch.randint(0, 24, (60, 2), device="cuda", generator=g)
    out = ops.router_losses(logits, idx, score=score, temperature=tau, switch_coef=1.0, sqprob_coef=1.0)
    if tau > 1:
        q = torch.full((60, 24), 1 / 24, dtype=torch.float64, device="cuda")
    else:
        q = (logits == 8.0 if score == "softmax" else logits > 0).double() + 0.5 * (logits == 0) * (score == "sigmoid")
        q = q / q.sum(1, keepdim=True)
    P, f = q.mean(0), torch.bincount(idx.flatten(), minlength=24).double() / 120
    want = float(24 * (f * P + P * P).sum())
    # quotients, 60 additions and 24 terms in fp32
    assert abs(float(out.balance) - want) <= 120 * U32 * want
