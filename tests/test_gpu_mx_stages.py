"""A layer over 4-bit experts with both sides in 4 bits, stage by stage: each operator's result against float64 of what the one
before it gave, so that a wrong row, expert, bias or scale anywhere in the chain is seen; and weights at the end of their range."""
import pytest
import torch

from oxidizr_amd import ops
from tests import mx_ref, ops_ref
from tests.ops_ref import U32
from tests.test_gpu_mx_chain import inputs, layer
from tests.test_gpu_ops import check_order, gen

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def stage(name, got, x, w, b, order, act="none", residual=None):
    def f64(t):
        return None if t is None else t.double()
    want, err = ops_ref.linear(f64(x), f64(w), f64(b), order.offsets.cpu(), act, f64(residual), None, BF16)["y"]
    ops_ref.assert_close(got, want, err, name)


# few rows, tiles, and tiles with experts of a few rows
@pytest.mark.parametrize("T,H,I,E,k,pad", [(16, 512, 256, 12, 3, 0.0), (1, 512, 256, 12, 3, 0.0), (20, 1056, 544, 40, 2, 0.3),
                                           (600, 288, 160, 9, 3, 0.1), (1500, 544, 416, 5, 2, 0.05)])
def test_both_sides_in_four_bits(T, H, I, E, k, pad):
    q1, q2, p = inputs(T, T, H, I, E)
    pad = torch.rand(T, device="cuda", generator=gen(T)) < pad
    w1, w2 = mx_ref.values(*q1), mx_ref.values(*q2)
    with torch.no_grad():
        y, losses = layer(q1, q2, p, k, pad, four=True)
        # the layer's calls again, with what is between them
        top, idx = torch.topk(p["logits"], k, dim=1)
        idx = torch.where(pad[:, None], -1, idx)
        order = ops.sort_tokens(idx, E)
        rows = ops.permute_tokens(p["x"], order)
        first = ops.quantize_mxfp4(rows)
        a1 = ops.mx_linear(first, q1, p["b1"], offsets=order.offsets)
        low = ops.expert_linear(rows, p["down"], offsets=order.offsets)
        a = ops.expert_linear(low, p["up"], offsets=order.offsets, residual=a1)
        second = ops.quantize_mxfp4(a)
        b = ops.mx_linear(second, q2, p["b2"], offsets=order.offsets, activation="silu")
        weights = torch.softmax(top, 1)
    check_order(order, idx, E)
    n = int(order.offsets[-1])
    assert torch.equal(rows[:n], p["x"][order.perm[:n].long() // k])
    for got, x in ((first, rows), (second, a)):
        codes, scales = mx_ref.quantize(x[:n])
        assert torch.equal(got.codes[:n], codes) and torch.equal(got.scales[:n], scales)
    stage("first product", a1, mx_ref.values(*first), w1, p["b1"], order)
    stage("adapter, down", low, rows, p["down"], None, order)
    stage("adapter, up", a, low, p["up"], None, order, residual=a1)
    stage("second product", b, mx_ref.values(*second), w2, p["b2"], order, "silu")
    taken = torch.where(pad[:, None, None], 0.0, b.double()[order.inv_perm.long()] * weights.double()[..., None])
    # k products and sums in fp32
    ops_ref.assert_close(y, taken.sum(1), 2 * k * U32 * taken.abs().sum(1), "combined")
    want = mx_ref.losses(p["logits"].double(), idx, "softmax", 1.0, 1.0, 1.0, None, None, None)
    assert torch.equal(losses.counts[None], want["counts"]) and torch.equal(losses.counts, order.counts)
    for name in ("balance", "z"):
        mx_ref.assert_close(getattr(losses, name).view(1), *want[name], name)


@pytest.mark.parametrize("M", [1, 300])
@pytest.mark.parametrize("N", [8, 264])
def test_weights_of_the_largest_scale(M, N):
    # 2 under the scale 254 is 2^128: infinite in bf16, and so over bf16 rows; the products of 4-bit numbers hold it
    codes = torch.zeros(N, 16, dtype=torch.uint8, device="cuda")
    codes[:, 0] = 3  # element 0: 1.5, 1.5 x 2^127 is a number in both
    codes[::2, 0] = 4
    w = ops.MxTensor(codes, torch.full((N, 1), 254, dtype=torch.uint8, device="cuda"))
    x = torch.zeros(M, 32, dtype=BF16, device="cuda")
    x[:, 0] = 2.0 ** -20
    y = ops.mx_linear(x, w)
    assert bool((y[:, ::2] == float("inf")).all()) and bool((y[:, 1::2] == 1.5 * 2.0 ** 107).all())
    y = ops.mx_linear(ops.quantize_mxfp4(x), w, dtype=F32)
    assert bool((y[:, ::2] == 2.0 ** 108).all()) and bool((y[:, 1::2] == 1.5 * 2.0 ** 107).all())
