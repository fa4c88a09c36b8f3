"""4-bit numbers and the products over them on the GPU, against plain float64 forms (tests/mx_ref.py, tests/ops_ref.py)."""
import pytest
import torch

from oxidizr_amd import ops
from oxidizr_amd.moe import ModelError
from tests import mx_ref, ops_ref
from tests.test_gpu_ops import gen, normal

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


# ---------------------------------------------------------------- quantisation

def check_quantize(x):
    q = ops.quantize_mxfp4(x)
    codes, scales = mx_ref.quantize(x)
    assert torch.equal(q.scales, scales)
    assert torch.equal(q.codes, codes)
    want = mx_ref.values(codes, scales)
    for dtype in (BF16, F32):
        got = ops.dequantize_mxfp4(q, dtype=dtype)
        assert got.dtype == dtype and got.shape == x.shape
        assert torch.equal(got.double().nan_to_num(nan=-777.0), want.nan_to_num(nan=-777.0))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(32,), (1, 32), (3, 64), (5, 96), (2, 3, 2048), (1000, 736), (64, 4096), (0, 64)])
def test_quantize(shape, dtype):
    check_quantize(normal(gen(sum(shape)), *shape, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_borders(dtype):
    # every border between two codes, its neighbours, and every exponent that a block may have
    base = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0])
    eps = torch.finfo(dtype).eps
    row = torch.cat((base, -base * (1 + eps), base * (1 - eps / 2), -base)).to(dtype)     # one block is 32 of these
    rows = torch.stack([row * 2.0 ** e for e in range(-130, 125)]).to(dtype)
    rows = torch.cat((rows, rows.flip(1), rows * (1 + 2 * eps)))
    check_quantize(rows.cuda())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_extremes(dtype):
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = torch.zeros(9, 64, dtype=dtype)
    x[0, 3] = float("inf")
    x[1, 40] = float("nan")
    x[2, :] = big
    x[3, 1] = -big
    x[4, 1] = tiny
    x[5, 2] = tiny / 8          # below the smallest normal number
    x[6, :] = -0.0
    x[7, 33], x[7, 1] = -float("inf"), 1.0
    x[8, 0], x[8, 1] = torch.finfo(dtype).smallest_normal * 2, tiny / 2
    check_quantize(x.cuda())


def test_every_scale_and_code_back():
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 2).view(256, 32, 16)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 32)
    q = ops.MxTensor(codes.reshape(256, 512).cuda(), scales.cuda())
    want = mx_ref.values(*q)
    for dtype in (F32, BF16):
        got = ops.dequantize_mxfp4(q, dtype=dtype)
        w = want.to(dtype).double()   # infinite above the dtype's largest number
        assert torch.equal(got.double().nan_to_num(nan=-777.0, posinf=1e300, neginf=-1e300),
                           w.nan_to_num(nan=-777.0, posinf=1e300, neginf=-1e300))


def test_quantize_of_views():
    x = normal(gen(5), 40, 128, dtype=BF16)
    for part in (x[:, 32:96], x[3:], x.t().contiguous().t()[:, :64], x[::2], x.view(-1)[8:8 + 64]):
        check_quantize(part)
    q = ops.quantize_mxfp4(x)
    part = ops.MxTensor(q.codes[:, 16:48], q.scales[:, 1:3])
    assert torch.equal(ops.dequantize_mxfp4(part), ops.dequantize_mxfp4(q)[:, 32:96])


def test_quantize_has_no_gradient():
    x = normal(gen(6), 4, 64).requires_grad_()
    assert not ops.dequantize_mxfp4(ops.quantize_mxfp4(x)).requires_grad


# ---------------------------------------------------------------- products

ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]
# M, K, N, group sizes (None: one weight), rows of no group, activation, bias, residual
FEW = [(1, 32, 8, None, 0, "none", False, False), (1, 2048, 1408, None, 0, "silu", True, False),
       (2, 2048, 1408, [0, 1, 0, 1], 0, "silu", True, False), (5, 736, 24, [2, 0, 3], 0, "gelu", True, True),
       (17, 96, 40, [17, 0], 0, "gelu_tanh", False, True), (33, 1376, 1368, None, 0, "relu", True, True),
       (40, 4096, 72, [1, 3, 0, 9, 16, 11], 0, "gelu", True, False), (21, 512, 520, [4, 4, 4], 9, "silu", True, True),
       (64, 544, 136, [8] * 8, 0, "none", True, False), (3, 4128, 8, [1, 1, 0], 1, "none", False, False),
       (66, 64, 16, [66], 0, "none", True, False), (130, 160, 2056, [65, 64], 1, "silu", False, False)]
MANY = [(200, 736, 136, None, 0, "silu", True, True), (513, 320, 264, None, 0, "none", False, False),
        (700, 64, 1032, [64, 65, 0, 571], 0, "gelu", True, False), (1300, 1376, 392, [319, 320, 321, 0, 257], 83, "relu", True, True),
        (2000, 288, 520, [1023, 0, 1, 127, 129, 600], 120, "gelu_tanh", True, False), (4100, 544, 776, None, 0, "gelu", True, True),
        (3000, 2080, 256, [577, 576, 640, 705, 192, 193], 117, "silu", True, True), (1024, 1024, 1024, [1024], 0, "none", True, True),
        (6000, 96, 136, [3000, 2990], 10, "none", False, True), (9000, 256, 1408, None, 0, "silu", True, False),
        (5000, 448, 2816, [1250] * 4, 0, "gelu", False, False), (777, 32, 8, [7, 700], 70, "none", True, False)]

# 256-row tiles with some left behind an XCD's last 32, forward (wide N) or back (wide K): 5, 12 and 24 of them, and of groups
CUT = [(9316, 64, 2048, None, 0, "silu", True, True), (11259, 2048, 96, None, 0, "none", False, False), (14300, 64, 2048, None, 0, "none", True, False),
       (12050, 96, 1368, [0, 1, 255, 257, 3000, 511, 513, 1100, 2000, 1700, 963, 1700], 50, "gelu", True, True),
       (9000, 1376, 1368, [600, 700, 800, 900, 1000, 1000, 1100, 900, 1000, 1000], 0, "silu", True, False)]


def problem(case, seed, std=1.0):
    M, K, N, sizes, tail, act, has_b, has_r = case
    g = gen(seed)
    x = normal(g, M, K, dtype=BF16, std=std)
    E = len(sizes) if sizes else 1
    w = ops.MxTensor(*mx_ref.quantize(normal(g, E, N, K, std=K ** -0.5)))
    offsets = None
    if sizes:
        offsets = torch.tensor([0] + sizes, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        assert int(offsets[-1]) + tail == M
    else:
        w = ops.MxTensor(w.codes[0], w.scales[0])
    b = normal(g, *((E, N) if sizes else (N,)), dtype=BF16, std=0.5) if has_b else None
    r = normal(g, M, N, dtype=BF16) if has_r else None
    return x, w, b, r, offsets, act


def reference(x, w, b, r, offsets, act, dy, dtype):
    def f64(t):
        return None if t is None else t.detach().double()
    return ops_ref.linear(x, mx_ref.values(*w), f64(b), None if offsets is None else offsets.cpu(), act, f64(r), f64(dy), dtype)


@pytest.mark.parametrize("case", FEW + MANY + CUT, ids=str)
def test_bf16_rows(case):
    x, w, b, r, offsets, act = problem(case, len(str(case)))
    if offsets is not None and int(offsets[-1]) < x.shape[0]:
        x[int(offsets[-1]):] = float("nan")   # rows of no expert are not read
    clean = torch.nan_to_num(x.double())
    want, err = reference(clean, w, b, r, offsets, act, None, BF16)["y"]
    got = ops.mx_linear(x, w, b, offsets=offsets, activation=act, residual=r)
    assert got.dtype == BF16
    ops_ref.assert_close(got, want, err, "y")
    assert torch.equal(got, ops.mx_linear(x, w, b, offsets=offsets, activation=act, residual=r))


@pytest.mark.parametrize("case", FEW + MANY + CUT, ids=str)
def test_gradients(case):
    x, w, b, r, offsets, act = problem(case, len(str(case)) + 1)
    dy = normal(gen(9), x.shape[0], case[2], dtype=BF16)
    want = reference(x.double(), w, b, r, offsets, act, dy, BF16)
    if offsets is not None and int(offsets[-1]) < x.shape[0]:
        x[int(offsets[-1]):] = float("nan")
        if r is None:
            dy = dy.clone()
            dy[int(offsets[-1]):] = float("nan")
    leaves = [t.requires_grad_() for t in (x, b, r) if t is not None]
    y = ops.mx_linear(x, w, b, offsets=offsets, activation=act, residual=r)
    ops_ref.assert_close(y.detach(), *want["y"], "y")
    got = dict(zip([n for n, t in (("dx", x), ("db", b), ("dr", r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    for name, t in got.items():
        ops_ref.assert_close(t, *want[name], name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", FEW + MANY + CUT, ids=str)
def test_both_sides_in_four_bits(case, dtype):
    x, w, b, r, offsets, act = problem(case, len(str(case)) + 2)
    if offsets is not None and int(offsets[-1]) < x.shape[0]:
        x[int(offsets[-1]):] = float("nan")
    q = ops.quantize_mxfp4(x)
    b, r = (None if t is None else t.to(dtype) for t in (b, r))
    want, err = reference(torch.nan_to_num(mx_ref.values(*q)), w, b, r, offsets, act, None, dtype)["y"]
    got = ops.mx_linear(q, w, b, offsets=offsets, activation=act, residual=r, dtype=dtype)
    assert got.dtype == dtype
    ops_ref.assert_close(got, want, err, "y")
    assert torch.equal(got, ops.mx_linear(q, w, b, offsets=offsets, activation=act, residual=r, dtype=dtype))


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("M", [3, 700])
def test_wide_scales(M, four):
    # blocks of very different exponents beside each other, rows of zeros, and weights of zeros
    g = gen(12)
    K, N = 416, 136
    x = normal(g, M, K, dtype=BF16) * torch.exp2(torch.randint(-30, 30, (M, K // 32), device="cuda", generator=g)).repeat_interleave(32, 1)
    x = x.to(BF16)
    x[M // 2] = 0
    w = normal(g, N, K) * torch.exp2(torch.randint(-30, 30, (N, K // 32), device="cuda", generator=g)).repeat_interleave(32, 1)
    w[5] = 0
    q = ops.MxTensor(*mx_ref.quantize(w))
    rows = ops.quantize_mxfp4(x) if four else x
    want, err = reference(mx_ref.values(*rows) if four else x.double(), q, None, None, None, "none", None, BF16)["y"]
    ops_ref.assert_close(ops.mx_linear(rows, q), want, err, "y")


@pytest.mark.parametrize("M", [3, 700])
def test_nan_blocks_reach_their_rows_alone(M):
    g = gen(13)
    K, N = 160, 264
    x, w = normal(g, M, K, dtype=BF16), normal(g, N, K)
    x[1, 159], w[7, 3] = float("inf"), float("nan")
    qx, qw = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    for rows in (x, qx):
        y = ops.mx_linear(rows, qw)
        bad = torch.zeros(M, N, dtype=torch.bool, device="cuda")
        bad[:, 7] = True
        if rows is qx:
            bad[1] = True
        else:
            assert not bool(torch.isfinite(y[1]).any())
            y, bad = y[[0, 2]], bad[[0, 2]]
        assert torch.equal(~torch.isfinite(y), bad)


def test_refusals_on_the_device():
    x = torch.zeros(4, 64, dtype=BF16, device="cuda")
    q = ops.quantize_mxfp4(x)
    w = ops.MxTensor(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8))
    with pytest.raises(ModelError, match="different devices"):
        ops.mx_linear(x, w)
    w = ops.MxTensor(*(t.cuda() for t in w))
    b = torch.zeros(8, dtype=BF16, device="cuda", requires_grad=True)
    with pytest.raises(ModelError, match="no gradient of a bias"):
        ops.mx_linear(q, w, b)
    with torch.no_grad():
        ops.mx_linear(q, w, b)
    r = torch.zeros(4, 8, dtype=BF16, device="cuda", requires_grad=True)
    y = ops.mx_linear(q, w, b.detach(), residual=r)
    d, = torch.autograd.grad(y, r, torch.ones_like(y))
    assert bool((d == 1).all())


@pytest.mark.parametrize("four", [False, True])
def test_no_rows(four):
    x = torch.zeros(0, 64, dtype=BF16, device="cuda")
    w = ops.MxTensor(torch.zeros(3, 8, 32, dtype=torch.uint8).cuda(), torch.zeros(3, 8, 2, dtype=torch.uint8).cuda())
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    b = torch.ones(3, 8, dtype=BF16, device="cuda")
    rows = ops.quantize_mxfp4(x) if four else x.requires_grad_()
    if not four:
        b.requires_grad_()
    y = ops.mx_linear(rows, w, b, offsets=off, activation="silu")
    assert y.shape == (0, 8)
    if not four:
        dx, db = torch.autograd.grad(y, (x, b), torch.zeros_like(y))
        assert dx.shape == x.shape and bool((db == 0).all())
