"""oxidizr_amd.ops on the GPU against plain float64 forms (tests/ops_ref.py), at the sizes, masks and
layouts where they can go wrong, with bounds from arithmetic."""
import threading

import pytest
import torch
import torch.utils.checkpoint

from oxidizr_amd import _lib, ops
from oxidizr_amd.moe import MoeBlock, MoeConfig, ModelError
from tests import ops_ref as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(mean, std, generator=g)


def routing(g, T, k, E, pad=0.0, skew=0.0):
    logits = torch.randn(T, E, device="cuda", generator=g)
    logits += skew * torch.randn(E, device="cuda", generator=g)
    idx = torch.topk(logits, min(k, E), dim=1).indices.to(torch.int32)
    if pad:
        idx[torch.rand(T, device="cuda", generator=g) < pad] = -1
    return idx


def check_order(got, idx, E):
    for name, a, b in zip(got._fields, got, ref.order(idx.cpu(), E)):
        assert torch.equal(a.cpu(), b), name


# ---------------------------------------------------------------- sorting

@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 16, 16), (7, 3, 5), (64, 8, 128), (255, 2, 1024),
                                   (257, 8, 64), (1023, 2, 7), (1025, 2, 300), (5000, 6, 64),
                                   (3001, 16, 1023), (40000, 2, 16)])
def test_sort_matches_brute_force(T, k, E):
    g = gen(T + E)
    idx = torch.randint(-1, E + 1, (T, k), device="cuda", generator=g, dtype=torch.int32)
    check_order(ops.sort_tokens(idx, E), idx, E)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort_index_types_and_what_has_no_expert(dtype):
    far = 2 ** 31 - 1 if dtype == torch.int32 else 2 ** 32 + 3  # 3 in its low half
    idx = torch.tensor([[3, 3], [-1, 0], [4, far], [-far, 1], [3, 0]], dtype=dtype, device="cuda")
    check_order(ops.sort_tokens(idx, 4), idx, 4)


def test_sort_edges():
    for idx, E in [(torch.full((33, 4), -1), 8), (torch.full((3000, 2), 5), 8), (torch.zeros(0, 2), 3),
                   (torch.arange(4096).view(2048, 2) % 1024, 1024)]:
        idx = idx.to(torch.int32).cuda()
        check_order(ops.sort_tokens(idx, E), idx, E)


def test_sort_of_a_strided_index():
    idx = routing(gen(3), 300, 5, 16)
    part = idx[1:, 1:4]
    check_order(ops.sort_tokens(part, 16), part, 16)


def test_sort_beyond_one_chunk_per_block():
    # more entries than the blocks take in one tile each: longer chunks
    T, k, E = 200000, 6, 33
    idx = torch.randint(-1, E, (T, k), device="cuda", generator=gen(8), dtype=torch.int32)
    got = ops.sort_tokens(idx, E)
    key = torch.where(idx.flatten() < 0, E, idx.flatten())
    perm = torch.argsort(key, stable=True)
    assert torch.equal(got.perm.long(), perm)
    assert torch.equal(got.inv_perm.flatten().long()[perm], torch.arange(T * k, device="cuda"))
    assert torch.equal(got.counts.long(), torch.bincount(key, minlength=E + 1)[:E])
    assert int(got.offsets[-1]) == int((key < E).sum())


# ---------------------------------------------------------------- rows to experts and back

ROWS = [(1, 8, 1, 1, 0.0), (1, 2048, 16, 16, 0.0), (5, 384, 7, 2, 0.0), (33, 520, 12, 3, 0.3),
        (64, 4096, 128, 8, 0.0), (130, 1032, 9, 5, 0.1), (259, 776, 64, 6, 0.5), (40, 7168, 256, 8, 0.2),
        (17, 64, 8, 16, 0.0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,E,k,pad", ROWS)
def test_permute_and_its_gradient(T, H, E, k, pad, dtype):
    g = gen(T * H)
    idx = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    idx[torch.rand(T, k, device="cuda", generator=g) < pad] = -1
    order = ops.sort_tokens(idx, E)
    x = normal(g, T, H, dtype=dtype).requires_grad_()
    out = ops.permute_tokens(x, order)
    kept = int(order.offsets[-1])
    want = x.detach()[(order.perm // k).long()]
    want[kept:] = 0
    assert torch.equal(out.detach(), want)
    d = normal(g, T * k, H, dtype=dtype)
    d[kept:] = float("nan")  # rows without an expert are not read
    dx, = torch.autograd.grad(out, x, d)
    rows = torch.where((order.inv_perm < kept).flatten()[:, None],
                       d.double()[order.inv_perm.flatten().long()], 0.0).view(T, k, H)
    ref.assert_close(dx, rows.sum(1), k * ref.U32 * rows.abs().sum(1), "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("T,H,E,k,pad", ROWS)
def test_unpermute_and_its_gradients(T, H, E, k, pad, weighted, dtype):
    g = gen(T * H + 1)
    idx = torch.randint(0, E, (T, k), device="cuda", generator=g, dtype=torch.int32)
    idx[torch.rand(T, k, device="cuda", generator=g) < pad] = -1
    order = ops.sort_tokens(idx, E)
    kept = int(order.offsets[-1])
    y = normal(g, T * k, H, dtype=dtype)
    y[kept:] = float("nan")
    w = torch.rand(T, k, device="cuda", generator=g)
    y.requires_grad_()
    w.requires_grad_()
    out = ops.unpermute_tokens(y, order, w if weighted else None)
    at = order.inv_perm.long()
    real = (at < kept)[..., None]
    rows = torch.where(real, y.detach().double()[at.flatten()].view(T, k, H), 0.0)
    w64 = w.detach().double() if weighted else torch.ones(T, k, device="cuda", dtype=torch.float64)
    terms = w64[..., None] * rows
    ref.assert_close(out.detach(), terms.sum(1), (k + 1) * ref.U32 * terms.abs().sum(1), "out")
    dout = normal(g, T, H, dtype=dtype)
    got = torch.autograd.grad(out, [y, w] if weighted else [y], dout)
    d64 = dout.double()[:, None, :]
    dy = torch.where(real, w64[..., None] * d64, 0.0).view(T * k, H)[order.perm.long()]
    ref.assert_close(got[0], dy, ref.U32 * dy.abs(), "dy")
    assert bool((got[0][kept:] == 0).all())
    if weighted:
        prod = d64 * rows
        ref.assert_close(got[1], prod.sum(2), (H + 8) * ref.U32 * prod.abs().sum(2), "dw")


def test_an_order_that_no_sort_made_stays_inside_the_buffers():
    # positions and a count of kept rows beyond T k
    g = gen(2)
    good = ops.sort_tokens(routing(g, 40, 3, 8), 8)
    inv = good.inv_perm.clone()
    inv[3, 1], inv[4, 2] = 10 ** 9, -5
    offsets = good.offsets.clone()
    offsets[-1] = 2 ** 31 - 1
    bad = ops.TokenOrder(good.counts, offsets, good.perm, inv)
    x, y = normal(g, 40, 64).requires_grad_(), normal(g, 120, 64).requires_grad_()
    w = torch.rand(40, 3, device="cuda", generator=g).requires_grad_()
    out = ops.unpermute_tokens(y, bad, w)
    rows = torch.where(((inv >= 0) & (inv < 120))[..., None], y.detach()[inv.long().clamp(0, 119)], 0.0)
    assert torch.allclose(out, (w[..., None] * rows).sum(1), atol=1e-5)
    torch.autograd.grad(out, [y, w], torch.ones_like(out))
    torch.autograd.grad(ops.permute_tokens(x, bad), x, torch.ones(120, 64, device="cuda"))


def test_an_order_written_to_before_the_backward_is_refused():
    g = gen(8)
    for weights in (None, torch.rand(20, 2, device="cuda", generator=g)):
        order = ops.sort_tokens(routing(g, 20, 2, 4), 4)
        x = normal(g, 20, 64).requires_grad_()
        out = ops.unpermute_tokens(ops.permute_tokens(x, order), order, weights)
        order.inv_perm.zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_gradient_of_the_rows_alone():
    # weights that need no gradient: the rows are not kept
    g = gen(5)
    order = ops.sort_tokens(routing(g, 50, 4, 8), 8)
    y = normal(g, 200, 64).requires_grad_()
    w = torch.rand(50, 4, device="cuda", generator=g)
    out = ops.unpermute_tokens(y, order, w)
    dy, = torch.autograd.grad(out, y, torch.ones_like(out))
    assert torch.equal(dy, w.flatten()[order.perm.long()][:, None].expand(200, 64))


# ---------------------------------------------------------------- expert products

def linear_case(g, sizes, K, N, act, dtype, bias, res, tail=0, grouped=True):
    """Runs expert_linear forward and backward over groups of the given sizes against the reference."""
    E = len(sizes)
    offsets = torch.tensor([0] + list(torch.tensor(sizes).cumsum(0)), dtype=torch.int32, device="cuda")
    M = sum(sizes) + tail
    t = {"x": normal(g, M, K, dtype=dtype),
         "w": normal(g, *((E, N, K) if grouped else (N, K)), dtype=dtype, std=K ** -0.5)}
    if bias:
        t["b"] = normal(g, *((E, N) if grouped else (N,)), dtype=dtype, std=0.3)
    if res:
        t["r"] = normal(g, M, N, dtype=dtype)
    dy = normal(g, M, N, dtype=dtype)
    for v in t.values():
        v.requires_grad_()
    y = ops.expert_linear(t["x"], t["w"], t.get("b"), offsets=offsets if grouped else None, activation=act,
                          residual=t.get("r"))
    got = dict(zip(t, torch.autograd.grad(y, list(t.values()), dy)))
    d = {n: v.detach().double() for n, v in t.items()}
    want = ref.linear(d["x"], d["w"], d.get("b"), offsets if grouped else None, act, d.get("r"), dy.double(),
                      dtype)
    ref.assert_close(y.detach(), *want["y"], "y")
    for n, v in got.items():
        ref.assert_close(v, *want["d" + n], "d" + n)
    with torch.no_grad():  # the forward that keeps nothing gives the same bits
        again = ops.expert_linear(t["x"], t["w"], t.get("b"), offsets=offsets if grouped else None,
                                  activation=act, residual=t.get("r"))
    assert torch.equal(again, y)


LINEAR = [  # group sizes, K, N, rows behind the last group
    ([1], 8, 8, 0),
    ([0, 3, 0, 1], 64, 40, 0),
    ([5, 0, 17, 64, 65, 0], 136, 72, 3),
    ([0, 0, 0], 64, 64, 9),
    ([130, 7, 257], 264, 328, 0),
    ([63, 320, 384, 31], 200, 776, 40),
    ([1] * 40, 512, 264, 2),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
@pytest.mark.parametrize("sizes,K,N,tail", LINEAR)
def test_grouped_linear(sizes, K, N, tail, act, dtype):
    linear_case(gen(K + N), sizes, K, N, act, dtype, bias=True, res=False, tail=tail)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("sizes,K,N,tail", LINEAR[1:6])
def test_grouped_linear_with_a_residual(sizes, K, N, tail, bias, act, dtype):
    linear_case(gen(K + N + 1), sizes, K, N, act, dtype, bias=bias, res=True, tail=tail)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,bias,res", [("none", False, False), ("gelu", True, True), ("relu", True, False)])
@pytest.mark.parametrize("M,K,N", [(1, 256, 48), (16, 1032, 40), (17, 64, 520), (64, 2048, 136),
                                   (65, 136, 264), (300, 520, 392), (700, 264, 1032)])
def test_dense_linear(M, K, N, act, bias, res, dtype):
    linear_case(gen(M + K), [M], K, N, act, dtype, bias, res, grouped=False)


# Row counts around the edges of 64- to 384-row tiles and of their tails
EDGES = [256, 257, 319, 320, 321, 383, 384, 385, 64, 65, 128, 129, 192, 193, 0, 1, 511, 512, 513, 576, 577, 640,
         300, 440]
# group sizes, and a pair of widths: the wider output takes the tiles named, the other way about the input
# gradient does (together with the weight gradient's tiles)
TILINGS = {"256 rows, group by group": (EDGES, 136, 1400),
           "256 rows, short tiles last": ([997, 640, 575, 1088, 832, 321, 1150, 797], 136, 2000),
           "384 rows": ([1152, 1217, 1534, 385, 1712], 136, 2704),
           "128 rows": ([225] * 40, 200, 520)}


@pytest.mark.parametrize("swap", [False, True])
@pytest.mark.parametrize("tiles", TILINGS)
def test_grouped_linear_over_the_tilings(tiles, swap):
    sizes, K, N = TILINGS[tiles]
    if swap:
        K, N = N, K
    linear_case(gen(len(sizes)), sizes, K, N, "silu", torch.bfloat16, bias=True, res=swap, tail=5)


@pytest.mark.parametrize("M,K,N", [(8192, 136, 2048), (8192, 2048, 136), (6144, 136, 2816), (6100, 2816, 136),
                                   (3000, 2048, 200)])
def test_dense_linear_over_the_tilings(M, K, N):
    linear_case(gen(M), [M], K, N, "gelu_tanh", torch.bfloat16, bias=True, res=True, grouped=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
@pytest.mark.parametrize("M", [1, 200])
def test_activations_far_from_zero(M, act, dtype):
    # from |z| = 30 on value and slope are z and 1, or within 1e-10 of 0, up to the type's range
    lim = torch.finfo(dtype).max
    v = [30.0, 100.0, 1e4, 1e13, 1e20, lim]
    z = torch.tensor(v + [-a for a in v] + [float("inf"), float("nan"), 0.0, -0.0], dtype=dtype, device="cuda")
    x = torch.zeros(M, 64, dtype=dtype, device="cuda")
    w = torch.zeros(16, 64, dtype=dtype, device="cuda")
    b = z.clone().requires_grad_()
    y = ops.expert_linear(x, w, b, activation=act)
    dy = torch.zeros_like(y)
    dy[0] = 1.0
    db, = torch.autograd.grad(y, b, dy)
    keep = act == "none"
    z64 = z[:12].double()
    value = z64 if keep else z64.clamp(min=0)
    slope = torch.ones_like(z64) if keep else (z64 > 0).double()
    tol = ref.u(dtype) + 2.0 ** -20
    for r in (0, M - 1):
        err = (y[r, :12].detach().double() - value).abs()
        assert bool((err <= tol * value.abs() + 1e-10).all()), err
    assert bool(((db[:12].double() - slope).abs() <= tol * slope + 1e-10).all()), db
    assert bool((y[:, 12] == float("inf")).all()) and bool(y[:, 13].isnan().all())
    assert bool((y[:, 14:] == 0).all())


def test_linear_gradients_one_at_a_time():
    g = gen(4)
    x, w, b = normal(g, 100, 64), normal(g, 3, 40, 64, std=0.1), normal(g, 3, 40)
    off = torch.tensor([0, 30, 30, 95], dtype=torch.int32, device="cuda")
    dy = normal(g, 100, 40)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(ops.expert_linear(*leaves, offsets=off, activation="gelu"), leaves, dy)
    for i in range(3):
        one = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(ops.expert_linear(*one, offsets=off, activation="gelu"), one[i], dy)
        assert torch.equal(got, want[i]), i
    assert bool((want[0][95:] == 0).all()) and bool((want[1][1] == 0).all()) and bool((want[2][1] == 0).all())


def test_linear_without_rows():
    w = torch.ones(2, 16, 8, device="cuda", requires_grad=True)
    b = torch.ones(2, 16, device="cuda", requires_grad=True)
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    y = ops.expert_linear(x, w, b, offsets=off)
    assert y.shape == (0, 16)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.zeros_like(y))
    assert dx.shape == x.shape and not bool(dw.any()) and not bool(db.any())


def test_linear_rows_behind_the_last_group_do_not_reach_the_gradients():
    g = gen(14)
    x = normal(g, 90, 64)
    x[70:] = float("nan")
    dy = normal(g, 90, 32)
    dy[70:] = float("inf")
    x.requires_grad_()
    w, b = normal(g, 2, 32, 64).requires_grad_(), normal(g, 2, 32).requires_grad_()
    off = torch.tensor([0, 33, 70], dtype=torch.int32, device="cuda")
    for act in ("none", "silu"):
        y = ops.expert_linear(x, w, b, offsets=off, activation=act)
        assert bool((y[70:] == 0).all()) and bool(torch.isfinite(y).all())
        for t in torch.autograd.grad(y, [x, w, b], dy):
            assert bool(torch.isfinite(t).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,res", [("none", True), ("gelu", False)])
@pytest.mark.parametrize("each", [1, 40, 300])
def test_a_range_of_the_experts(each, act, res, dtype):
    # offsets 3 .. 7 of nine experts' with four weights: the other experts' rows are no expert's
    g = gen(each)
    sizes = torch.full((9,), each, dtype=torch.int64)
    sizes[4] = 0
    off = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)]).int().cuda()
    M = int(off[-1])
    x, r, dy = normal(g, M, 64, dtype=dtype), normal(g, M, 72, dtype=dtype), normal(g, M, 72, dtype=dtype)
    w, b = normal(g, 9, 72, 64, dtype=dtype, std=0.125), normal(g, 9, 72, dtype=dtype)
    a, z = int(off[3]), int(off[7])
    x[:a], x[z:] = float("nan"), float("nan")
    part = [t.clone().requires_grad_() for t in (x, w[3:7].contiguous(), b[3:7].contiguous())]
    y = ops.expert_linear(*part, offsets=off[3:8], activation=act, residual=r if res else None)
    got = torch.autograd.grad(y, part, dy)
    only = [t.clone().requires_grad_() for t in (x[a:z].contiguous(), w[3:7].contiguous(), b[3:7].contiguous())]
    yo = ops.expert_linear(*only, offsets=off[3:8] - off[3], activation=act,
                           residual=r[a:z].contiguous() if res else None)
    want = torch.autograd.grad(yo, only, dy[a:z].contiguous())
    # the tilings may add the products of a sum of n terms in different orders (n 2^-24 S each, S the
    # sum of the terms' sizes, less than the figures below), which may round dz the other way (a step,
    # 2 u, of each term) and the result too
    def close(u, v, n, S, rounded):
        off = 2 * n * 2.0 ** -24 * S + (2 * ref.u(dtype) * S if rounded else 0.0)
        err = (u.double() - v.double()).abs()
        assert bool((err <= off + 2 * ref.u(dtype) * (v.double().abs() + off)).all()), float(err.max())
    close(y[a:z].detach(), yo.detach(), 65, 16.0, False)
    dz = act != "none"
    close(got[0][a:z], want[0], 72, 24.0, dz)
    close(got[1], want[1], each, 2.0 * each + 16.0, dz)
    close(got[2], want[2], each, 2.0 * each + 16.0, dz)
    rest = r if res else torch.zeros_like(r)
    assert torch.equal(y[:a], rest[:a]) and torch.equal(y[z:], rest[z:])
    assert not bool(got[0][:a].any()) and not bool(got[0][z:].any())


def test_more_columns_than_a_launch_of_few_rows_holds():
    # 600 rows of as many experts, 2^20 columns: above 2^32 threads of the few-row kernel
    E, K, N = 600, 8, 1 << 20
    x = torch.ones(E, K, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(E, N, K, dtype=torch.bfloat16, device="cuda")
    ids = torch.arange(E, device="cuda")
    w[:, :, 0] = (ids % 120).to(torch.bfloat16)[:, None]
    w[:, -1, 1] = 0.5
    off = torch.arange(E + 1, dtype=torch.int32, device="cuda")
    y = ops.expert_linear(x, w, offsets=off)
    want = (ids % 120).to(torch.bfloat16)
    assert bool((y[:, :-1] == want[:, None]).all()) and torch.equal(y[:, -1], want + 0.5)


@pytest.mark.parametrize("rows", [20, 3000])
def test_offsets_that_are_none_stay_inside_the_buffers(rows):
    # clamped to the running maximum and to the number of rows
    g = gen(rows)
    x, w = normal(g, rows, 64, dtype=torch.bfloat16), normal(g, 4, 32, 64, dtype=torch.bfloat16)
    bad = torch.tensor([0, rows // 2, -7, rows // 4, 10 ** 9], dtype=torch.int32, device="cuda")
    y = ops.expert_linear(x, w, offsets=bad)
    assert y.shape == (rows, 32) and bool(torch.isfinite(y.float()).all())


# ---------------------------------------------------------------- norms around a block

NORMS = [(1, 8), (1, 2048), (3, 64), (9, 512), (33, 520), (130, 776), (66, 2048), (21, 2056), (17, 4104),
         (600, 1032), (70, 7168), (5, 8200), (3, 16392), (1100, 384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", [None, "channel", "token", "full"])
@pytest.mark.parametrize("T,H", NORMS)
def test_residual_norm(T, H, gate, dtype):
    for post, nxt in ((True, True), (True, False), (False, True), (False, False)):
        norm_case(gen(T + H), T, H, gate, dtype, post, nxt, 0.75)


def norm_case(g, T, H, gate, dtype, post, nxt, scale, eps=1e-5):
    t = {"h": normal(g, T, H, dtype=dtype, std=2.0), "y": normal(g, T, H, dtype=dtype)}
    if post:
        t["w2"] = normal(g, H, dtype=dtype, std=0.2, mean=1.0)
    if gate:
        t["gate"] = normal(g, *{"channel": (H,), "token": (T, 1), "full": (T, H)}[gate], dtype=dtype)
    if nxt:
        t["w3"] = normal(g, H, dtype=dtype, std=0.2, mean=1.0)
    for v in t.values():
        v.requires_grad_()
    d_out = normal(g, T, H, dtype=dtype)
    d_n = normal(g, T, H, dtype=dtype) if nxt else None
    out = ops.residual_norm(t["h"], t["y"], t.get("w2"), gate=t.get("gate"), next_weight=t.get("w3"),
                            residual_scale=scale, eps=eps)
    outs = out if nxt else (out,)
    got = dict(zip(t, torch.autograd.grad(outs, list(t.values()), (d_out, d_n) if nxt else (d_out,))))
    d = {n: v.detach().double() for n, v in t.items()}
    want = ref.norm(d["h"], d["y"], d.get("w2"), d.get("gate"), d.get("w3"), scale, eps, d_out.double(),
                    d_n.double() if nxt else None, dtype)
    for name, v in zip(("h", "n"), outs):
        ref.assert_close(v.detach(), *want[name], name)
    for n, v in got.items():
        ref.assert_close(v, *want["d" + n], f"d{n} post={post} next={nxt}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H", NORMS)
def test_rms_norm(T, H, dtype):
    g = gen(H)
    x, w = normal(g, T, H, dtype=dtype, std=3.0), normal(g, H, dtype=dtype)
    x.requires_grad_()
    w.requires_grad_()
    n = ops.rms_norm(x, w, eps=1e-5)
    d = normal(g, T, H, dtype=dtype)
    dx, dw = torch.autograd.grad(n, [x, w], d)
    want = ref.norm(x.detach().double(), None, None, None, w.detach().double(), 1.0, 1e-5, None, d.double(), dtype)
    ref.assert_close(n.detach(), *want["n"], "n")
    ref.assert_close(dx, *want["dh"], "dx")
    ref.assert_close(dw, *want["dw3"], "dw")


def test_residual_norm_when_one_output_has_no_gradient():
    g = gen(77)
    leaves = [normal(g, 40, 264).requires_grad_(), normal(g, 40, 264).requires_grad_(),
              normal(g, 264).requires_grad_(), normal(g, 264).requires_grad_()]
    h, n = ops.residual_norm(leaves[0], leaves[1], leaves[2], next_weight=leaves[3])
    d = normal(g, 40, 264)
    z = torch.zeros_like(d)
    for only, full in (((h, d), (d, z)), ((n, d), (z, d))):
        got = torch.autograd.grad(only[0], leaves, only[1], retain_graph=True, allow_unused=True)
        want = torch.autograd.grad((h, n), leaves, full, retain_graph=True)
        for a, b in zip(got, want):
            assert torch.allclose(a if a is not None else torch.zeros_like(b), b, rtol=1e-6, atol=1e-6)


def test_norms_without_rows():
    w = torch.ones(64, device="cuda", requires_grad=True)
    gate = torch.ones(64, device="cuda", requires_grad=True)
    h = torch.zeros(0, 64, device="cuda", requires_grad=True)
    out, n = ops.residual_norm(h, h, w, gate=gate, next_weight=w)
    assert out.shape == n.shape == (0, 64)
    for t in torch.autograd.grad((out, n), [h, w, gate], (torch.zeros_like(out), torch.zeros_like(n))):
        assert not bool(t.any())


def test_a_second_derivative_is_refused():
    x = torch.ones(4, 64, device="cuda", requires_grad=True)
    n = ops.rms_norm(x, torch.ones(64, device="cuda"))
    dx, = torch.autograd.grad(n.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_rows_of_zeros_and_large_values():
    # a row of zeros has rstd 1 / sqrt(eps); squares of 1e18 still fit fp32's range
    h = torch.zeros(3, 64, device="cuda")
    y = torch.zeros(3, 64, device="cuda")
    y[1] = 1e18
    w = torch.ones(64, device="cuda")
    out, n = ops.residual_norm(h, y, w, next_weight=w, eps=1e-6)
    assert torch.equal(out[0], h[0]) and torch.equal(n[2], h[0])
    assert torch.allclose(out[1], torch.ones(64, device="cuda"), rtol=1e-6)


def test_shapes_with_a_batch_and_broadcast_gradients():
    g = gen(6)
    h, y = normal(g, 2, 5, 64).requires_grad_(), normal(g, 2, 5, 64)
    gate = normal(g, 2, 5, 1).requires_grad_()
    out, n = ops.residual_norm(h, y, gate=gate, next_weight=torch.ones(64, device="cuda"))
    assert out.shape == n.shape == h.shape
    # sum()'s gradient is a broadcast view with stride 0
    dh, dg = torch.autograd.grad(out.sum(), [h, gate])
    assert torch.equal(dh, torch.ones_like(h)) and torch.allclose(dg, y.sum(2, keepdim=True), atol=1e-5)


# ---------------------------------------------------------------- as a user runs them

def chain(x, idx, w, p, E):
    """Tokens to biased experts of two products and back, then the norms around the block."""
    n = ops.rms_norm(x, p["pre"])
    order = ops.sort_tokens(idx, E)
    a = ops.expert_linear(ops.permute_tokens(n, order), p["w1"], p["b1"], offsets=order.offsets, activation="gelu")
    b = ops.expert_linear(a, p["w2"], p["b2"], offsets=order.offsets)
    return ops.residual_norm(x, ops.unpermute_tokens(b, order, w), p["post"], gate=p["gate"], next_weight=p["next"])


def chain_inputs(g, T, H, I, E, k, dtype):
    p = {"pre": normal(g, H, dtype=dtype, std=0.1, mean=1.0), "post": normal(g, H, dtype=dtype, std=0.1, mean=1.0),
         "next": normal(g, H, dtype=dtype, std=0.1, mean=1.0), "gate": normal(g, H, dtype=dtype, std=0.5),
         "w1": normal(g, E, I, H, dtype=dtype, std=H ** -0.5), "b1": normal(g, E, I, dtype=dtype, std=0.1),
         "w2": normal(g, E, H, I, dtype=dtype, std=I ** -0.5), "b2": normal(g, E, H, dtype=dtype, std=0.1)}
    return p, normal(g, T, H, dtype=dtype), routing(g, T, k, E, pad=0.1), torch.rand(T, k, device="cuda", generator=g)


def chain_plain(x, idx, w, p, E):
    """The same in torch, every expert on every token."""
    def rms(t, weight):
        return t * torch.rsqrt(t.square().mean(1, keepdim=True) + 1e-6) * weight
    n = rms(x, p["pre"])
    y = torch.zeros_like(x)
    for e in range(E):
        out = torch.nn.functional.gelu(n @ p["w1"][e].t() + p["b1"][e]) @ p["w2"][e].t() + p["b2"][e]
        y = y + (w * (idx == e)).sum(1, keepdim=True) * out
    h = x + p["gate"] * rms(y, p["post"])
    return h, rms(h, p["next"])


def test_a_run_of_them_with_its_gradients():
    T, H, I, E, k = 150, 136, 200, 6, 2
    p, x, idx, w = chain_inputs(gen(21), T, H, I, E, k, torch.float32)
    leaves = [x, w] + list(p.values())
    for t in leaves:
        t.requires_grad_()
    h, n = chain(x, idx, w, p, E)
    dh, dn = normal(gen(22), T, H), normal(gen(23), T, H)
    got = torch.autograd.grad((h, n), leaves, (dh, dn))
    d = [t.detach().double().requires_grad_() for t in leaves]
    q = dict(zip(p, d[2:]))
    h64, n64 = chain_plain(d[0], idx, d[1], q, E)
    want = torch.autograd.grad((h64, n64), d, (dh.double(), dn.double()))
    # sums of up to T k I = 60000 fp32 terms, whose roundings add up like their root: 2^-24 sqrt(60000)
    # = 1.5e-5 of the magnitudes
    for name, a, b in zip(["h", "n", "x", "w"] + list(p), (h, n) + got, (h64, n64) + want):
        err = float(((a.double() - b).norm() / b.norm()).detach())
        assert err < 1.5e-5, (name, err)


def test_gradients_against_differences():
    T, H, I, E, k = 12, 16, 24, 3, 2
    p, x, idx, w = chain_inputs(gen(31), T, H, I, E, k, torch.float32)
    leaves = {"x": x, "w": w, **p}
    for t in leaves.values():
        t.requires_grad_()
    up = [normal(gen(32), T, H), normal(gen(33), T, H)]

    def loss():
        h, n = chain(x, idx, w, p, E)
        return (h.double() * up[0]).sum() + (n.double() * up[1]).sum()
    grads = dict(zip(leaves, torch.autograd.grad(loss(), list(leaves.values()))))
    step = 2.0 ** -7
    for name, t in leaves.items():
        way = normal(gen(len(name)), *t.shape)
        slope = float((grads[name].double() * way.double()).sum())
        with torch.no_grad():
            keep = t.clone()
            values = []
            for s in (-2, -1, 1, 2):
                t.copy_(keep + s * step * way)
                values.append(float(loss()))
            t.copy_(keep)
        # five points: off by step^4 of the fifth derivative; the loss is a sum of 2 T H = 384 fp32
        # outputs of size about 1, each off by some 2^-22: 384^(1/2) 2^-22 / step = 6e-4 at most here
        diff = (values[0] - 8 * values[1] + 8 * values[2] - values[3]) / (12 * step)
        assert abs(diff - slope) < 2e-3 * max(1.0, float(grads[name].norm()) * float(way.norm()) ** 0.5), \
            (name, diff, slope)


@pytest.mark.parametrize("post,gate,scale", [(True, False, 1.0), (False, True, 1.0), (True, True, 0.5),
                                             (False, False, 0.75)])
def test_block_with_norms_on_both_sides(post, gate, scale):
    cfg = MoeConfig(hidden_size=64, num_experts=6, experts_per_tok=2, intermediate_size=48, post_norm=post,
                    residual_gate=gate, residual_scale=scale)
    block = MoeBlock(cfg, torch.float32)
    g = gen(17)
    with torch.no_grad():
        for name, p in block.trainable_parameters():
            p.normal_(1.0 if "layernorm" in name or name == "residual_gate" else 0.0, 0.1, generator=g)
    names = [n for n, _ in block.trainable_parameters()]
    assert ("post_ffn_layernorm.weight" in names) == post and ("residual_gate" in names) == gate
    h = normal(g, 2, 35, 64).requires_grad_()
    out, aux, z = block(h)
    # the same from the layer's own forward and torch, in float64 around it
    def rms(t, w):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + cfg.rms_norm_eps) * w
    h2 = h.detach().double().requires_grad_()
    leaves = {n: p for n, p in block.named_parameters() if not n.startswith("ffn.")}
    d = {n: p.detach().double().requires_grad_() for n, p in leaves.items()}
    x = rms(h2, d["post_attention_layernorm.weight"])
    y, aux2, z2 = block.ffn(x.float())
    y = y.double()
    u = rms(y, d["post_ffn_layernorm.weight"]) if post else y
    want = scale * h2 + (d["residual_gate"] if gate else 1.0) * u
    up = normal(gen(18), 2, 35, 64)
    got = torch.autograd.grad(out, [h] + list(leaves.values()), up)
    ref64 = torch.autograd.grad(want, [h2] + list(d.values()), up.double())
    # the layer runs in fp32 on both sides, on inputs that differ by an fp32 rounding: sums of 64 and 48
    # terms there, 70 x 64 in the weights' gradients; 2^-24 sqrt(4480) = 4e-6 of the magnitudes
    assert torch.allclose(aux, aux2, rtol=1e-5) and torch.allclose(z, z2, rtol=1e-5)
    for name, a, b in zip(["out", "h"] + list(leaves), (out,) + got, (want,) + ref64):
        err = float(((a.double() - b).norm() / b.norm()).detach())
        assert err < 4e-6, (name, err)
    plain = MoeBlock(MoeConfig(hidden_size=64, num_experts=6, experts_per_tok=2, intermediate_size=48),
                     torch.float32)
    assert plain.ffn.cfg.fused_block and not block.ffn.cfg.fused_block


@pytest.mark.parametrize("T", [3, 500])
def test_replayed_graph_gives_the_eager_results(T):
    H, I, E, k = 264, 136, 9, 3
    p, x, idx, w = chain_inputs(gen(T), T, H, I, E, k, torch.bfloat16)
    leaves = [x, w] + list(p.values())
    for t in leaves:
        t.requires_grad_()
    dh, dn = normal(gen(1), T, H, dtype=torch.bfloat16), normal(gen(2), T, H, dtype=torch.bfloat16)

    def step():
        h, n = chain(x, idx, w, p, E)
        return (h.detach(), n.detach()) + torch.autograd.grad((h, n), leaves, (dh, dn))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        q, x2, idx2, w2 = chain_inputs(gen(100 + seed), T, H, I, E, k, torch.bfloat16)
        with torch.no_grad():
            for a, b in zip(leaves, [x2, w2] + list(q.values())):
                a.copy_(b)
            idx.copy_(idx2)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = step()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (seed, i)


def test_calls_on_two_streams_at_once():
    H, I, E, k = 520, 264, 8, 2
    sets = [chain_inputs(gen(s), 400, H, I, E, k, torch.bfloat16) for s in (1, 2)]
    want = [chain(x, idx, w, p, E) for p, x, idx, w in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, (p, x, idx, w) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i] = chain(x, idx, w, p, E)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_kept_tensors_may_move_or_be_made_again():
    # saved tensors offloaded to the host and back, and a forward run again in the backward
    p, x, idx, w = chain_inputs(gen(8), 120, 264, 136, 5, 2, torch.bfloat16)
    leaves = [x, w] + list(p.values())
    for t in leaves:
        t.requires_grad_()
    d = normal(gen(9), 2, 120, 264, dtype=torch.bfloat16)

    def grads(h, n):
        return torch.autograd.grad((h, n), leaves, (d[0], d[1]))
    want = grads(*chain(x, idx, w, p, 5))
    with torch.autograd.graph.save_on_cpu():
        out = chain(x, idx, w, p, 5)
    again = torch.utils.checkpoint.checkpoint(lambda a: chain(a, idx, w, p, 5), x, use_reentrant=False)
    for got in (grads(*out), grads(*again)):
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_threads_with_streams_of_their_own():
    sets = [chain_inputs(gen(s), 300, 264, 136, 6, 2, torch.bfloat16) for s in range(3)]
    want = [chain(x, idx, w, p, 6) for p, x, idx, w in sets]
    torch.cuda.synchronize()
    got = [None] * 3

    def work(i):
        p, x, idx, w = sets[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = chain(x, idx, w, p, 6)
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_strided_and_misaligned_inputs():
    g = gen(9)
    base = normal(g, 64, 3 * 64)
    x = base[:, 64:128]
    w = normal(g, 64, 48).t()                              # [48, 64], columns first
    flat = normal(g, 64 * 48 + 1)[1:].view(64, 48)         # 4 bytes off a 16-byte boundary
    want = ops.expert_linear(x.contiguous(), w.contiguous(), residual=flat.clone())
    assert torch.equal(ops.expert_linear(x, w, residual=flat), want)
    n = ops.rms_norm(x, base[0, :64])
    assert torch.equal(n, ops.rms_norm(x.contiguous(), base[0, :64].clone()))
    order = ops.sort_tokens(routing(g, 64, 2, 4), 4)
    assert torch.equal(ops.permute_tokens(x, order), ops.permute_tokens(x.contiguous(), order))


def test_results_are_the_same_bits_every_time():
    p, x, idx, w = chain_inputs(gen(41), 300, 264, 392, 7, 3, torch.bfloat16)
    leaves = [x, w] + list(p.values())
    for t in leaves:
        t.requires_grad_()

    def step():
        h, n = chain(x, idx, w, p, 7)
        return (h, n) + torch.autograd.grad((h, n), leaves, (torch.ones_like(h), torch.ones_like(n)))
    first = step()
    for _ in range(3):
        for a, b in zip(first, step()):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- offsets past 32 bits

def test_rows_past_2_31_elements():
    T, k, H, E = 70000, 8, 4104, 16  # 2.3e9 elements of rows
    g = gen(3)
    order = ops.sort_tokens(routing(g, T, k, E, pad=0.05), E)
    x = normal(g, T, H, dtype=torch.bfloat16).requires_grad_()
    rows = ops.permute_tokens(x, order)
    kept = int(order.offsets[-1])
    assert kept * H > 2 ** 31
    at = torch.cat([torch.arange(64), torch.arange(kept - 64, kept + 64), torch.arange(T * k - 64, T * k)]).cuda()
    assert torch.equal(rows[at], torch.where((at < kept)[:, None], x.detach()[order.perm[at].long() // k], 0.0))
    w = torch.rand(T, k, device="cuda", generator=g).requires_grad_()
    y = rows.detach().requires_grad_()
    out = ops.unpermute_tokens(y, order, w)
    dout = normal(g, T, H, dtype=torch.bfloat16)
    dy, dw = torch.autograd.grad(out, [y, w], dout)
    few = torch.cat([torch.arange(32), torch.arange(T - 32, T)]).cuda()
    pos = order.inv_perm[few].long()
    real = (pos < kept).double()
    v, d, w64 = y.detach()[pos].double(), dout[few].double(), w.detach()[few].double() * real
    ref.assert_close(out.detach()[few], (w64[:, :, None] * v).sum(1),
                     k * ref.U32 * (w64[:, :, None] * v.abs()).sum(1), "out")
    ref.assert_close(dy[pos.flatten()], (w64[:, :, None] * d[:, None]).flatten(0, 1), 0.0, "dy")
    ref.assert_close(dw[few], (d[:, None] * v).sum(2) * real, H * ref.U32 * (d[:, None] * v).abs().sum(2), "dw")
    del v
    dx, = torch.autograd.grad(rows, x, dy)
    ref.assert_close(dx[few], (dy[pos].double() * real[:, :, None]).sum(1),
                     k * ref.U32 * dy[pos].double().abs().sum(1), "dx")


def test_norm_past_2_31_elements():
    T, H = 300000, 7176
    g = gen(4)
    w = [normal(g, H, dtype=torch.bfloat16).requires_grad_() for _ in range(3)]
    h, y = (normal(g, T, H, dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    dh, dn = normal(g, T, H, dtype=torch.bfloat16), normal(g, T, H, dtype=torch.bfloat16)

    def step(a, b):
        p, q = (t.detach()[a:b].requires_grad_() for t in (h, y))
        out, n = ops.residual_norm(p, q, w[0], gate=w[1], next_weight=w[2])
        return (out.detach(), n.detach()) + torch.autograd.grad((out, n), [p, q], (dh[a:b], dn[a:b]))
    for big, small in zip(step(0, T), step(T - 40, T)):  # a row's results are its own
        assert torch.equal(big[-40:], small)


@pytest.mark.parametrize("grouped", [True, False])
def test_linear_past_2_31_elements(grouped):
    M, K, N = 1050003, 64, 2056
    g = gen(5)
    x = normal(g, M, K, dtype=torch.bfloat16)
    w = normal(g, *((3, N, K) if grouped else (N, K)), dtype=torch.bfloat16, std=0.125)
    off = torch.tensor([0, 500000, 500000, M - 3], dtype=torch.int32, device="cuda") if grouped else None
    res = normal(g, M, N, dtype=torch.bfloat16)
    y = ops.expert_linear(x, w, offsets=off, residual=res)
    at = torch.cat([torch.arange(40), torch.arange(M - 300, M - 3)]).cuda()
    for part, e in ((at[:40], 0), (at[40:], 2)):
        a, b = x[part].double(), (w[e] if grouped else w).double()
        ref.assert_close(y[part], a @ b.t() + res[part].double(),
                         (K + 1) * ref.U32 * (a.abs() @ b.abs().t() + res[part].double().abs()), "y")
    if grouped:
        assert torch.equal(y[-3:], res[-3:])


# ---------------------------------------------------------------- empty batches

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("grouped", [True, False])
def test_linear_gradients_without_rows(grouped, act, dtype):
    w = torch.ones(*((2, 64, 128) if grouped else (64, 128)), dtype=dtype, device="cuda", requires_grad=True)
    b = torch.ones(*((2, 64) if grouped else (64,)), dtype=dtype, device="cuda", requires_grad=True)
    x = torch.zeros(0, 128, dtype=dtype, device="cuda", requires_grad=True)
    r = torch.zeros(0, 64, dtype=dtype, device="cuda", requires_grad=True)
    off = torch.zeros(3, dtype=torch.int32, device="cuda") if grouped else None
    y = ops.expert_linear(x, w, b, offsets=off, activation=act, residual=r)
    assert y.shape == (0, 64)
    dx, dw, db, dr = torch.autograd.grad(y, [x, w, b, r], torch.zeros_like(y))
    assert dx.shape == x.shape and dr.shape == r.shape
    assert dw.shape == w.shape and not bool(dw.any()) and db.shape == b.shape and not bool(db.any())


# ---------------------------------------------------------------- what the norm's backward is taken of

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", [None, "channel", "token", "full"])
@pytest.mark.parametrize("T,H", [(1, 64), (130, 776), (66, 2048), (70, 7168), (5, 8200), (3, 16392)])
def test_norm_gradients_are_those_of_the_unrounded_residual(T, H, gate, dtype):
    # no rounding of h_out to the dtype between the forward and its gradients
    for post in (True, False):
        g = gen(T + H + 7)
        t = {"h": normal(g, T, H, dtype=dtype, std=2.0), "y": normal(g, T, H, dtype=dtype)}
        if post:
            t["w2"] = normal(g, H, dtype=dtype, std=0.2, mean=1.0)
        if gate:
            t["gate"] = normal(g, *{"channel": (H,), "token": (T, 1), "full": (T, H)}[gate], dtype=dtype)
        t["w3"] = normal(g, H, dtype=dtype, std=0.2, mean=1.0)
        for v in t.values():
            v.requires_grad_()
        d_out, d_n = normal(g, T, H, dtype=dtype), normal(g, T, H, dtype=dtype)
        out, n = ops.residual_norm(t["h"], t["y"], t.get("w2"), gate=t.get("gate"), next_weight=t["w3"],
                                   residual_scale=1.25, eps=1e-5)
        got = dict(zip(t, torch.autograd.grad((out, n), list(t.values()), (d_out, d_n))))
        d = {name: v.detach().double() for name, v in t.items()}
        want = ref.norm(d["h"], d["y"], d.get("w2"), d.get("gate"), d["w3"], 1.25, 1e-5, d_out.double(),
                        d_n.double(), dtype, hn_rounded=False)
        for name, v in got.items():
            ref.assert_close(v, *want["d" + name], f"d{name} post={post}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", [0, 1, 2, 3])
def test_the_c_entry_that_takes_the_rounded_residual(kind, dtype):
    T, H, scale = 37, 520, 0.5
    g = gen(kind)
    h, y = normal(g, T, H, dtype=dtype, std=2.0), normal(g, T, H, dtype=dtype)
    w2, w3 = normal(g, H, dtype=dtype, std=0.2, mean=1.0), normal(g, H, dtype=dtype, std=0.2, mean=1.0)
    gate = [None, normal(g, H, dtype=dtype), normal(g, T, 1, dtype=dtype), normal(g, T, H, dtype=dtype)][kind]
    d_out, d_n = normal(g, T, H, dtype=dtype), normal(g, T, H, dtype=dtype)
    L, code = _lib.load(), _lib.MOE_DTYPE_F32 if dtype == torch.float32 else _lib.MOE_DTYPE_BF16
    out, n = torch.empty_like(h), torch.empty_like(h)
    r2, r3 = (torch.empty(T, device="cuda") for _ in range(2))
    stream = torch.cuda.current_stream().cuda_stream

    def p(t):
        return None if t is None else t.data_ptr()
    _lib.check(L.moe_residual_norm(0, stream, code, T, H, p(h), p(y), p(w2), p(gate), kind, p(w3), scale, 1e-5,
                                   p(out), p(n), p(r2), p(r3)))
    ws = torch.empty(L.moe_residual_norm_workspace_bytes(T, H), dtype=torch.uint8, device="cuda")
    d = [None if t is None else t.double() for t in (h, y, w2, gate, w3)]
    for entry, kept, rounded in ((L.moe_residual_norm_backward, out, True),
                                 (L.moe_residual_norm_backward_from_input, h, False)):
        got = {"h": torch.empty_like(h), "y": torch.empty_like(y), "w2": torch.empty_like(w2),
               "gate": None if gate is None else torch.empty_like(gate), "w3": torch.empty_like(w3)}
        _lib.check(entry(0, stream, code, T, H, p(d_out), p(d_n), p(kept), p(y), p(w2), p(gate), kind, p(w3), scale,
                         p(r2), p(r3), p(got["h"]), p(got["y"]), p(got["w2"]), p(got["gate"]), p(got["w3"]), p(ws)))
        want = ref.norm(*d, scale, 1e-5, d_out.double(), d_n.double(), dtype, hn_rounded=rounded)
        for name, t in got.items():
            if t is not None:
                ref.assert_close(t, *want["d" + name], "d" + name)


# ---------------------------------------------------------------- activations relative to their value

def activation_of(z, act, rows):
    """act(z) and act'(z) of each z through expert_linear, by way of its bias."""
    n = (z.numel() + 7) // 8 * 8
    b = torch.cat([z, z.new_zeros(n - z.numel())]).requires_grad_()
    y = ops.expert_linear(z.new_zeros(rows, 64), z.new_zeros(n, 64), b, activation=act)
    dy = torch.zeros_like(y)
    dy[rows - 1] = 1.0
    slope, = torch.autograd.grad(y, b, dy)
    return y.detach()[:, :z.numel()], slope[:z.numel()]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 200])
def test_gelu_keeps_its_relative_error_in_the_tails(rows, dtype):
    z = torch.linspace(-12.0, 12.0, 2401).to(dtype).cuda()
    y, slope = activation_of(z, "gelu", rows)
    z64 = z.double()
    cdf = 0.5 * torch.special.erfc(-z64 * 0.5 ** 0.5)
    pdf = torch.exp(-z64 * z64 / 2) / (2.0 * torch.pi) ** 0.5
    # fp32: erfc to 16 steps (2^-20) of its value; its argument and exp's are off by 1.5 steps and one, which
    # moves their values by up to z^2 2^-23 and less.  bf16: 2^-18 for the polynomial and the approximate exp
    # and reciprocal; exp's argument, rounded twice, by z^2 2^-23
    rel = (2.0 ** -20 if dtype == torch.float32 else 2.0 ** -18) + z64 * z64 * 2.0 ** -23
    for r in (0, rows - 1):
        ref.assert_close(y[r], z64 * cdf, (z64 * cdf).abs() * rel, "gelu")
    ref.assert_close(slope, cdf + z64 * pdf, (cdf + (z64 * pdf).abs()) * rel, "gelu'")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_logistic_activations_keep_their_relative_error(act, rows, dtype):
    z = torch.linspace(-9.0, 9.0, 2401).to(dtype).cuda()
    if act == "silu":
        z = z * 8
    y, _ = activation_of(z, act, rows)
    z64 = z.double()
    # z logistic(a); a of gelu_tanh takes five roundings.  fp32: exp, sum, division and product to some eight
    # steps together; bf16: v_exp_f32's argument rounded once more, a reciprocal of one step
    a = z64 if act == "silu" else 2 * (2 / torch.pi) ** 0.5 * (z64 + 0.044715 * z64 ** 3)
    steps = (0.0 if act == "silu" else 5.0) + (0.0 if dtype == torch.float32 else 2.0)
    want = z64 * torch.sigmoid(a)
    for r in (0, rows - 1):
        ref.assert_close(y[r], want, want.abs() * (8 + steps * a.abs()) * 2.0 ** -24, act)


# ---------------------------------------------------------------- derivatives that the operators do not have

def test_forward_mode_and_traces_are_refused_on_the_device():
    from torch.fx.experimental.proxy_tensor import make_fx
    g = gen(2)
    x, w = normal(g, 40, 64), normal(g, 64)
    order = ops.sort_tokens(routing(g, 40, 2, 4), 4)
    calls = [lambda t: ops.rms_norm(t, w), lambda t: ops.permute_tokens(t, order),
             lambda t: ops.unpermute_tokens(torch.cat([t, t]), order), lambda t: ops.expert_linear(t, w[None].repeat(8, 1)),
             lambda t: ops.residual_norm(t, t)]
    for call in calls:
        want = call(x)
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match="forward mode"):
                call(torch.autograd.forward_ad.make_dual(x, x))
            assert torch.equal(call(x), want)
        with pytest.raises(ModelError, match="traced"):
            make_fx(call)(x)
        assert torch.equal(call(x), want)


# ---------------------------------------------------------------- gradients past 2^31 bytes, without the weight's

@pytest.mark.parametrize("grouped", [True, False])
@pytest.mark.parametrize("K,N", [(64, 4104), (4104, 64)])
def test_gradients_of_rows_past_2_31_bytes_without_the_weights(K, N, grouped):
    M, dt = 262151, torch.bfloat16
    assert M * max(K, N) * 2 > 2 ** 31
    g = gen(K)
    x, r = normal(g, M, K, dtype=dt).requires_grad_(), normal(g, M, N, dtype=dt).requires_grad_()
    w = normal(g, *((3, N, K) if grouped else (N, K)), dtype=dt, std=K ** -0.5)
    b = normal(g, *((3, N) if grouped else (N,)), dtype=dt, std=0.3).requires_grad_()
    edges = [0, 100000, 100000, M - 4]
    off = torch.tensor(edges, dtype=torch.int32, device="cuda") if grouped else None
    dy = normal(g, M, N, dtype=dt)
    y = ops.expert_linear(x, w, b, offsets=off, activation="silu", residual=r)
    dx, db, dr = torch.autograd.grad(y, [x, b, r], dy)
    assert torch.equal(dr, dy)
    for e, (lo, hi) in enumerate(zip(edges, edges[1:]) if grouped else [(0, M)]):
        want, bound = torch.zeros(N, dtype=torch.float64, device="cuda"), 0.0
        for i in range(lo, hi, 16384):
            s = slice(i, min(i + 16384, hi))
            part = ref.linear(x.detach()[s].double(), (w[e] if grouped else w).double(),
                              (b.detach()[e] if grouped else b.detach()).double(), None, "silu",
                              r.detach()[s].double(), dy[s].double(), dt)
            ref.assert_close(y.detach()[s], *part["y"], "y")
            ref.assert_close(dx[s], *part["dx"], "dx")
            want += part["db"][0]
            bound = bound + part["db"][1] + (hi - lo) / 64 * ref.U32 * part["db"][0].abs()
        # the chunks' sums add up in fp32: at most (hi - lo) / 64 more terms, each smaller than their bounds' sums
        ref.assert_close(db[e] if grouped else db, want, bound + (hi - lo) * ref.U32 * dy[lo:hi].double().abs().sum(0), "db")
    if grouped:
        assert not bool(dx[M - 4:].any()) and torch.equal(y[M - 4:], r[M - 4:])


# ---------------------------------------------------------------- what of an order a backward needs

def test_counts_and_perm_may_be_written_before_a_backward():
    g = gen(8)
    idx = routing(g, 20, 2, 4, pad=0.2)
    w = torch.rand(20, 2, device="cuda", generator=g)
    x = normal(g, 20, 64).requires_grad_()

    def run(write):
        order = ops.sort_tokens(idx, 4)
        check_order(order, idx, 4)
        out = ops.unpermute_tokens(ops.permute_tokens(x, order), order, w)
        write(order)
        return torch.autograd.grad(out, x, torch.ones_like(out))[0]
    want = run(lambda o: None)
    assert torch.equal(run(lambda o: (o.counts.add_(1), o.perm.zero_())), want)
    for field in ("inv_perm", "offsets"):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            run(lambda o: getattr(o, field).zero_())


# ---------------------------------------------------------------- past what one launch holds

def test_a_backward_of_too_many_tiles_is_refused_in_the_forward():
    E, N = 1024, 1 << 20
    w = torch.empty(E, N, 8, device="cuda", requires_grad=True)  # 32 GiB, not read
    x = torch.zeros(100, 8, device="cuda")
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.MoeError, match="too many rows or tiles"):
        ops.expert_linear(x, w, offsets=off)
    del w
    torch.cuda.empty_cache()


def test_the_gradient_of_no_rows_past_2_36_bytes():
    # zeros over more bytes than one launch of 16-byte stores covers
    shape = (33, 32768, 32760)
    w = torch.empty(shape, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    assert w.numel() * 2 > 2 ** 36
    block = torch.ones(shape, dtype=torch.bfloat16, device="cuda")
    del block  # its memory is the gradient's next
    off = torch.zeros(34, dtype=torch.int32, device="cuda")
    y = ops.expert_linear(torch.zeros(0, 32760, dtype=torch.bfloat16, device="cuda"), w, offsets=off)
    dw, = torch.autograd.grad(y, w, torch.zeros_like(y))
    for part in dw:
        assert not bool(part.any())
    del w, dw, y
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- the block in bf16

@pytest.mark.parametrize("post,gate,scale", [(True, False, 1.0), (False, True, 1.0), (True, True, 0.5),
                                             (False, False, 0.75)])
def test_block_with_norms_on_both_sides_in_bf16(post, gate, scale):
    dt = torch.bfloat16
    cfg = MoeConfig(hidden_size=136, num_experts=6, experts_per_tok=2, intermediate_size=48, post_norm=post,
                    residual_gate=gate, residual_scale=scale)
    block = MoeBlock(cfg, dt)
    g = gen(27)
    with torch.no_grad():
        for name, p in block.trainable_parameters():
            p.normal_(1.0 if "layernorm" in name or name == "residual_gate" else 0.0, 0.1, generator=g)
    h, up = normal(g, 2, 65, 136, dtype=dt).requires_grad_(), normal(g, 2, 65, 136, dtype=dt)
    norms = {n: p for n, p in block.named_parameters() if not n.startswith("ffn.")}
    leaves = [h] + list(norms.values()) + [block.ffn.router.gate.weight]
    out, aux, z = block(h)
    got = torch.autograd.grad((out, aux, z), leaves, (up, torch.ones_like(aux), torch.ones_like(z)))
    # the same calls one by one: the same bits
    x = ops.rms_norm(h, block.post_attention_layernorm.weight, cfg.rms_norm_eps)
    y, aux2, z2 = block.ffn(x)
    w2 = block.post_ffn_layernorm.weight if post else None
    out2 = ops.residual_norm(h, y, w2, gate=block.residual_gate, residual_scale=scale, eps=cfg.rms_norm_eps)
    want = torch.autograd.grad((out2, aux2, z2), leaves, (up, torch.ones_like(aux), torch.ones_like(z)))
    for a, b in zip((out, aux, z) + got, (out2, aux2, z2) + want):
        assert torch.equal(a, b)
    # and what is around the layer against float64
    d = [None if t is None else t.detach().double() for t in (h.view(-1, 136), y.view(-1, 136), w2, block.residual_gate)]
    ref64 = ref.norm(*d, None, scale, cfg.rms_norm_eps, up.view(-1, 136).double(), None, dt)
    ref.assert_close(out.detach().view(-1, 136), *ref64["h"], "out")
    pre = ref.norm(d[0], None, None, None, block.post_attention_layernorm.weight.detach().double(), 1.0,
                   cfg.rms_norm_eps, None, None, dt)
    ref.assert_close(x.detach().view(-1, 136), *pre["n"], "x")
    for name, key in (("post_ffn_layernorm.weight", "dw2"), ("residual_gate", "dgate")):
        if name in norms:
            ref.assert_close(got[1 + list(norms).index(name)], *ref64[key], name)


def test_rows_of_few_columns_past_2_24():
    # four rows to a block: 2^24 rows are a quarter of what a launch takes
    T, H = (1 << 24) + 5, 64
    g = gen(6)
    x = normal(g, T, H, dtype=torch.bfloat16)
    w = normal(g, H, dtype=torch.bfloat16)
    n = ops.rms_norm(x, w)
    idx = torch.arange(T, device="cuda", dtype=torch.int32)[:, None] % 7
    order = ops.sort_tokens(idx, 7)
    weights = torch.rand(T, 1, device="cuda", generator=g).requires_grad_()
    y = x.requires_grad_()
    dy, dw = torch.autograd.grad(ops.unpermute_tokens(y, order, weights), [y, weights], n)
    for at in (slice(0, 50), slice(T - 50, T)):
        d = x.detach()[at].double()
        want = ref.norm(d, None, None, None, w.double(), 1.0, 1e-6, None, None, torch.bfloat16)
        ref.assert_close(n[at], *want["n"], "n")
        pos = order.inv_perm[at, 0].long()
        rows, up = x.detach()[pos].double(), n[at].double()
        ref.assert_close(dy[pos], weights.detach()[at].double() * up, 0.0, "dy")
        ref.assert_close(dw[at, 0], (rows * up).sum(1), (H + 8) * ref.U32 * (rows * up).abs().sum(1), "dw")
