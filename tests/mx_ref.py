"""Plain float64 forms of the router's losses and of 4-bit numbers, with bounds on what the kernels may be off, from
arithmetic (see ops_ref for the conventions)."""
import torch

from tests.ops_ref import U32, u

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


# ---- 4-bit numbers
def quantize(x):
    """(codes, scales) uint8 of x [..., K], from the definition; float64 holds every step exactly."""
    v = x.double().unflatten(-1, (-1, 32))
    a = v.abs()
    amax = a.amax(-1, keepdim=True)
    bad = ~torch.isfinite(a).all(-1, keepdim=True)
    exp = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp(min=-127)
    a = a * torch.exp2(-exp.double())
    grid = GRID.to(x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    code = torch.bucketize(a.contiguous(), mid)               # below or at a border: the lower code
    tie = torch.isin(a, mid) & (code % 2 == 1)   # at it, the even one
    code = code + tie
    code = (code + 8 * torch.signbit(v)).to(torch.uint8)
    code = torch.where(bad, torch.zeros_like(code), code).flatten(-2)
    scale = torch.where(bad, 255, exp + 127).to(torch.uint8).squeeze(-1)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def values(codes, scales):
    """float64 numbers that codes and scales stand for."""
    grid = torch.cat((GRID, -GRID)).to(codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, float("nan"), s)
    return (grid[both.int()].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


# ---- losses of a router
def losses(logits, idx, score, tau, c_sw, c_sq, offsets, d_balance, d_z):
    """{name: (reference, error bound)} of router_losses and its gradient. logits float64 of what the kernel reads.

    fp32 roundings counted: x = logits / tau twice, x - max once, each exponential and quotient a few; a sum over
    a row's E <= 1024 columns takes at most 16 in a lane and 6 over lanes. So q and p are within c = (8 R + 64) U32 of
    themselves, R the row's largest |x|, and lse within c + U32 |lse|. Column sums: at most rows / 4096 + 1 in a lane, and
    some 30 over lanes, waves and in the last division."""
    T, E = logits.shape
    k = idx.shape[1]
    bounds = offsets.tolist() if offsets is not None else [0, T]
    S = len(bounds) - 1
    f64 = dict(dtype=torch.float64, device=logits.device)
    balance, z, be, ze = (torch.zeros(S, **f64) for _ in range(4))
    counts = torch.zeros(S, E, dtype=torch.int32, device=logits.device)
    d, de = torch.zeros(T, E, **f64), torch.zeros(T, E, **f64)
    cs = (T // 4096 + 40) * U32
    for s, (a, b) in enumerate(zip(bounds[:-1], bounds[1:])):
        i = idx[a:b].long()
        ok = (i >= 0) & (i < E)
        real = ok.any(1)
        counts[s] = torch.bincount(i[ok], minlength=E).to(torch.int32)
        n = int(real.sum())
        if n == 0:
            continue
        x = logits[a:b][real] / tau
        lse = torch.logsumexp(x, 1)
        p = torch.softmax(x, 1)
        R = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(1, keepdim=True)
        c = (8 * R + 64) * U32
        le = (c[:, 0] + U32 * lse.abs())
        if score == "softmax":
            q, curve = p, torch.ones_like(p)
        else:
            ls = torch.nn.functional.logsigmoid(x)
            q, curve = torch.softmax(ls, 1), torch.sigmoid(-x)
        P = q.sum(0) / n
        Pe = (q * c).sum(0) / n + cs * P
        f = counts[s].double() / (k * n)
        lin, sq = abs(c_sw) * f * P, abs(c_sq) * P * P
        balance[s] = E * (c_sw * f * P + c_sq * P * P).sum()
        be[s] = E * (abs(c_sw) * f * Pe + 2 * abs(c_sq) * P * Pe + 40 * U32 * (lin + sq)).sum()
        z[s] = lse.square().mean()
        ze[s] = (2 * lse.abs() * le).mean() + cs * z[s]
        if d_balance is None and d_z is None:
            continue
        db = float(d_balance[s]) if d_balance is not None else 0.0
        dz = float(d_z[s]) if d_z is not None else 0.0
        g = db * E * (c_sw * f + 2 * c_sq * P) / n
        gm = abs(db) * E * (abs(c_sw) * f + 2 * abs(c_sq) * P) / n
        ge = abs(db) * E * 2 * abs(c_sq) * Pe / n + 12 * U32 * gm
        h = 2 * dz / n
        dot = (q * g).sum(1, keepdim=True)
        dote = (q * (ge + (2 * c + 30 * U32) * gm)).sum(1, keepdim=True)
        t = q * curve * (g - dot)
        te = q * curve * (ge + dote + (2 * c + 16 * U32) * (gm + (q * gm).sum(1, keepdim=True)))
        w = h * lse[:, None] * p
        we = w.abs() * (2 * c + 16 * U32) + abs(h) * p * le[:, None]
        rows = torch.arange(a, b, device=logits.device)[real]
        d[rows], de[rows] = (t + w) / tau, (te + we) / tau + 8 * U32 * (t.abs() + w.abs()) / tau
    return {"balance": (balance, be), "z": (z, ze), "counts": counts, "d": (d, de)}


def assert_close(got, ref, err, what):
    """|got - ref| <= err + u |ref|, and the same infinities and NaN."""
    g, bound = got.double(), (err + u(got.dtype) * ref.abs()) * (1 + 2 * u(got.dtype)) + 1e-37
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (g - ref).abs()
    bad = ~((off <= bound) | (g == ref) | (g.isnan() & ref.isnan()))
    if bool(bad.any()):
        at = int(torch.where(bad, off.nan_to_num(nan=1e300) / bound.nan_to_num(nan=1.0), -1.0).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst at {at}: {float(g.flatten()[at])} for "
                             f"{float(ref.flatten()[at])}, bound {float(bound.flatten()[at])}")
