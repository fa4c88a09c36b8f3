"""Plain float64 forms of oxidizr_amd.ops and bounds on what the kernels may be off, from arithmetic.

u(dtype) is half a step of a rounding relative to the value: finfo.eps / 2 (bf16 2^-8, fp32 2^-24).
A sum of n fp32 terms in any order is off by at most n 2^-24 times the sum of the terms'
magnitudes. Every bound below is the output's own rounding, plus fp32 sums over magnitudes, plus, for
bf16, the roundings of what a backward reads again, carried to the output by the derivative's size."""
import math

import torch

U32 = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def assert_close(got, ref, err, what):
    """|got - ref| <= err + u |ref| element by element (and nothing that is not finite)."""
    got64, bound = got.double(), err + u(got.dtype) * ref.abs()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert bool(torch.isfinite(got64).all()), f"{what}: not finite"
    # u |ref| covers the rounding of ref; that of a value err away is u err more
    over = (got64 - ref).abs() - bound * (1 + 2 * u(got.dtype)) - 1e-30
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3g} above the bound ({float(bound.max()):.3g} at most)"


# ---- sorting
def order(idx, E):
    """counts, offsets, perm, inv_perm of idx [T, k] by brute force."""
    T, k = idx.shape
    flat = [e if 0 <= e < E else E for e in idx.flatten().tolist()]
    perm = [i for e in range(E + 1) for i in range(T * k) if flat[i] == e] if T * k < 5000 else \
        sorted(range(T * k), key=lambda i: flat[i])
    counts = [0] * (E + 1)
    for e in flat:
        counts[e] += 1
    offsets = [0]
    for c in counts[:E]:
        offsets.append(offsets[-1] + c)
    inv = [0] * (T * k)
    for p, i in enumerate(perm):
        inv[i] = p

    def ints(v):
        return torch.tensor(v, dtype=torch.int32)
    return ints(counts[:E]), ints(offsets), ints(perm), ints(inv).view(T, k)


# ---- activations: value, slope, and a bound on the second derivative
def activation(z, act):
    if act == "none":
        return z, torch.ones_like(z), 0.0
    if act == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).to(z.dtype), 0.0
    if act == "silu":  # |silu''| <= 1/2
        g = torch.sigmoid(z)
        return z * g, g * (1 + z * (1 - g)), 0.5
    if act == "gelu":  # gelu'' = phi(z) (2 - z^2), at most 2 phi(0)
        cdf = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.8
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return (0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z),
            0.85)


# fp32 evaluation of an activation or its slope: exp and erf to a few steps at arguments up to
# z^2, so within 2^-20 (1 + |z|)
FN = 2.0 ** -20


def linear(x, w, b, offsets, act, res, dy, dtype):
    """{name: (reference, error bound)} of expert_linear and its gradients. Inputs are float64."""
    M, K = x.shape
    grouped = offsets is not None
    off = offsets.tolist() if grouped else [0, M]
    ws = w if grouped else w[None]
    N = ws.shape[1]
    y, ye, dx, dxe = (x.new_zeros(M, n) for n in (N, N, K, K))
    dw, dwe = torch.zeros_like(ws), torch.zeros_like(ws)
    db, dbe = x.new_zeros(len(ws), N), x.new_zeros(len(ws), N)
    ud = u(dtype)
    for e in range(len(ws)):
        r = slice(off[e], off[e + 1])
        xe, we = x[r], ws[e]
        n = xe.shape[0]
        z = xe @ we.t()
        zm = xe.abs() @ we.abs().t()
        if b is not None:
            be = b[e] if grouped else b
            z, zm = z + be, zm + be.abs()
        ze = (K + 1) * U32 * zm
        val, slope, second = activation(z, act)
        y[r], ye[r] = val, 1.2 * ze + FN * (1 + z.abs()) * (act != "none") * z.abs().clamp(max=1.0)
        if dy is None:
            continue
        g = dy[r]
        dz = g * slope
        # the slope: of the kept pre-activation (rounded to the dtype), evaluated in fp32; relu's may
        # differ only where z's sign is in doubt
        doubt = (z.abs() <= ze).to(z.dtype) if act == "relu" else 0.0
        se = second * (ze + ud * z.abs()) + FN * (1 + z.abs()) * (act not in ("none", "relu")) + doubt
        dze = g.abs() * se + U32 * dz.abs()
        db[e], dbe[e] = dz.sum(0), dze.sum(0) + (n + 8) * U32 * dz.abs().sum(0)
        if act != "none":
            dze = dze + ud * (dz.abs() + dze)  # dz is rounded to the dtype for the products
        dx[r], dxe[r] = dz @ we, dze @ we.abs() + N * U32 * ((dz.abs() + dze) @ we.abs())
        dw[e] = dz.t() @ xe
        dwe[e] = dze.t() @ xe.abs() + (n + 1) * U32 * ((dz.abs() + dze).t() @ xe.abs())
    if res is not None:
        y, ye = y + res, ye + U32 * (y.abs() + res.abs())
    out = {"y": (y, ye)}
    if dy is not None:
        out.update(dx=(dx, dxe), dw=(dw, dwe) if grouped else (dw[0], dwe[0]))
        if b is not None:
            out["db"] = (db, dbe) if grouped else (db[0], dbe[0])
        if res is not None:
            out["dr"] = (dy, torch.zeros_like(dy))
    return out


def norm(h, y, w2, gate, w3, scale, eps, d_out, d_n, dtype, hn_rounded=True):
    """{name: (reference, error bound)} of residual_norm and its gradients. Inputs are float64.
    hn_rounded: the backward may have read h_out in dtype."""
    T, H = h.shape
    c = (H + 32) * U32
    ud = u(dtype)
    out, oute = h, torch.zeros_like(h)
    if y is not None:
        r2 = torch.rsqrt(y.square().mean(1, keepdim=True) + eps) if w2 is not None else torch.ones_like(y[:, :1])
        yh = y * r2
        uu = yh * w2 if w2 is not None else yh
        g = gate if gate is not None else torch.ones_like(uu[:1, :1])
        out = scale * h + g * uu
        oute = c * ((scale * h).abs() + (g * uu).abs())
    ref = {}
    if y is not None:
        ref["h"] = (out, oute)
    if w3 is not None:
        r3 = torch.rsqrt(out.square().mean(1, keepdim=True) + eps)
        hh = out * r3
        ref["n"] = (hh * w3, (oute * r3 + hh.abs() * (c + (oute * r3).square().mean(1, keepdim=True).sqrt())) * w3.abs())
    if d_out is None and d_n is None:
        return ref
    D = d_out if d_out is not None else torch.zeros_like(h)
    De = U32 * D.abs()
    if d_n is not None:
        # h_out as the backward reads it again (without y the input itself)
        hhe = hh.abs() * (c + (ud if y is not None and hn_rounded else 0.0)) + oute * r3
        a = d_n * w3
        m = (hh * a).mean(1, keepdim=True)
        mm = (hh * a).abs().mean(1, keepdim=True)
        me = (hhe * a.abs()).mean(1, keepdim=True) + c * mm
        ref["dw3"] = ((d_n * hh).sum(0), (d_n.abs() * hhe).sum(0) + (T + 40) * U32 * (d_n * hh).abs().sum(0))
        D = D + r3 * (a - hh * m)
        De = De + r3 * (c * a.abs() + hh.abs() * me + hhe * (m.abs() + me)) + 8 * U32 * (
            D.abs() + r3 * (a.abs() + hh.abs() * mm))
    if y is None:
        ref["dh"] = (D, De)
        return ref
    ref["dh"] = (scale * D, abs(scale) * De + U32 * (scale * D).abs())
    yhe = c * yh.abs() if w2 is not None else torch.zeros_like(yh)
    if gate is not None:
        p = D * uu
        pe = De * uu.abs() + (D.abs() + De) * 2 * c * uu.abs()
        if gate.shape == (H,):
            ref["dgate"] = (p.sum(0), pe.sum(0) + (T + 40) * U32 * p.abs().sum(0))
        elif gate.shape == (T, 1):
            # formed from sums over dh' + r3 w3 dn and over hh: both magnitudes count
            big = D.abs()
            if d_n is not None:
                big = big + (d_out.abs() if d_out is not None else 0) + r3 * (a.abs() + hh.abs() * mm)
            ref["dgate"] = (p.sum(1, keepdim=True), pe.sum(1, keepdim=True) +
                            2 * c * (big * uu.abs()).sum(1, keepdim=True))
        else:
            ref["dgate"] = (p, pe)
    dg = D * g
    dge = De * g.abs() + U32 * dg.abs()
    if w2 is None:
        ref["dy"] = (dg, dge)
        return ref
    ref["dw2"] = ((dg * yh).sum(0), (dge * yh.abs() + (dg.abs() + dge) * yhe).sum(0) +
                  (T + 40) * U32 * (dg * yh).abs().sum(0))
    v, ve = dg * w2, dge * w2.abs() + U32 * (dg * w2).abs()
    m2 = (v * yh).mean(1, keepdim=True)
    big = (v * yh).abs()
    if d_n is not None:
        big = big + ((d_out.abs() if d_out is not None else 0) + r3 * (a.abs() + hh.abs() * mm)) * (g * w2 * yh).abs()
    m2e = (ve * yh.abs() + v.abs() * yhe).mean(1, keepdim=True) + 2 * c * big.mean(1, keepdim=True)
    ref["dy"] = (r2 * (v - yh * m2),
                 r2 * (ve + yh.abs() * m2e + yhe * (m2.abs() + m2e) + 2 * c * (v.abs() + yh.abs() * m2.abs())))
    return ref
