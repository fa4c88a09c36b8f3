"""Performance cases of the operators around the experts: tokens sorted by expert and back, the experts'
products with bias, activation and residual, and the norms before and after a block.

A case is a dict of plain values:
  kind     "dispatch": sort_tokens and permute_tokens, with a gradient of x in training
           "combine": unpermute_tokens with weights, with the gradients of the rows and the weights
           "linear": expert_linear over rows sorted by expert, or over all rows with one weight (E = 0)
           "norm": residual_norm, with the gradients of everything that it reads
  train    a forward and its backward; otherwise the forward alone
  dtype    "bf16" or "f32" of activations, weights and gradients (combine weights are fp32)
  T, H, E, k, pad        tokens, hidden size, experts, experts per token, share of padding tokens (expert -1)
  K, N, act, bias, res   linear: input and output widths, activation, whether it has a bias and a residual
  gate, post, next       norm: "none", "channel" [H], "token" [T, 1] or "full" [T, H]; which norms it has

Inputs are made on the GPU from the seed alone: activations and upstream gradients N(0, 1), as after a
norm; weights N(0, 1 / K); routing from noisy logits with uneven experts.
"""
import math

import torch

own = False

EPS = 1e-6


def dispatch(T, H, E, k, train, dtype="bf16", pad=0.0):
    return {"kind": "dispatch", "T": T, "H": H, "E": E, "k": k, "train": train, "dtype": dtype, "pad": pad}


def combine(T, H, E, k, train, dtype="bf16", pad=0.0):
    return dict(dispatch(T, H, E, k, train, dtype, pad), kind="combine")


def linear(T, k, E, K, N, train, act, dtype="bf16", bias=True, res=False, pad=0.0):
    return {"kind": "linear", "T": T, "k": k, "E": E, "K": K, "N": N, "train": train, "act": act,
            "dtype": dtype, "bias": bias, "res": res, "pad": pad}


def norm(T, H, train, gate, dtype="bf16", post=True, next=True, scale=1.0):
    return {"kind": "norm", "T": T, "H": H, "train": train, "gate": gate, "dtype": dtype, "post": post,
            "next": next, "scale": scale}


def listed():
    named = {
        # a serving batch's tokens sorted and copied to their experts: launches and latency
        "dispatch_decode_64": dispatch(64, 4096, 128, 8, False),
        # the widest training layer's tokens, some of them padding of a ragged batch, and their gradient
        "dispatch_train_8k": dispatch(8192, 7168, 256, 8, True, pad=0.06),
        # fp32 at odd sizes
        "dispatch_f32_odd": dispatch(1999, 776, 12, 3, True, dtype="f32", pad=0.1),
        # a few sequences decoding: the experts' rows added up with their weights
        "combine_decode_16": combine(16, 2048, 16, 2, False),
        # a long training batch, the gradients of the rows and of the weights
        "combine_train_16k": combine(16384, 2048, 64, 6, True),
        # a serving batch over many experts, a few rows each: the stream of the weights that it touches
        "linear_decode_64": linear(64, 8, 128, 4096, 1536, False, "gelu"),
        # the first half of biased experts in training
        "linear_train_16k": linear(8192, 2, 16, 2048, 1408, True, "silu"),
        # one weight for all tokens with the residual added in the epilogue: a dense layer's last product
        "linear_dense_8k": linear(8192, 1, 0, 2816, 2048, True, "none", res=True),
        # fp32 at odd sizes, padding rows behind the last expert's
        "linear_f32_odd": linear(1999, 3, 12, 776, 1368, True, "relu", dtype="f32", pad=0.05),
        # one token between two blocks: latency
        "norm_decode_1": norm(1, 2048, False, "channel"),
        # the widest hidden size in training: norm, gate, residual and the next block's norm in one pass
        "norm_train_8k": norm(8192, 7168, True, "channel"),
        # fp32 at odd sizes, one gate to a token, a scaled residual
        "norm_f32_odd": norm(1999, 776, True, "token", dtype="f32", scale=0.8125),
    }
    return [dict(c, name=n) for n, c in named.items()]


def draw(rng):
    """A case of the listed ones' ranges: sizes spread over their logarithm, odd ones among them."""
    def size(lo, hi, step=1):
        return max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step)

    while True:
        kind = rng.choice(("dispatch", "combine", "linear", "linear", "norm", "norm"))
        train = rng.random() < 0.6
        dtype = "f32" if rng.random() < 0.3 else "bf16"
        T = size(256, 16384) if train else size(1, 8192)
        H = size(384, 7168, rng.choice((8, 128)))
        E = rng.choice((8, 12, 16, 24, 32, 64, 100, 128, 256))
        k = min(E, rng.choice((1, 2, 2, 3, 4, 6, 8)))
        pad = rng.choice((0.0, 0.0, 0.0, 0.03, 0.2))
        if kind == "norm":
            post, next = rng.choice(((True, True), (True, True), (True, False), (False, True)))
            c = norm(T, H, train, rng.choice(("none", "channel", "channel", "token", "full")), dtype, post,
                     next, rng.choice((1.0, 1.0, 0.5, 1.75)))
        elif kind == "linear":
            if rng.random() < 0.3:
                E, k, pad = 0, 1, 0.0
            N = size(512, 2816, rng.choice((8, 64)))
            K, N = rng.choice(((H, N), (N, H)))
            c = linear(T, k, E, K, N, train, rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")), dtype,
                       rng.random() < 0.7, rng.random() < 0.3, pad)
        else:
            c = (dispatch if kind == "dispatch" else combine)(T, H, E, k, train, dtype, pad)
        w = work(c)
        # within the largest listed case's work (fp32 products run at 1/16 of the bf16 rate)
        most = 3.6e10 if dtype == "f32" else 2.8e11
        if w["bytes"] < 2e9 and (kind != "linear" or w["flops"] < most):
            return c


def work(case):
    b = 4.0 if case["dtype"] == "f32" else 2.0
    T, train = case["T"], case["train"]
    if case["kind"] == "norm":
        H = case["H"]
        full = 1 if case["gate"] == "full" else 0
        read, wrote = 2 + full, 1 + int(case["next"])
        if train:
            # backward: both upstream gradients, the new residual (for the next norm), the rows, the gate
            read += 2 + 2 * int(case["next"]) + full
            wrote += 2 + full
        return {"bytes": b * T * H * (read + wrote), "flops": (30.0 if train else 10.0) * T * H}
    k = case["k"]
    kept = T * k * (1.0 - case["pad"])
    if case["kind"] == "linear":
        K, N, E = case["K"], case["N"], case["E"]
        touched = E * (1.0 - (1.0 - k / E) ** T) if E else 1.0
        act, res = case["act"] != "none", int(case["res"])
        weights = b * touched * K * N
        n = b * kept * N
        total = b * kept * K + weights + n * (1 + res)
        if train:
            # the pre-activation kept for the backward; then dy, x, w and it read, dx and dw written
            total += n * (2 * int(act) + 1) + 2 * b * kept * K + weights + b * max(E, 1) * K * N
        return {"bytes": total, "flops": (6.0 if train else 2.0) * kept * K * N}
    H = case["H"]
    x, rows = b * T * H, b * kept * H
    if case["kind"] == "dispatch":
        return {"bytes": (x + rows) * (2 if train else 1) + 12.0 * T * k, "flops": (kept * H if train else 0.0)}
    back = x + 2 * rows + 4.0 * T * k
    return {"bytes": x + rows + 8.0 * T * k + (back if train else 0.0),
            "flops": (5.0 if train else 2.0) * kept * H}


def routing(case, g):
    """[T, k] int32 experts of noisy logits over uneven experts; padding tokens have -1."""
    dev = g.device
    T, E, k = case["T"], case["E"], case["k"]
    logits = torch.randn(T, E, device=dev, generator=g) + 0.5 * torch.randn(E, device=dev, generator=g)
    top, idx = torch.topk(logits, k, dim=1)
    idx = idx.to(torch.int32)
    if case["pad"]:
        idx[torch.rand(T, device=dev, generator=g) < case["pad"]] = -1
    return idx, torch.softmax(top, 1)


def order_of(idx, E):
    """counts, offsets, perm, inv_perm of a stable sort by expert; what has no expert comes last."""
    flat = idx.flatten().long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    perm = torch.argsort(key, stable=True)
    inv = torch.empty_like(perm).scatter_(0, perm, torch.arange(perm.numel(), device=perm.device))
    counts = torch.zeros(E + 1, dtype=torch.int64, device=perm.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cumsum(counts, 0) - counts
    return tuple(t.to(torch.int32) for t in (counts[:E], offsets, perm, inv.view(idx.shape)))


def inputs(case, seed):
    """Every input tensor of a case, by name."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, dtype=dt, device=dev).normal_(mean, std, generator=g)

    T, train, p = case["T"], case["train"], {}
    if case["kind"] == "norm":
        H = case["H"]
        p["h"], p["y"] = normal(T, H, std=2.0), normal(T, H)
        if case["post"]:
            p["post_w"] = normal(H, std=0.1, mean=1.0)
        shape = {"channel": (H,), "token": (T, 1), "full": (T, H)}.get(case["gate"])
        if shape:
            p["gate"] = torch.rand(shape, device=dev, generator=g).to(dt)
        if case["next"]:
            p["next_w"] = normal(H, std=0.1, mean=1.0)
        if train:
            p["dh"] = normal(T, H)
            if case["next"]:
                p["dn"] = normal(T, H)
        return p
    if case["kind"] == "linear":
        K, N, E, M = case["K"], case["N"], case["E"], case["T"] * case["k"]
        p["x"] = normal(M, K)
        p["w"] = normal(*((E, N, K) if E else (N, K)), std=K ** -0.5)
        if case["bias"]:
            p["b"] = normal(*((E, N) if E else (N,)), std=0.1)
        if case["res"]:
            p["r"] = normal(M, N)
        if train:
            p["dy"] = normal(M, N)
        if E:
            p["offsets"] = order_of(routing(case, g)[0], E)[1]
        return p
    T, H, E, k = (case[n] for n in "THEk")
    p["idx"], p["w"] = routing(case, g)
    if case["kind"] == "dispatch":
        p["x"] = normal(T, H)
        if train:
            p["dxp"] = normal(T * k, H)
    else:
        p["y"] = normal(T * k, H)
        if train:
            p["dout"] = normal(T, H)
    return p


#: The tensors that a training pass returns gradients of.
LEAVES = {"dispatch": ("x",), "combine": ("y", "w"), "linear": ("x", "w", "b", "r"),
          "norm": ("h", "y", "post_w", "gate", "next_w")}


def prepare(case, seed):
    p = inputs(case, seed)
    s = {"case": case, "p": p}
    if case["kind"] == "combine":
        s["order"] = order_of(p["idx"], case["E"])
    if case["kind"] == "linear" and case["E"]:
        # rows of the busiest expert: the height of the plain form's batched products
        s["cap"] = max(1, int((p["offsets"][1:] - p["offsets"][:-1]).max()))
    if case["train"]:
        s["leaves"] = [n for n in LEAVES[case["kind"]] if n in p]
        for n in s["leaves"]:
            p[n].requires_grad_()
    return s


def grads(s, outputs, upstream):
    """Gradients of a training pass by name, through the framework's autograd nodes."""
    got = torch.autograd.grad(outputs, [s["p"][n] for n in s["leaves"]], upstream)
    return {"d_" + n: t for n, t in zip(s["leaves"], got)}


def run(s):
    if own:
        return run_own(s)
    with torch.no_grad():
        return {"dispatch": plain_dispatch, "combine": plain_combine, "linear": plain_linear,
                "norm": plain_norm}[s["case"]["kind"]](s)


def run_own(s):
    from oxidizr_amd import ops
    c, p = s["case"], s["p"]
    if c["kind"] == "dispatch":
        order = ops.sort_tokens(p["idx"], c["E"])
        out = ops.permute_tokens(p["x"], order)
        r = {"counts": order.counts, "offsets": order.offsets, "perm": order.perm, "inv_perm": order.inv_perm}
        up = p.get("dxp")
    elif c["kind"] == "combine":
        out, r, up = ops.unpermute_tokens(p["y"], ops.TokenOrder(*s["order"]), p["w"]), {}, p.get("dout")
    elif c["kind"] == "linear":
        out = ops.expert_linear(p["x"], p["w"], p.get("b"), offsets=p.get("offsets"), activation=c["act"],
                                residual=p.get("r"))
        r, up = {}, p.get("dy")
    else:
        out = ops.residual_norm(p["h"], p["y"], p.get("post_w"), gate=p.get("gate"), next_weight=p.get("next_w"),
                                residual_scale=c["scale"], eps=EPS)
        r = {}
        if c["next"]:
            h, n = out
            r = {"h": h.detach(), "n": n.detach()}
            return dict(r, **grads(s, (h, n), (p["dh"], p["dn"]))) if c["train"] else r
        up = p.get("dh")
    r["out"] = out.detach()
    if c["train"]:
        r.update(grads(s, out, up))
    return r


# The plain forms: elementary torch operations in fp32, rounded once at the end.

def plain_dispatch(s):
    c, p = s["case"], s["p"]
    T, k = c["T"], c["k"]
    counts, offsets, perm, inv = order_of(p["idx"], c["E"])
    kept = torch.arange(T * k, device=perm.device) < offsets[-1]
    xp = torch.where(kept[:, None], p["x"][(perm // k).long()], 0.0)
    r = {"counts": counts, "offsets": offsets, "perm": perm, "inv_perm": inv, "out": xp}
    if c["train"]:
        d = torch.where(kept[:, None], p["dxp"].float(), 0.0)[inv.flatten().long()]
        r["d_x"] = d.view(T, k, -1).sum(1).to(p["x"].dtype)
    return r


def plain_combine(s):
    c, p = s["case"], s["p"]
    T, k = c["T"], c["k"]
    counts, offsets, perm, inv = s["order"]
    at = inv.flatten().long()
    kept = (at < offsets[-1]).view(T, k)
    y = p["y"].float()[at].view(T, k, -1)
    y = torch.where(kept[..., None], y, 0.0)
    r = {"out": (p["w"][..., None] * y).sum(1).to(p["y"].dtype)}
    if c["train"]:
        d = p["dout"].float()[:, None, :]
        r["d_w"] = (d * y).sum(2)
        dy = torch.where(kept, p["w"], 0.0)[..., None] * d
        r["d_y"] = dy.view(T * k, -1)[perm.long()].to(p["y"].dtype)
    return r


def activate(z, act):
    """The activation of z and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0.0), (z > 0).to(z.dtype)
    if act == "silu":
        g = 1.0 / (1.0 + torch.exp(-z))
        return z * g, g * (1.0 + z * (1.0 - g))
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)


def plain_linear(s):
    c, p = s["case"], s["p"]
    x, w, dt = p["x"].float(), p["w"].float(), p["x"].dtype
    E, M = c["E"], x.shape[0]
    if E:
        # rows of each expert in a batch of their own, padded to the busiest expert's
        off, cap = p["offsets"].long(), s["cap"]
        row = torch.arange(M, device=x.device)
        e = torch.searchsorted(off[1:], row, right=True).clamp(max=E - 1)
        kept = (row < off[-1])[:, None]
        slot = torch.where(kept[:, 0], e * cap + row - off[e], E * cap)

        def batched(t):
            return t.new_zeros(E * cap + 1, t.shape[1]).index_copy_(0, slot, t)[:E * cap].view(E, cap, -1)

        def rows(t):
            return torch.where(kept, t.reshape(E * cap, -1)[slot.clamp(max=E * cap - 1)], 0.0)
        xb = batched(x)
        z = torch.bmm(xb, w.transpose(1, 2).contiguous())
        if "b" in p:
            z = z + p["b"].float()[:, None, :]
    else:
        z = x @ w.t()
        if "b" in p:
            z = z + p["b"].float()
    y, slope = activate(z, c["act"])
    out = rows(y) if E else y
    r = {"out": (out + p["r"].float() if "r" in p else out).to(dt)}
    if c["train"]:
        dy = p["dy"].float()
        if E:
            dz = batched(torch.where(kept, dy, 0.0)) * slope
            r["d_x"] = rows(torch.bmm(dz, w)).to(dt)
            r["d_w"] = torch.bmm(dz.transpose(1, 2).contiguous(), xb).to(dt)
            db = dz.sum(1)
        else:
            dz = dy * slope
            r["d_x"], r["d_w"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
            db = dz.sum(0)
        if "b" in p:
            r["d_b"] = db.to(dt)
        if "r" in p:
            r["d_r"] = p["dy"]
    return r


def plain_norm(s):
    c, p = s["case"], s["p"]
    dt = p["h"].dtype
    f = {n: t.float() for n, t in p.items()}
    h, y = f["h"], f["y"]
    if c["post"]:
        r2 = torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
        yh = y * r2
        u = yh * f["post_w"]
    else:
        u = y
    g = f.get("gate")
    new = c["scale"] * h + (u if g is None else g * u)
    r = {"h" if c["next"] else "out": new.to(dt)}
    if c["next"]:
        r3 = torch.rsqrt((new * new).mean(1, keepdim=True) + EPS)
        r["n"] = (new * r3 * f["next_w"]).to(dt)
    if not c["train"]:
        return r
    d = f["dh"]
    if c["next"]:
        hh, dn = new * r3, f["dn"] * f["next_w"]
        d = d + r3 * (dn - hh * (dn * hh).mean(1, keepdim=True))
        r["d_next_w"] = (f["dn"] * hh).sum(0).to(dt)
    r["d_h"] = (c["scale"] * d).to(dt)
    if g is not None:
        du = d * u
        r["d_gate"] = {"channel": lambda: du.sum(0), "token": lambda: du.sum(1, keepdim=True),
                       "full": lambda: du}[c["gate"]]().to(dt)
        d = d * g
    if c["post"]:
        r["d_post_w"] = (d * yh).sum(0).to(dt)
        d = d * f["post_w"]
        d = r2 * (d - yh * (d * yh).mean(1, keepdim=True))
    r["d_y"] = d.to(dt)
    return r


def exact(case, seed):
    """What run() returns, in float64 from the same inputs: gradients by torch's autograd of the definition,
    experts one after another."""
    p = inputs(case, seed)
    kind, train = case["kind"], case["train"]
    q = {n: t.double() if t.is_floating_point() else t for n, t in p.items()}
    names = [n for n in LEAVES[kind] if n in q] if train else []
    for n in names:
        q[n].requires_grad_()
    r, up = {}, None
    if kind in ("dispatch", "combine"):
        T, E, k = case["T"], case["E"], case["k"]
        e = p["idx"].flatten().cpu().tolist()
        perm = sorted(range(T * k), key=lambda i: e[i] if 0 <= e[i] < E else E)
        rows = sum(1 for v in e if 0 <= v < E)
        dev = p["idx"].device
        perm = torch.tensor(perm, device=dev)
        kept = perm[:rows]
        if kind == "dispatch":
            counts = [0] * E
            for v in e:
                if 0 <= v < E:
                    counts[v] += 1
            offsets = [0]
            for n in counts:
                offsets.append(offsets[-1] + n)
            inv = torch.empty_like(perm)
            inv[perm] = torch.arange(T * k, device=dev)
            r = {"counts": torch.tensor(counts, dtype=torch.int32),
                 "offsets": torch.tensor(offsets, dtype=torch.int32), "perm": perm.int(),
                 "inv_perm": inv.view(T, k).int()}
            out = torch.cat((q["x"][kept // k], q["x"].new_zeros(T * k - rows, case["H"])))
            up = q.get("dxp")
        else:
            out = torch.zeros(T, case["H"], dtype=torch.float64, device=dev)
            out = out.index_add(0, kept // k, q["w"].flatten()[kept, None] * q["y"][:rows])
            up = q.get("dout")
    elif kind == "linear":
        M, E = case["T"] * case["k"], case["E"]
        off = p["offsets"].tolist() if E else [0, M]
        parts = []
        for i in range(max(E, 1)):
            w = q["w"][i] if E else q["w"]
            z = q["x"][off[i]:off[i + 1]] @ w.t()
            if "b" in q:
                z = z + (q["b"][i] if E else q["b"])
            parts.append(activate(z, case["act"])[0])
        parts.append(q["x"].new_zeros(M - off[-1], case["N"]))
        out = torch.cat(parts)
        if "r" in q:
            out = out + q["r"]
        up = q.get("dy")
    else:
        def rms(t, w):
            return t / torch.sqrt(t.square().mean(1, keepdim=True) + EPS) * w
        u = rms(q["y"], q["post_w"]) if case["post"] else q["y"]
        out = case["scale"] * q["h"] + q.get("gate", 1.0) * u
        up = q.get("dh")
        if case["next"]:
            n = rms(out, q["next_w"])
            r = {"h": out.detach(), "n": n.detach()}
            if train:
                got = torch.autograd.grad((out, n), [q[m] for m in names], (q["dh"], q["dn"]))
                r.update({"d_" + m: t for m, t in zip(names, got)})
            return r
    r["out"] = out.detach()
    if train:
        got = torch.autograd.grad(out, [q[m] for m in names], up)
        r.update({"d_" + m: t for m, t in zip(names, got)})
    return r
