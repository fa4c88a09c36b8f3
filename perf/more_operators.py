"""Performance cases of the operators around a router and around experts that are held in 4 bits: the router's
losses and counts, microscaled 4-bit quantisation and back, and the experts' products over 4-bit weights.

A case is a dict of plain values:
  kind     "losses": router_losses, with the gradient of the logits in training
           "quant": quantize_mxfp4 and dequantize_mxfp4
           "mx": mx_linear over bf16 rows, with the gradients of rows, bias and residual in training
           "mxmx": quantize_mxfp4 of the rows, and mx_linear over both in 4 bits
  train    a forward and its backward; otherwise the forward alone
  dtype    "bf16" or "f32" of logits, or of what is quantised (products are bf16)
  T, E, k, pad           tokens, experts, experts per token, share of padding tokens (expert -1)
  seqs, score, tau       losses: sequences (0: one loss for all tokens), "softmax" or "sigmoid", temperature
  K, N, act, bias, res   mx: input and output widths, activation, whether it has a bias and a residual (E = 0:
                         one weight for all rows); quant: T rows of K

Four-bit elements are E2M1 numbers, 32 along the last dimension under one power of two (E8M0), as the
OCP microscaling formats define them. Inputs are made on the GPU from the seed alone: activations and upstream
gradients N(0, 1), as after a norm; weights N(0, 1 / K), quantised before the call, as a checkpoint holds
them; routing from noisy logits with uneven experts.
"""
import math

import torch

own = False

BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def losses(T, E, k, train, dtype="f32", score="softmax", seqs=0, pad=0.0, tau=1.0):
    return {"kind": "losses", "T": T, "E": E, "k": k, "train": train, "dtype": dtype, "score": score, "seqs": seqs,
            "pad": pad, "tau": tau}


def quant(T, K, dtype="bf16"):
    return {"kind": "quant", "T": T, "K": K, "dtype": dtype, "train": False}


def mx(T, k, E, K, N, train, act, bias=True, res=False, pad=0.0):
    return {"kind": "mx", "T": T, "k": k, "E": E, "K": K, "N": N, "train": train, "act": act, "bias": bias,
            "res": res, "pad": pad, "dtype": "bf16"}


def mxmx(T, k, E, K, N, act, bias=True, res=False, pad=0.0):
    return dict(mx(T, k, E, K, N, False, act, bias, res, pad), kind="mxmx")


def listed():
    named = {
        # a short batch's validation: losses and counts without gradients, launches and latency
        "losses_eval_512": losses(512, 16, 2, False),
        # the widest router in training, some tokens padding of a ragged batch
        "losses_train_8k": losses(8192, 256, 8, True, pad=0.06),
        # packed sequences with a loss each over normalised sigmoid scores, bf16 logits
        "losses_seqs_64k": losses(65536, 160, 6, True, dtype="bf16", score="sigmoid", seqs=48, pad=0.02),
        # a decoding batch's activations to 4 bits and back
        "quant_decode_64": quant(64, 4096),
        # the weights of some experts, as when a checkpoint is converted
        "quant_weights_f32": quant(16 * 1408, 2048, dtype="f32"),
        # one token through a layer's first experts: latency
        "mx_decode_1": mx(1, 2, 16, 2048, 1408, False, "silu"),
        # a serving batch over many experts, a few rows each: the stream of the weights that it touches
        "mx_decode_64": mx(64, 8, 128, 4096, 1536, False, "gelu"),
        # a prompt over frozen 4-bit experts
        "mx_prefill_16k": mx(8192, 2, 16, 2048, 1408, False, "silu"),
        # training through frozen 4-bit experts at odd sizes: gradients of the rows, the bias and the residual
        "mx_train_odd": mx(3999, 3, 12, 1376, 1368, True, "gelu_tanh", res=True, pad=0.05),
        # the serving batch with both sides in 4 bits
        "mxmx_decode_64": mxmx(64, 8, 128, 4096, 1536, "gelu"),
        # a long prompt with both sides in 4 bits
        "mxmx_prefill_64k": mxmx(8192, 8, 128, 4096, 1536, "silu"),
        # one weight for all rows, a residual added in the epilogue, odd sizes
        "mxmx_dense_odd": mxmx(1999, 1, 0, 2784, 2056, "none", res=True),
    }
    return [dict(c, name=n) for n, c in named.items()]


def draw(rng):
    """A case of the listed ones' ranges: sizes spread over their logarithm, odd ones among them."""
    def size(lo, hi, step=1):
        return max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step)

    while True:
        kind = rng.choice(("losses", "losses", "quant", "mx", "mx", "mx", "mxmx", "mxmx"))
        train = rng.random() < 0.6
        E = rng.choice((8, 12, 16, 24, 32, 64, 100, 128, 256))
        k = min(E, rng.choice((1, 2, 2, 3, 4, 6, 8)))
        pad = rng.choice((0.0, 0.0, 0.0, 0.03, 0.2))
        if kind == "losses":
            T = size(64, 65536)
            c = losses(T, E, k, train, rng.choice(("f32", "f32", "bf16")), rng.choice(("softmax", "softmax", "sigmoid")),
                       rng.choice((0, 0, 1, 3, max(1, T // 1500))), pad, rng.choice((1.0, 1.0, 0.7, 2.5)))
        elif kind == "quant":
            c = quant(size(1, 65536), size(384, 7168, BLOCK), rng.choice(("f32", "bf16")))
        else:
            T = size(256, 8192) if train and kind == "mx" else size(1, 8192)
            if rng.random() < 0.3:
                E, k, pad = 0, 1, 0.0
            K, N = size(384, 4096, rng.choice((32, 128))), size(512, 2816, rng.choice((8, 64)))
            act = rng.choice(("none", "silu", "gelu", "gelu_tanh"))
            bias, res = rng.random() < 0.7, rng.random() < 0.3
            c = mx(T, k, E, K, N, train, act, bias, res, pad) if kind == "mx" else mxmx(T, k, E, K, N, act, bias, res, pad)
        w = work(c)
        if w["bytes"] < 1.2e9 and w["flops"] < 8e11:
            return c


def work(case):
    kind, T, train = case["kind"], case["T"], case["train"]
    b = 4.0 if case["dtype"] == "f32" else 2.0
    four = 0.5 + 1.0 / BLOCK
    if kind == "quant":
        n = float(T) * case["K"]
        return {"bytes": 2 * n * (b + four), "flops": 4 * n}
    E, k = case["E"], case["k"]
    if kind == "losses":
        n = float(T) * E
        return {"bytes": n * b * (3 if train else 1) + 4.0 * T * k, "flops": (25.0 if train else 10.0) * n}
    K, N = case["K"], case["N"]
    kept = T * k * (1.0 - case["pad"])
    touched = E * (1.0 - (1.0 - k / E) ** T) if E else 1.0
    act, res = case["act"] != "none", int(case["res"])
    weights, n = four * touched * K * N, 2.0 * kept * N
    # bf16 rows are read by the product, or read, written and read in 4 bits
    total = kept * K * (2.0 if kind == "mx" else 2.0 + 2 * four) + weights + n * (1 + res)
    if train:
        # the pre-activation kept for the backward; then dy, w and it read, dx written
        total += n * (2 * int(act) + 1) + weights + 2.0 * kept * K
    return {"bytes": total, "flops": (4.0 if train else 2.0) * kept * K * N}


def routing(case, g):
    """Logits [T, E] fp32 of uneven experts, and the [T, k] int32 experts chosen; padding tokens have -1."""
    dev = g.device
    T, E, k = case["T"], case["E"], case["k"]
    logits = torch.randn(T, E, device=dev, generator=g) + 0.5 * torch.randn(E, device=dev, generator=g)
    idx = torch.topk(logits, k, dim=1).indices.to(torch.int32)
    if case["pad"]:
        idx[torch.rand(T, device=dev, generator=g) < case["pad"]] = -1
    return logits, idx


def offsets_of(idx, E):
    """[E + 1] int32 row offsets of the experts in rows sorted by expert."""
    flat = idx.flatten().long()
    counts = torch.bincount(flat[flat >= 0], minlength=E)
    return torch.cat((counts.new_zeros(1), torch.cumsum(counts, 0))).to(torch.int32)


# Four-bit numbers in elementary operations. float64 holds every product with a power of two and every
# border between two codes exactly.

def to_four(x):
    """Codes (0 .. 7, the sign apart) and exponents of x [..., K]: 32 elements' largest magnitude has exponent 2 (6 is
    the largest code), nearest code, ties to the even one, and what is above the largest becomes it."""
    v = x.unflatten(-1, (-1, BLOCK)).double()
    amax = v.abs().amax(-1, keepdim=True)
    exp = (torch.frexp(amax)[1] - 3).clamp(-127, 127)
    exp = torch.where(amax > 0, exp, -127)
    a = v.abs() * torch.exp2(-exp.double())
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return code, exp, v < 0


def packed(x):
    """(codes [..., K / 2], scales [..., K / 32]) uint8: element 2 i in the low half of byte i, the sign in
    bit 3; a scale is its exponent plus 127."""
    code, exp, neg = to_four(x)
    code = (code | (neg.to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (exp.squeeze(-1) + 127).to(torch.uint8)


def four_values(codes, scales, dtype=torch.float32):
    """What packed() made, as numbers."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=dtype, device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    s = torch.exp2(scales.to(dtype) - 127.0)
    return (grid[both.int()].unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)


def inputs(case, seed):
    """Every input tensor of a case, by name."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16

    def normal(*shape, std=1.0, dtype=dt):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, std, generator=g)

    kind, T, p = case["kind"], case["T"], {}
    if kind == "quant":
        p["x"] = normal(T, case["K"])
        return p
    if kind == "losses":
        logits, p["idx"] = routing(case, g)
        p["logits"] = logits.to(dt)
        S = case["seqs"]
        if S:
            cuts = torch.randint(0, T + 1, (S - 1,), device=dev, generator=g).sort().values
            p["offsets"] = torch.cat((cuts.new_zeros(1), cuts, cuts.new_full((1,), T))).to(torch.int32)
        if case["train"]:
            # the losses' coefficients, spread over the sequences
            shape = (S,) if S else ()
            p["d_balance"] = torch.full(shape, 0.01 / max(S, 1), device=dev)
            p["d_z"] = torch.full(shape, 0.001 / max(S, 1), device=dev)
        return p
    K, N, E, M = case["K"], case["N"], case["E"], T * case["k"]
    p["x"] = normal(M, K)
    parts = [packed(normal(N, K, std=K ** -0.5)) for _ in range(max(E, 1))]
    p["codes"], p["scales"] = (torch.stack([q[i] for q in parts]) if E else parts[0][i] for i in (0, 1))
    if case["bias"]:
        p["b"] = normal(*((E, N) if E else (N,)), std=0.1)
    if case["res"]:
        p["r"] = normal(M, N)
    if case["train"]:
        p["dy"] = normal(M, N)
    if E:
        p["offsets"] = offsets_of(routing(case, g)[1], E)
    return p


#: The tensors that a training pass returns gradients of.
LEAVES = {"losses": ("logits",), "mx": ("x", "b", "r")}


def prepare(case, seed):
    p = inputs(case, seed)
    s = {"case": case, "p": p}
    if "offsets" in p:
        # rows of the busiest expert, or of the longest sequence: the height of the plain form's batches
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
        return {"losses": plain_losses, "quant": plain_quant, "mx": plain_mx, "mxmx": plain_mx}[s["case"]["kind"]](s)


def run_own(s):
    from oxidizr_amd import ops
    c, p = s["case"], s["p"]
    if c["kind"] == "quant":
        return {"values": ops.dequantize_mxfp4(ops.quantize_mxfp4(p["x"]), dtype=p["x"].dtype)}
    if c["kind"] == "losses":
        out = ops.router_losses(p["logits"], p["idx"], score=c["score"], temperature=c["tau"], offsets=p.get("offsets"))
        r = {"balance": out.balance.detach(), "z": out.z.detach(), "counts": out.counts}
        if c["train"]:
            r.update(grads(s, (out.balance, out.z), (p["d_balance"], p["d_z"])))
        return r
    x = p["x"] if c["kind"] == "mx" else ops.quantize_mxfp4(p["x"])
    y = ops.mx_linear(x, ops.MxTensor(p["codes"], p["scales"]), p.get("b"), offsets=p.get("offsets"),
                      activation=c["act"], residual=p.get("r"))
    r = {"out": y.detach()}
    if c["train"]:
        r.update(grads(s, y, p["dy"]))
    return r


# The plain forms: elementary torch operations in fp32 (64-bit sums over tokens), rounded once at the end.

def sequences(case, p):
    """Which tokens count, the sequence of each, and how many sequences there are."""
    T, E, idx = case["T"], case["E"], p["idx"]
    real = ((idx >= 0) & (idx < E)).any(1)
    if not case["seqs"]:
        return real, torch.zeros(T, dtype=torch.long, device=idx.device), 1
    row = torch.arange(T, device=idx.device)
    return real, torch.searchsorted(p["offsets"][1:].long(), row, right=True), case["seqs"]


def plain_losses(s):
    c, p = s["case"], s["p"]
    T, E, k = c["T"], c["E"], c["k"]
    real, seq, S = sequences(c, p)
    x = p["logits"].float() / c["tau"]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    den = e.sum(1, keepdim=True)
    lse = (top + torch.log(den))[:, 0]
    soft = e / den
    if c["score"] == "softmax":
        q, curve = soft, None
    else:
        sig = 1.0 / (1.0 + torch.exp(-x))
        q, curve = sig / sig.sum(1, keepdim=True), 1.0 - sig

    def total(t):
        """Sums over each sequence's tokens, [S, ...], in a batch padded to the longest one."""
        if not c["seqs"]:
            return t.sum(0, keepdim=True)
        slot = seq * s["cap"] + torch.arange(T, device=t.device) - p["offsets"].long()[seq]
        return t.new_zeros(S * s["cap"], *t.shape[1:]).index_copy_(0, slot, t).view(S, s["cap"], *t.shape[1:]).sum(1)
    n = total(real.double())
    many = n.clamp(min=1.0)
    prob = total(torch.where(real[:, None], q, 0.0).double()) / many[:, None]
    z = total(torch.where(real, lse * lse, 0.0).double()) / many
    expert = torch.arange(E, device=x.device)
    counts = total(sum((p["idx"][:, j, None] == expert).to(torch.int32) for j in range(k)))
    f = counts.double() / (k * many[:, None])
    balance = E * (f * prob + prob * prob).sum(1)
    shape = (S,) if c["seqs"] else ()
    r = {"balance": balance.float().view(shape), "z": z.float().view(shape),
         "counts": counts.to(torch.int32).view(shape + (E,))}
    if c["train"]:
        g = p["d_balance"].double().view(S, 1) * E * (f + 2.0 * prob) / many[:, None]
        g = g.float()[seq]
        d = q * (g - (q * g).sum(1, keepdim=True))
        if curve is not None:
            d = d * curve
        dz = (p["d_z"].double().view(S) * 2.0 / many).float()[seq]
        d = (d + (dz * lse)[:, None] * soft) / c["tau"]
        r["d_logits"] = torch.where(real[:, None], d, 0.0).to(p["logits"].dtype)
    return r


def plain_quant(s):
    x = s["p"]["x"]
    code, exp, neg = to_four(x)
    a = torch.tensor(GRID, device=x.device)[code.int()] * torch.exp2(exp.float())
    return {"values": torch.where(neg, -a, a).flatten(-2).to(x.dtype)}


def activate(z, act):
    """The activation of z and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "silu":
        g = 1.0 / (1.0 + torch.exp(-z))
        return z * g, g * (1.0 + z * (1.0 - g))
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)


def plain_mx(s):
    c, p = s["case"], s["p"]
    x = p["x"].float() if c["kind"] == "mx" else four_values(*packed(p["x"]))
    w, dt = four_values(p["codes"], p["scales"]), p["x"].dtype
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
        z = torch.bmm(batched(x), w.transpose(1, 2).contiguous())
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
            r["d_x"], db = rows(torch.bmm(dz, w)).to(dt), dz.sum(1)
        else:
            dz = dy * slope
            r["d_x"], db = (dz @ w).to(dt), dz.sum(0)
        if "b" in p:
            r["d_b"] = db.to(dt)
        if "r" in p:
            r["d_r"] = p["dy"]
    return r


def nearest_four(x):
    """float64 values of x in 4 bits, from the format's definition: the nearest of all numbers that a block can
    hold, among two as near the one whose last mantissa bit is zero."""
    v = x.double().unflatten(-1, (-1, BLOCK))
    amax = v.abs().amax(-1, keepdim=True)
    s = torch.exp2(torch.floor(torch.log2(amax.clamp(min=2.0 ** -140))) - 2.0).clamp(min=2.0 ** -127)
    # log2 may round up to a whole number just below a power of two
    s = torch.where(s * 4.0 > amax, (s / 2.0).clamp(min=2.0 ** -127), s)
    best, gap = torch.zeros_like(v), (v / s).abs()
    for i, m in enumerate(GRID[1:], 1):
        d = ((v / s).abs() - m).abs()
        closer = (d < gap) | ((d == gap) & (i % 2 == 0))
        best, gap = torch.where(closer, m, best), torch.where(closer, d, gap)
    return (best * s * torch.sign(v)).flatten(-2)


def exact(case, seed):
    """What run() returns, in float64 from the same inputs: gradients by torch's autograd of the definition, sequences
    and experts one after another."""
    p = inputs(case, seed)
    kind, train = case["kind"], case["train"]
    if kind == "quant":
        return {"values": torch.cat([nearest_four(t) for t in p["x"].split(4096)])}
    if kind == "losses":
        T, E, k = case["T"], case["E"], case["k"]
        x = p["logits"].double().requires_grad_(train)
        bounds = p["offsets"].tolist() if case["seqs"] else [0, T]
        balance, z, counts = [], [], []
        for a, b in zip(bounds[:-1], bounds[1:]):
            idx = p["idx"][a:b].long()
            here = (idx >= 0).any(1)
            one = torch.bincount(idx[idx >= 0], minlength=E)
            counts.append(one.to(torch.int32))
            n = int(here.sum())
            l = x[a:b][here] / case["tau"]
            if n == 0:
                balance.append(l.sum() * 0.0)
                z.append(l.sum() * 0.0)
                continue
            q = torch.softmax(l, 1) if case["score"] == "softmax" else torch.sigmoid(l) / torch.sigmoid(l).sum(1, keepdim=True)
            prob = q.mean(0)
            balance.append(E * (one.double() / (k * n) * prob).sum() + E * prob.square().sum())
            z.append(torch.logsumexp(l, 1).square().mean())
        pick = torch.stack if case["seqs"] else (lambda t: t[0])
        r = {"balance": pick(balance), "z": pick(z), "counts": pick(counts)}
        if train:
            r["d_logits"], = torch.autograd.grad((r["balance"], r["z"]), x, (p["d_balance"].double(), p["d_z"].double()))
        return {n: t.detach() for n, t in r.items()}
    M, E, N = case["T"] * case["k"], case["E"], case["N"]
    # one expert after another, whose weights alone are held in 64 bits
    off = p["offsets"].tolist() if E else [0, M]
    out = torch.zeros(M, N, dtype=torch.float64, device=p["x"].device)
    d_x, d_b = (torch.zeros(M, case["K"], dtype=torch.float64, device=out.device),
                torch.zeros(max(E, 1), N, dtype=torch.float64, device=out.device)) if train else (None, None)
    for i in range(max(E, 1)):
        a, b = off[i], off[i + 1]
        if a == b:
            continue
        x = p["x"][a:b].double() if kind == "mx" else nearest_four(p["x"][a:b])
        codes, scales = (p[n][i] if E else p[n] for n in ("codes", "scales"))
        w = four_values(codes, scales, torch.float64)
        x.requires_grad_(train)
        bias = (p["b"][i] if E else p["b"]).double().requires_grad_(train) if "b" in p else None
        zz = x @ w.t()
        y = activate(zz if bias is None else zz + bias, case["act"])[0]
        out[a:b] = y.detach()
        if train:
            got = torch.autograd.grad(y, [x] if bias is None else [x, bias], p["dy"][a:b].double())
            d_x[a:b] = got[0]
            if bias is not None:
                d_b[i] = got[1]
    r = {"out": out + p["r"].double() if "r" in p else out}
    if train:
        r["d_x"] = d_x
        if "b" in p:
            r["d_b"] = d_b if E else d_b[0]
        if "r" in p:
            r["d_r"] = p["dy"].double()
    return r
