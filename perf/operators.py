"""Measured cases of the token-sequence operators: scaled embedding lookup with its gradient by sorted tokens, short causal
convolution, selective state space scan (sequences, training and single tokens) and global gradient-norm clipping.

Sequences are time-major ([steps, batch, channels]) as everywhere in this framework; fp32 cases come from its protein
views (128 pairs a batch, 9048 words + padding, 22-wide embeddings, 512-wide latent, up to 232 or 1024 segments), 16-bit
cases are generic language-model shapes.
"""
import math
import random

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # ---- embedding
        # one step of a decoder over 16 running sequences: launch latency
        dict(name="embedding decode", op="embedding", train=False, n=16, vocab=32000, d=1024, dtype="bf16", pad=False),
        # the word ids of a Davis-shaped batch: 128 proteins x 85 segments x 11 words, rows of 22 floats, 9048 = padding
        dict(name="embedding protein words", op="embedding", train=True, n=119680, vocab=9049, d=22, dtype="fp32", pad=True),
        # a language-model training batch: 64 k tokens with natural (Zipf) frequencies over a large vocabulary
        dict(name="embedding long batch", op="embedding", train=True, n=65536, vocab=131072, d=2048, dtype="bf16", pad=False),
        # ---- short causal convolution
        # single tokens of 64 running sequences
        dict(name="conv step", op="conv_step", batch=64, d=2048, width=4, dtype="bf16"),
        # protein segments of one batch (ragged lengths), training in fp32
        dict(name="conv protein train", op="conv", train=True, t=232, batch=128, d=512, width=4, dtype="fp32", ragged=True),
        # a batch of long prompts
        dict(name="conv prompt", op="conv", train=False, t=8192, batch=4, d=4096, width=4, dtype="bf16", ragged=False),
        # ---- selective scan
        # single tokens of 4 running sequences: latency
        dict(name="scan step few", op="scan_step", batch=4, d=2048, state=16, groups=1, dtype="bf16"),
        # protein segments of one batch (ragged lengths), training in fp32
        dict(name="scan protein train", op="scan", train=True, t=232, batch=128, d=512, state=16, groups=1, dtype="fp32",
             ragged=True),
        # one long prompt: few channels, many steps, so the time axis has to be split
        dict(name="scan long prompt", op="scan", train=False, t=16384, batch=1, d=4096, state=16, groups=1, dtype="bf16",
             ragged=False),
        # training on 2048-token sequences
        dict(name="scan long train", op="scan", train=True, t=2048, batch=8, d=2048, state=16, groups=1, dtype="bf16",
             ragged=False),
        # ---- gradient norm and clipping
        # the parameters of this framework's joint model (a few dozen tensors, 4 M floats)
        dict(name="clip joint model", op="clip", tensors=48, total=4000000, dtype="fp32"),
        # a few hundred tensors of a 400 M parameter model with bf16 gradients
        dict(name="clip large model", op="clip", tensors=290, total=400000000, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _types(rng):
    return rng.choice(["fp32", "bf16", "bf16", "fp16"])


def draw(rng):
    op = rng.choice(["embedding", "conv", "conv_step", "scan", "scan", "scan_step", "clip"])
    dtype = _types(rng)
    if op == "embedding":
        d = rng.choice([_log(rng, 8, 2048), 8 * _log(rng, 2, 256)])
        n = min(_log(rng, 1, 131072), 134217728 // d)
        return dict(op=op, train=rng.random() < 0.7, n=n, vocab=min(_log(rng, 500, 131072), 268435456 // d), d=d, dtype=dtype,
                    pad=rng.random() < 0.5)
    if op == "clip":
        return dict(op=op, tensors=_log(rng, 1, 400), total=_log(rng, 2000, 200000000), dtype=dtype)
    d = rng.choice([_log(rng, 20, 4096), 64 * _log(rng, 1, 64)])
    if op == "conv_step":
        return dict(op=op, batch=_log(rng, 1, 512), d=d, width=rng.randint(2, 8), dtype=dtype)
    if op == "scan_step":
        groups = rng.choice([1, 1, 2]) if d % 2 == 0 else 1
        return dict(op=op, batch=_log(rng, 1, 512), d=d, state=rng.choice([4, 8, 11, 16, 16, 16, 32]), groups=groups, dtype=dtype)
    t = _log(rng, 1, 16384)
    ragged = rng.random() < 0.5
    if op == "conv":
        batch = max(1, min(_log(rng, 1, 128), 134217728 // (t * d)))
        return dict(op=op, train=rng.random() < 0.5, t=t, batch=batch, d=d, width=rng.randint(2, 8), dtype=dtype, ragged=ragged)
    groups = rng.choice([1, 1, 2]) if d % 2 == 0 else 1
    state = rng.choice([4, 8, 11, 16, 16, 16, 32])
    d = min(d, max(20, 536870912 // (t * state)) // 2 * 2)
    batch = max(1, min(_log(rng, 1, 128), 536870912 // (t * d * state)))
    return dict(op=op, train=rng.random() < 0.6, t=t, batch=batch, d=d, state=state, groups=groups, dtype=dtype, ragged=ragged)


# ------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    return g


def _lengths(case, g):
    """Ragged lengths over the whole range, the longest of them the full length."""
    if not case["ragged"]:
        return None
    t, b = case["t"], case["batch"]
    n = (torch.rand(b, device=_DEV, generator=g) * t).long() + 1
    n = n.clamp(1, t)
    n[int(torch.randint(b, (1,), device=_DEV, generator=g))] = t
    return n.to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    dt = _TYPES[case["dtype"]]
    op = case["op"]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device=_DEV, generator=g) * scale).to(dtype)

    s = dict(case=case)
    if op == "embedding":
        n, v, d = case["n"], case["vocab"], case["d"]
        s["weight"] = normal(v, d, scale=d ** -0.5)
        if case["pad"]:                                   # uniform words, one row in six behind a sequence's end
            idx = torch.randint(v - 1, (n,), device=_DEV, generator=g)
            idx[torch.rand(n, device=_DEV, generator=g) < 1.0 / 6] = v - 1
        else:                                             # p(rank) ~ 1 / rank
            idx = torch.exp(torch.rand(n, device=_DEV, generator=g, dtype=torch.float64) * math.log(v)).long() - 1
            idx = idx.clamp(0, v - 1)
        s["idx"], s["pad"], s["scale"] = idx, (v - 1 if case["pad"] else None), math.sqrt(d)
        if case["train"]:
            s["weight"].requires_grad_(True)
            s["dout"] = normal(n, d, scale=1e-2)
        return s
    if op == "clip":
        k, total = case["tensors"], case["total"]
        sized = random.Random(k * 1000003 + total)        # the sizes are the model's, the same whatever the gradients
        part = [sized.random() ** 3 + 1e-4 for _ in range(k)]                           # few large, many small tensors
        sizes = [max(1, int(x * total / sum(part))) for x in part]
        s["grads"] = [normal(n, scale=1e-2) for n in sizes]
        pad = [(n + 63) // 64 * 64 for n in sizes]        # views of one flat buffer, each on a 64-element boundary
        s["flat"] = torch.zeros(sum(pad), dtype=dt, device=_DEV)
        s["out"], o = [], 0
        for n, p in zip(sizes, pad):
            s["out"].append(s["flat"][o:o + n])
            o += p
        s["max_norm"] = 1.0                               # below the norm of all but the smallest sets
        return s
    b, d = case["batch"], case["d"]
    train = case.get("train", False)
    if op in ("conv", "conv_step"):
        w = case["width"]
        s["weight"], s["bias"] = normal(d, w, scale=w ** -0.5), normal(d, scale=0.1)
        if op == "conv_step":
            s["x"], s["state"] = normal(b, d), normal(w - 1, b, d)
            s["new"] = torch.empty_like(s["state"])
            return s
        s["x"], s["lengths"] = normal(case["t"], b, d), _lengths(case, g)
        if train:
            s["dy"] = normal(case["t"], b, d, scale=1e-1)
            for k in ("x", "weight", "bias"):
                s[k].requires_grad_(True)
        return s
    n, gr = case["state"], case["groups"]
    lead = (b,) if op == "scan_step" else (case["t"], b)
    s["x"], s["z"] = normal(*lead, d), normal(*lead, d)
    s["dt"] = normal(*lead, d, scale=0.5)
    # the usual start of such a layer: A = -1 .. -N, time steps between 1e-3 and 1e-1
    s["A"] = -(torch.arange(1, n + 1, device=_DEV).float() * torch.exp(0.1 * torch.randn(d, n, device=_DEV, generator=g)))
    step = torch.exp(torch.rand(d, device=_DEV, generator=g) * math.log(100.0) + math.log(1e-3))
    s["bias"] = step + torch.log(-torch.expm1(-step))
    s["D"] = torch.ones(d, device=_DEV) + 0.1 * torch.randn(d, device=_DEV, generator=g)
    s["B"], s["C"] = normal(*lead, gr, n), normal(*lead, gr, n)
    if op == "scan_step":
        s["state"] = torch.randn(b, d, n, device=_DEV, generator=g)
        s["new"] = torch.empty_like(s["state"])
        return s
    s["lengths"] = _lengths(case, g)
    if train:
        s["dy"] = normal(*lead, d, scale=1e-1)
        for k in ("x", "z", "dt", "A", "bias", "D", "B", "C"):
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------- plain forms
def _plain_embedding(s):
    w, idx = s["weight"].detach(), s["idx"]
    out = (w.float()[idx] * s["scale"]).to(w.dtype)
    if not s["case"]["train"]:
        return {"out": out}
    keep = torch.ones_like(idx, dtype=torch.bool) if s["pad"] is None else idx != s["pad"]
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, idx[keep], s["dout"][keep].float())
    return {"out": out, "dweight": (dw * s["scale"]).to(w.dtype)}


def _alive(x, lengths):
    """[steps, batch, 1] truth values: the step belongs to the sequence."""
    return torch.arange(x.shape[0], device=x.device)[:, None, None] < lengths[None, :, None]


def _shifted(xp, t, width):
    return [xp[k:k + t] for k in range(width)]


def _plain_conv(s):
    x, w, b = s["x"].detach(), s["weight"].detach().float(), s["bias"].detach().float()
    t, width = x.shape[0], w.shape[1]
    xf = x.float()
    if s["lengths"] is not None:
        alive = _alive(x, s["lengths"])
        xf = torch.where(alive, xf, torch.zeros_like(xf))
    xp = torch.cat([torch.zeros((width - 1,) + x.shape[1:], device=x.device), xf])
    p = b + sum(v * w[:, k] for k, v in enumerate(_shifted(xp, t, width)))
    sg = 1.0 / (1.0 + torch.exp(-p))
    y = p * sg
    if s["lengths"] is not None:
        y = torch.where(alive, y, torch.zeros_like(y))
    if not s["case"]["train"]:
        return {"y": y.to(x.dtype)}
    dp = s["dy"].float() * sg * (1.0 + p * (1.0 - sg))
    if s["lengths"] is not None:
        dp = torch.where(alive, dp, torch.zeros_like(dp))
    dw = torch.stack([(dp * v).sum((0, 1)) for v in _shifted(xp, t, width)], 1)
    dpp = torch.cat([dp, torch.zeros((width - 1,) + x.shape[1:], device=x.device)])
    dx = sum(v * w[:, width - 1 - k] for k, v in enumerate(_shifted(dpp, t, width)))
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dweight": dw.to(x.dtype), "dbias": dp.sum((0, 1)).to(x.dtype)}


def _plain_conv_step(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    full = torch.cat([s["state"], s["x"][None]])
    p = b + (full.float() * w.t()[:, None, :]).sum(0)
    return {"y": (p / (1.0 + torch.exp(-p))).to(s["x"].dtype), "state": full[1:]}


def _linear_scan(a, u):
    """h[t] = a[t] h[t-1] + u[t] along the first axis, by doubling."""
    t, k = a.shape[0], 1
    while k < t:
        u = torch.cat([u[:k], torch.addcmul(u[k:], a[k:], u[:-k])])
        if 2 * k < t:
            a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return u


def _softplus(v):
    return torch.where(v > 20.0, v, torch.log1p(torch.exp(v.clamp(max=20.0))))


def _to_channels(v, d):
    """[.., groups, N] -> [.., d, N]: the channels of a group share its row."""
    return v.repeat_interleave(d // v.shape[-2], dim=-2)


def _plain_scan(s):
    x, z, raw = (s[k].detach().float() for k in ("x", "z", "dt"))
    A, D, bias = (s[k].detach() for k in ("A", "D", "bias"))
    kind, d, n, gr = s["x"].dtype, x.shape[-1], A.shape[1], s["B"].shape[-2]
    Bc, Cc = s["B"].detach().float(), s["C"].detach().float()
    Bd, Cd = _to_channels(Bc, d), _to_channels(Cc, d)
    raw = raw + bias
    e = _softplus(raw)
    if s["lengths"] is not None:
        alive = _alive(x, s["lengths"])
        zero = torch.zeros((), device=x.device)
        e, x, z, Bd, Cd = (torch.where(alive if v.dim() == 3 else alive[..., None], v, zero) for v in (e, x, z, Bd, Cd))
    a = torch.exp(e[..., None] * A)
    h = _linear_scan(a, (e * x)[..., None] * Bd)
    sg = 1.0 / (1.0 + torch.exp(-z))
    pre = (h * Cd).sum(-1) + D * x
    y = pre * z * sg
    if not s["case"]["train"]:
        return {"y": y.to(kind), "state": h[-1]}
    dy = s["dy"].float()
    if s["lengths"] is not None:
        dy = torch.where(alive, dy, zero)
    gy = dy * z * sg
    after = torch.cat([a[1:], torch.ones_like(a[:1])])
    q = _linear_scan(after.flip(0), (gy[..., None] * Cd).flip(0)).flip(0)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    flow = q * a * before
    qb = (q * Bd).sum(-1)
    de = (flow * A).sum(-1) + qb * x
    draw_ = de * torch.where(raw > 20.0, torch.ones_like(raw), 1.0 / (1.0 + torch.exp(-raw)))
    if s["lengths"] is not None:
        draw_ = torch.where(alive, draw_, zero)

    def to_groups(v):
        return v.reshape(v.shape[:2] + (gr, d // gr, n)).sum(3).to(kind)

    return {"y": y.to(kind), "dx": (gy * D + qb * e).to(kind), "ddt": draw_.to(kind),
            "dz": (dy * pre * sg * (1.0 + z * (1.0 - sg))).to(kind), "dA": (flow * e[..., None]).sum((0, 1)),
            "dB": to_groups(q * (e * x)[..., None]), "dC": to_groups(h * gy[..., None]), "dD": (gy * x).sum((0, 1)),
            "dbias": draw_.sum((0, 1))}


def _plain_scan_step(s):
    x, z, e = s["x"].float(), s["z"].float(), _softplus(s["dt"].float() + s["bias"])
    d = x.shape[-1]
    h = torch.exp(e[..., None] * s["A"]) * s["state"] + (e * x)[..., None] * _to_channels(s["B"].float(), d)
    y = ((h * _to_channels(s["C"].float(), d)).sum(-1) + s["D"] * x) * z / (1.0 + torch.exp(-z))
    return {"y": y.to(s["x"].dtype), "state": h}


def _plain_clip(s):
    norm = torch.sqrt(torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]]).sum())
    c = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    for g, o in zip(s["grads"], s["out"]):
        o.copy_(g.float() * c)
    return {"norm": norm.float(), "grads": s["flat"]}


# ------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if not own:
        with torch.no_grad():
            return {"embedding": _plain_embedding, "conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan,
                    "scan_step": _plain_scan_step, "clip": _plain_clip}[op](s)
    train = s["case"].get("train", False)
    if op == "clip":
        from jova_amd.train import clip_grad_norm_
        return {"norm": clip_grad_norm_(s["grads"], s["max_norm"], out=s["out"]), "grads": s["flat"]}
    from jova_amd.nn import functional as F
    if op == "embedding":
        out = F.embedding(s["idx"], s["weight"], scale=s["scale"], padding_idx=s["pad"])
        if not train:
            return {"out": out}
        return {"out": out.detach(), "dweight": torch.autograd.grad(out, s["weight"], s["dout"])[0]}
    if op == "conv_step":
        y = F.causal_conv1d_step(s["x"], s["state"], s["weight"], s["bias"], activation="silu", out_state=s["new"])
        return {"y": y, "state": s["new"]}
    if op == "conv":
        y = F.causal_conv1d(s["x"], s["weight"], s["bias"], activation="silu", lengths=s["lengths"])
        if not train:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if op == "scan_step":
        y = F.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"], dt_bias=s["bias"],
                                  dt_softplus=True, out_state=s["new"])
        return {"y": y, "state": s["new"]}
    if not train:
        y, h = F.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["bias"],
                                dt_softplus=True, lengths=s["lengths"], return_final_state=True)
        return {"y": y, "state": h}
    y = F.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["bias"], dt_softplus=True,
                         lengths=s["lengths"])
    keys = ("x", "dt", "z", "A", "B", "C", "D", "bias")
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(keys, torch.autograd.grad(y, [s[k] for k in keys], s["dy"]))}}


# ------------------------------------------------------------------------------------------------------------- work
def work(case):
    op, es = case["op"], _SIZE[case["dtype"]]
    if op == "embedding":
        n, d, v = case["n"], case["d"], case["vocab"]
        if not case["train"]:
            return {"bytes": n * (8 + 2 * d * es), "flops": n * d}
        return {"bytes": n * (8 + 3 * d * es) + v * d * es, "flops": 3 * n * d}
    if op == "clip":
        return {"bytes": 2 * case["total"] * es + 4, "flops": 3 * case["total"]}
    b, d = case["batch"], case["d"]
    if op == "conv_step":
        w = case["width"]
        return {"bytes": es * (b * d * (2 + 2 * (w - 1)) + d * (w + 1)), "flops": b * d * (2 * w + 6)}
    if op == "conv":
        m, w = case["t"] * b * d, case["width"]
        if not case["train"]:
            return {"bytes": es * (2 * m + d * (w + 1)), "flops": m * (2 * w + 6)}
        return {"bytes": es * (4 * m + 2 * d * (w + 1)), "flops": m * (8 * w + 20)}
    n, gr = case["state"], case["groups"]
    if op == "scan_step":
        return {"bytes": 8 * b * d * n + es * (4 * b * d + 2 * b * gr * n) + 4 * d * (n + 2), "flops": b * d * (7 * n + 20)}
    m, bc = case["t"] * b * d, 2 * case["t"] * b * gr * n
    if not case["train"]:
        return {"bytes": es * (4 * m + bc) + 4 * (b * d * n + d * (n + 2)), "flops": m * (7 * n + 20)}
    return {"bytes": es * (8 * m + 2 * bc) + 8 * d * (n + 2), "flops": m * (23 * n + 50)}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"embedding": _exact_embedding, "conv": _exact_conv, "conv_step": _exact_conv_step, "scan": _exact_scan,
                "scan_step": _exact_scan_step, "clip": _exact_clip}[case["op"]](s)


def _exact_embedding(s):
    w, idx = s["weight"].detach(), s["idx"]
    out = w[idx].double() * s["scale"]
    if not s["case"]["train"]:
        return {"out": out}
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    dw.index_put_((idx,), s["dout"].double() * s["scale"], accumulate=True)
    if s["pad"] is not None:
        dw[s["pad"]] = 0
    return {"out": out, "dweight": dw}


def _exact_conv(s):
    """One step at a time over a window of inputs; the gradient step by step into the inputs that fed it."""
    w, bias = s["weight"].detach().double(), s["bias"].detach().double()
    x = s["x"].detach()
    t, b, d = x.shape
    width = w.shape[1]
    y = torch.zeros(t, b, d, dtype=torch.float64, device=x.device)
    train = s["case"]["train"]
    dx = torch.zeros_like(y) if train else None
    dw, db = torch.zeros_like(w), torch.zeros_like(bias)
    for i in range(t):
        lo = max(0, i - width + 1)
        win = x[lo:i + 1].double()
        ww = w[:, width - (i + 1 - lo):].t()
        p = bias + (win * ww[:, None, :]).sum(0)
        live = torch.ones(b, 1, dtype=torch.bool, device=x.device) if s["lengths"] is None else (s["lengths"] > i)[:, None]
        sg = torch.sigmoid(p)
        y[i] = torch.where(live, p * sg, torch.zeros_like(p))
        if train:
            dp = torch.where(live, s["dy"][i].double() * (sg + p * sg * (1 - sg)), torch.zeros_like(p))
            dx[lo:i + 1] += dp[None] * ww[:, None, :]
            dw[:, width - (i + 1 - lo):] += (win * dp[None]).sum(1).t()
            db += dp.sum(0)
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db} if train else {"y": y}


def _exact_conv_step(s):
    w = s["weight"].double()
    p = s["bias"].double() + s["x"].double() * w[:, -1]
    for k in range(w.shape[1] - 1):
        p = p + s["state"][k].double() * w[:, k]
    new = s["state"].double().roll(-1, 0)
    if new.shape[0]:
        new[-1] = s["x"].double()
    return {"y": p * torch.sigmoid(p), "state": new}


def _exact_terms(s, i=None):
    """x, z, dt + bias, its softplus, B and C of one step in 64 bits."""
    def at(k):
        v = s[k].detach()
        return (v if i is None else v[i]).double()
    raw = at("dt") + s["bias"].detach().double()
    d, gr = raw.shape[-1], s["B"].shape[-2]
    of = torch.arange(d, device=raw.device) // (d // gr)
    return at("x"), at("z"), raw, torch.logaddexp(raw, torch.zeros_like(raw)), at("B")[:, of], at("C")[:, of], of


def _exact_scan(s):
    """The recurrence one step at a time, and its adjoint one step at a time backwards."""
    t, b, d = s["x"].shape
    A, D = s["A"].detach().double(), s["D"].detach().double()
    n, gr, dev, train = A.shape[1], s["B"].shape[-2], A.device, s["case"]["train"]
    h = torch.zeros(b, d, n, dtype=torch.float64, device=dev)
    y = torch.zeros(t, b, d, dtype=torch.float64, device=dev)
    kept = []
    len_ = torch.full((b,), t, device=dev) if s["lengths"] is None else s["lengths"].long()
    for i in range(t):
        x, z, raw, e, B, C, _ = _exact_terms(s, i)
        live = (len_ > i)[:, None, None]
        if train:
            kept.append(h)
        h = torch.where(live, torch.exp(e[..., None] * A) * h + (e * x)[..., None] * B, h)
        y[i] = torch.where(live[..., 0], ((C * h).sum(-1) + D * x) * z * torch.sigmoid(z), torch.zeros_like(x))
    if not train:
        return {"y": y, "state": h}
    dx, dr, dz = (torch.zeros_like(y) for _ in range(3))
    dB, dC = (torch.zeros(t, b, gr, n, dtype=torch.float64, device=dev) for _ in range(2))
    dA, dD, db = torch.zeros_like(A), torch.zeros_like(D), torch.zeros_like(D)
    q = torch.zeros_like(h)
    for i in reversed(range(t)):
        x, z, raw, e, B, C, of = _exact_terms(s, i)
        live = (len_ > i)[:, None]
        old = kept.pop()
        a = torch.exp(e[..., None] * A)
        now = torch.where(live[..., None], a * old + (e * x)[..., None] * B, old)
        dy = torch.where(live, s["dy"][i].double(), torch.zeros_like(x))
        sg = torch.sigmoid(z)
        dz[i] = dy * ((C * now).sum(-1) + D * x) * (sg + z * sg * (1 - sg))
        gy = dy * z * sg
        q = q + C * gy[..., None]
        m = torch.where(live[..., None], q, torch.zeros_like(q))
        dC[i].index_add_(1, of, now * gy[..., None])
        dB[i].index_add_(1, of, m * (e * x)[..., None])
        dD += (gy * x).sum(0)
        through = m * a * old
        dA += (through * e[..., None]).sum(0)
        mb = (m * B).sum(-1)
        dr[i] = ((through * A).sum(-1) + mb * x) * torch.sigmoid(raw)
        db += dr[i].sum(0)
        dx[i] = gy * D + mb * e
        q = torch.where(live[..., None], a * q, q)
    return {"y": y, "dx": dx, "ddt": dr, "dz": dz, "dA": dA, "dB": dB, "dC": dC, "dD": dD, "dbias": db}


def _exact_scan_step(s):
    x, z, _, e, B, C, _ = _exact_terms(s)
    h = torch.exp(e[..., None] * s["A"].double()) * s["state"].double() + (e * x)[..., None] * B
    return {"y": ((C * h).sum(-1) + s["D"].double() * x) * z * torch.sigmoid(z), "state": h}


def _exact_clip(s):
    total = torch.zeros((), dtype=torch.float64, device=_DEV)
    for g in s["grads"]:
        total += torch.linalg.vector_norm(g.double()) ** 2
    norm = total.sqrt()
    c = torch.minimum(s["max_norm"] / (norm + 1e-6), torch.ones_like(norm))
    flat, o = torch.zeros(s["flat"].shape, dtype=torch.float64, device=_DEV), 0
    for g in s["grads"]:
        n = g.numel()
        flat[o:o + n] = g.double() * c
        o += (n + 63) // 64 * 64
    return {"norm": norm, "grads": flat}
