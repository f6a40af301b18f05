"""What the operators of packed training are timed on: the norm and rotation of
queries and keys, attention over packed sequences with grouped heads, and the
cross-entropy of a linear layer that keeps no logits.

A batch is packed: `T` tokens of `n` sequences lie one behind the other, and
`starts` (int32, n + 1) says where each begins. Every tensor is f32, the type
the entry points take. A case is a dict: "op" names the operator, "train" says
whether the pass runs the backward after the forward, the other keys are sizes
and options. Where `own` is true, `run` calls the library (include/vearo_hip.h);
otherwise it computes the same in elementary torch operations.
"""
import math
import random

import torch

own = False

EPS = 1e-6
IGNORE = -100.0


# ------------------------------------------------------------------- cases --

def listed():
    return [
        # Queries and keys of a small model's block (the tests' medium model): bound by launches.
        {"name": "qk_rope_256x4x4x32", "op": "qk_rope", "T": 256, "n": 2, "ragged": False, "Hq": 4, "Hk": 4, "D": 32,
         "rotary": 32, "interleaved": False, "base": 1e4, "far": 0, "train": True},
        # The GPT-2-small batch of 16 x 1024 tokens, 12 heads on 4 key heads, forward alone (evaluation).
        {"name": "qk_rope_fwd_16384x12x4x64", "op": "qk_rope", "T": 16384, "n": 16, "ragged": False, "Hq": 12, "Hk": 4,
         "D": 64, "rotary": 64, "interleaved": False, "base": 1e4, "far": 0, "train": False},
        # Ragged documents, far positions, neighbouring pairs, half of each head rotated, odd token count.
        {"name": "qk_rope_10007x12x2x80", "op": "qk_rope", "T": 10007, "n": 23, "ragged": True, "Hq": 12, "Hk": 2, "D": 80,
         "rotary": 40, "interleaved": True, "base": 5e5, "far": 100000, "train": True},
        # One block's training pass at width 2048 in 16 heads of 128.
        {"name": "qk_rope_16384x16x4x128", "op": "qk_rope", "T": 16384, "n": 9, "ragged": True, "Hq": 16, "Hk": 4, "D": 128,
         "rotary": 128, "interleaved": False, "base": 1e4, "far": 0, "train": True},
        # The smallest attention: two short sequences of a small model.
        {"name": "attention_2x128x4x4x32", "op": "attention", "T": 256, "n": 2, "ragged": False, "Hq": 4, "Hk": 4, "D": 32,
         "causal": True, "train": True},
        # The GPT-2-small batch, forward alone, grouped heads.
        {"name": "attention_fwd_16x1024x12x4x64", "op": "attention", "T": 16384, "n": 16, "ragged": False, "Hq": 12, "Hk": 4,
         "D": 64, "causal": True, "train": False},
        # The same number of tokens in 40 documents of uneven length, every head its own keys: the ordinary training pass.
        {"name": "attention_packed_16384x12x12x64", "op": "attention", "T": 16384, "n": 40, "ragged": True, "Hq": 12,
         "Hk": 12, "D": 64, "causal": True, "train": True},
        # Short sentences seen from both sides, a head of 80 and an odd token count.
        {"name": "attention_both_ways_5003x12x6x80", "op": "attention", "T": 5003, "n": 37, "ragged": True, "Hq": 12, "Hk": 6,
         "D": 80, "causal": False, "train": True},
        # One long document, 16 heads of 128 on 2 key heads.
        {"name": "attention_1x8192x16x2x128", "op": "attention", "T": 8192, "n": 1, "ragged": False, "Hq": 16, "Hk": 2,
         "D": 128, "causal": True, "train": True},
        # The loss of a small model (the tests' medium vocabulary), its backward as a call of its own (a tape's).
        {"name": "linear_xent_apart_256x128x1000", "op": "linear_xent", "R": 256, "D": 128, "V": 1000, "ignored": 0.0,
         "apart": True, "train": True},
        # The loss alone (evaluation) on a short ragged batch.
        {"name": "linear_xent_fwd_4001x768x50257", "op": "linear_xent", "R": 4001, "D": 768, "V": 50257, "ignored": 0.3,
         "apart": True, "train": False},
        # The GPT-2-small lm_head and loss as a step's root: loss, input and weight gradient in one call; padding is not counted.
        {"name": "linear_xent_16384x768x50257", "op": "linear_xent", "R": 16384, "D": 768, "V": 50257, "ignored": 0.1,
         "apart": False, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk_rope", "attention", "attention", "linear_xent"])
    if op == "linear_xent":
        return {"op": op, "R": _log(rng, 100, 8192), "D": 4 * _log(rng, 32, 256), "V": _log(rng, 1000, 50257),
                "ignored": rng.choice([0.0, 0.1, 0.5]), "apart": rng.random() < 0.4, "train": rng.random() < 0.7}
    Hk = rng.choice([1, 2, 3, 4, 8])
    c = {"op": op, "T": _log(rng, 200, 16384), "Hk": Hk, "Hq": Hk * rng.choice([1, 2, 3, 4]) if Hk < 8 else 8,
         "D": rng.choice([32, 40, 64, 64, 80, 96, 112, 128]), "train": rng.random() < 0.7}
    c["n"] = min(_log(rng, 1, 64), c["T"])
    c["ragged"] = rng.random() < 0.8
    if op == "qk_rope":
        c |= {"rotary": rng.choice([c["D"], c["D"] // 2]), "interleaved": rng.random() < 0.4,
              "base": rng.choice([1e4, 5e5]), "far": rng.choice([0, 0, 30000, 1000000])}
    else:
        c["causal"] = rng.random() < 0.8
        if c["n"] < 4:  # no costlier than the long document above
            c["T"] = min(c["T"], 8192)
    return c


def _lengths(c):
    """The sequences' lengths, from the case alone: even ones (the rest in the last), or uneven ones with a single token
    among them."""
    T, n = c["T"], c["n"]
    if not c["ragged"] or n == 1:
        return [T // n] * (n - 1) + [T - T // n * (n - 1)]
    rng = random.Random("%d tokens in %d" % (T, n))
    part = [0.1 + rng.random() ** 2 for _ in range(n)]
    lens = [max(1, int(T * p / sum(part))) for p in part]
    lens[rng.randrange(n)] = 1
    lens[lens.index(max(lens))] += T - sum(lens)
    return lens


# ----------------------------------------------------------------- prepare --

def _inputs(c, seed):
    """The arrays a pass reads: the same values for run() and exact()."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, device="cuda").normal_(mean, std, generator=g)

    if c["op"] == "linear_xent":
        R, D, V = c["R"], c["D"], c["V"]
        t = torch.randint(0, V, (R,), device="cuda", generator=g).float()
        left = torch.rand(R, device="cuda", generator=g) < c["ignored"]
        return {"x": normal(R, D), "w": normal(V, D, std=0.05), "t": t.masked_fill_(left, IGNORE),
                "go": torch.ones(1, device="cuda")}
    T, Hq, Hk, D = c["T"], c["Hq"], c["Hk"], c["D"]
    lens = torch.tensor(_lengths(c), dtype=torch.int64)
    starts = torch.cat([lens.new_zeros(1), lens.cumsum(0)])
    # Queries, keys and values as column blocks of one projection, as a block holds them.
    s = {"qkv": normal(T, Hq + 2 * Hk, D), "starts": starts.to(torch.int32).cuda()}
    if c["op"] == "qk_rope":
        place = torch.arange(T) - starts[:-1].repeat_interleave(lens) + c["far"]
        s |= {"positions": place.float().cuda(), "wq": normal(D, std=0.1, mean=1.0), "wk": normal(D, std=0.1, mean=1.0),
              "dyq": normal(T, Hq, D), "dyk": normal(T, Hk, D)}
    else:
        s["do"] = normal(T, Hq, D)
    return s


def prepare(case, seed):
    from vearo_amd import _abi as vh

    vh.init(0)
    c, s = case, _inputs(case, seed)
    e = lambda *shape: torch.empty(shape, device="cuda")  # noqa: E731
    s["case"] = c
    if c["op"] == "linear_xent":
        s |= {"loss": e(1), "stats": e(c["R"], 2), "dx": torch.empty_like(s["x"]), "dw": torch.empty_like(s["w"])}
        return s
    T, Hq, Hk, D = c["T"], c["Hq"], c["Hk"], c["D"]
    s["heads"] = {H: vh.layout([T, H, D]) for H in (Hq, Hk)}
    s["cols"] = {H: vh.layout([T, H, D], [(Hq + 2 * Hk) * D, D, 1]) for H in (Hq, Hk)}
    s["longest"] = max(_lengths(c))
    s["dqkv"] = torch.zeros_like(s["qkv"])
    if c["op"] == "qk_rope":
        s |= {"yq": e(T, Hq, D), "yk": e(T, Hk, D), "dwq": e(D), "dwk": e(D)}
    else:
        s |= {"o": e(T, Hq, D), "lse": e(Hq, T)}
    return s


# --------------------------------------------------------------------- run --

def run(s):
    if own:
        return _library(s)
    with torch.no_grad():
        return {"qk_rope": _qk_rope, "attention": _attention, "linear_xent": _linear_xent}[s["case"]["op"]](s)


def _library(s):
    from vearo_amd import _abi as vh

    c, L = s["case"], vh.lib
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if c["op"] == "linear_xent":
        R, D, V = c["R"], c["D"], c["V"]
        if c["apart"] or not c["train"]:
            vh.check(L.vh_linear_cross_entropy_fwd(p["x"], D, p["w"], D, p["t"], IGNORE, p["loss"], p["stats"], R, D, V,
                                                   None, 0, None))
            if not c["train"]:
                return {k: s[k] for k in ("loss", "stats")}
            vh.check(L.vh_linear_cross_entropy_bwd(p["x"], D, p["w"], D, p["t"], IGNORE, p["stats"], p["go"], p["dx"], D,
                                                   p["dw"], D, R, D, V, None, 0, None))
            return {k: s[k] for k in ("loss", "stats", "dx", "dw")}
        vh.check(L.vh_linear_cross_entropy_fwd_bwd(p["x"], D, p["w"], D, p["t"], IGNORE, p["go"], p["loss"], p["dx"], D,
                                                   p["dw"], D, R, D, V, None, 0, None))
        return {k: s[k] for k in ("loss", "dx", "dw")}
    Hq, Hk, D = c["Hq"], c["Hk"], c["D"]
    cols, heads = s["cols"], s["heads"]
    k, v, dk, dv = (p[x] + 4 * (Hq + i * Hk) * D for x in ("qkv", "dqkv") for i in (0, 1))
    q, dq = p["qkv"], p["dqkv"]
    if c["op"] == "qk_rope":
        rope = (p["positions"], EPS, c["base"], c["rotary"], int(c["interleaved"]))
        vh.check(L.vh_qk_norm_rope_fwd(q, cols[Hq], k, cols[Hk], p["wq"], p["wk"], *rope, p["yq"], heads[Hq], p["yk"],
                                       heads[Hk], None))
        if not c["train"]:
            return {x: s[x] for x in ("yq", "yk")}
        vh.check(L.vh_qk_norm_rope_bwd(q, cols[Hq], k, cols[Hk], p["wq"], p["wk"], *rope, p["dyq"], heads[Hq], p["dyk"],
                                       heads[Hk], dq, cols[Hq], dk, cols[Hk], p["dwq"], p["dwk"], None, 0, None))
        return {x: s[x] for x in ("yq", "yk", "dqkv", "dwq", "dwk")}
    args = (q, cols[Hq], k, cols[Hk], v, cols[Hk], p["starts"], c["n"], D ** -0.5, int(c["causal"]))
    vh.check(L.vh_packed_attention_fwd(*args, p["o"], heads[Hq], p["lse"], None, 0, None))
    if not c["train"]:
        return {x: s[x] for x in ("o", "lse")}
    vh.check(L.vh_packed_attention_bwd(*args, p["o"], heads[Hq], p["lse"], p["do"], heads[Hq], dq, cols[Hq], dk, cols[Hk],
                                       dv, cols[Hk], None, 0, None))
    return {x: s[x] for x in ("o", "lse", "dqkv")}


def _turn(x, cos, sin, R, interleaved):
    """The first R of each head's elements, turned pair by pair."""
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., R:]], -1)


def _qk_rope(s):
    c = s["case"]
    Hq, Hk, R = c["Hq"], c["Hk"], c["rotary"]
    rate = c["base"] ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    angle = (s["positions"].double()[:, None] * rate)[:, None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    q, k = s["qkv"][:, :Hq], s["qkv"][:, Hq:Hq + Hk]

    def forward(x, w):
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        return r, _turn(x * r * w, cos, sin, R, c["interleaved"])

    def backward(x, w, r, dy):
        g = _turn(dy, cos, -sin, R, c["interleaved"])
        n, h = x * r, g * w
        return r * (h - n * (h * n).mean(-1, keepdim=True)), (g * n).sum((0, 1))

    rq, yq = forward(q, s["wq"])
    rk, yk = forward(k, s["wk"])
    if not c["train"]:
        return {"yq": yq, "yk": yk}
    dq, dwq = backward(q, s["wq"], rq, s["dyq"])
    dk, dwk = backward(k, s["wk"], rk, s["dyk"])
    dqkv = torch.zeros_like(s["qkv"])
    dqkv[:, :Hq] = dq
    dqkv[:, Hq:Hq + Hk] = dk
    return {"yq": yq, "yk": yk, "dqkv": dqkv, "dwq": dwq, "dwk": dwk}


def _attention(s):
    """Every sequence padded to the longest: [n, Hk, G, L, D] blocks, G query heads on a key head."""
    c = s["case"]
    T, n, Hq, Hk, D, L = c["T"], c["n"], c["Hq"], c["Hk"], c["D"], s["longest"]
    G, scale = Hq // Hk, D ** -0.5
    starts = s["starts"].long()
    lens = starts[1:] - starts[:-1]
    at = torch.arange(L, device="cuda")
    live = at < lens[:, None]
    token = (starts[:-1, None] + at).clamp_(max=T - 1)
    rows = torch.arange(T, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), rows, right=True)
    off = rows - starts[seq]

    def pad(x, H):
        return torch.where(live[:, :, None, None], x[token], 0.0).permute(0, 2, 1, 3).reshape(n, Hk, H // Hk, L, D)

    def packed(x):
        return x.reshape(n, -1, L, D)[seq, :, off]

    q, k, v = pad(s["qkv"][:, :Hq], Hq), pad(s["qkv"][:, Hq:Hq + Hk], Hk), pad(s["qkv"][:, Hq + Hk:], Hk)
    mask = live[:, None, :]
    if c["causal"]:
        mask = mask & (at <= at[:, None])
    flat = lambda x: x.reshape(n * Hk, G * L, -1)  # noqa: E731
    one = lambda x: x.reshape(n * Hk, L, D)  # noqa: E731
    turned = lambda x: x.transpose(1, 2).contiguous()  # noqa: E731
    S = torch.bmm(flat(q), turned(one(k))).mul_(scale).reshape(n, Hk, G, L, L)
    S.masked_fill_(~mask[:, None, None], -math.inf)
    top = S.amax(-1, keepdim=True)
    P = S.sub_(top).exp_()
    total = P.sum(-1, keepdim=True)
    P = P.div_(total).reshape(n * Hk, G * L, L)
    o = torch.bmm(P, one(v))
    out = {"o": packed(o), "lse": (top + total.log()).reshape(n, Hq, L)[seq, :, off].t().contiguous()}
    if not c["train"]:
        return out
    do = flat(pad(s["do"], Hq))
    dv = torch.bmm(turned(P), do)
    dS = torch.bmm(do, turned(one(v))).sub_((do * o).sum(-1, keepdim=True)).mul_(P).mul_(scale)
    dq, dk = torch.bmm(dS, one(k)), torch.bmm(turned(dS), flat(q))
    out["dqkv"] = torch.cat([packed(dq), packed(dk), packed(dv)], 1)
    return out


def _linear_xent(s):
    x, w, t = s["x"], s["w"], s["t"]
    counted = t != IGNORE
    number = counted.sum().clamp(min=1)
    target = torch.where(counted, t, 0.0).long()[:, None]
    logits = x @ w.t()
    top = logits.amax(-1, keepdim=True)
    e = (logits - top).exp_()
    total = e.sum(-1, keepdim=True)
    row = (top + total.log() - logits.gather(1, target))[:, 0]
    loss = (torch.where(counted, row, 0.0).sum() / number).reshape(1)
    out = {"loss": loss}
    if s["case"]["apart"] or not s["case"]["train"]:
        out["stats"] = torch.cat([top, total], 1)
    if not s["case"]["train"]:
        return out
    d = e.div_(total)
    d.scatter_add_(1, target, torch.full_like(total, -1.0))
    d.mul_((counted * (s["go"] / number))[:, None])
    return out | {"dx": d @ w, "dw": d.t().contiguous() @ x}


# ------------------------------------------------------------- work, exact --

def work(c):
    if c["op"] == "linear_xent":
        R, D, V = c["R"], c["D"], c["V"]
        io = 4 * (R * D + V * D + R + (2 * R if c["apart"] or not c["train"] else 0))
        if not c["train"]:
            return {"bytes": io, "flops": 2 * R * D * V}
        return {"bytes": io + 4 * (R * D + V * D), "flops": 6 * R * D * V}
    T, Hq, Hk, D = c["T"], c["Hq"], c["Hk"], c["D"]
    if c["op"] == "qk_rope":
        x = T * (Hq + Hk) * D
        # Forward: read x, write y; backward: read x and dy, write dx.
        return {"bytes": 4 * (x * (4 if c["train"] else 2) + T), "flops": x * (30 if c["train"] else 10)}
    pairs = sum(L * (L + 1) // 2 if c["causal"] else L * L for L in _lengths(c)) * Hq
    io = 4 * T * D * (2 * Hq + 2 * Hk) + 4 * T * Hq
    if not c["train"]:
        return {"bytes": io, "flops": 4 * pairs * D}
    return {"bytes": io + 4 * T * D * (2 * Hq + 2 * Hk), "flops": 14 * pairs * D}


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    d = {k: v.double() for k, v in s.items()}
    if c["op"] == "linear_xent":
        x, w = d["x"], d["w"]
        keep = (s["t"] != IGNORE).nonzero()[:, 0]
        t = d["t"][keep].long()
        z = x @ w.t()
        lse, top = torch.logsumexp(z, -1, keepdim=True), z.max(-1, keepdim=True).values
        lp = z.sub_(lse)[keep]
        loss = -lp[torch.arange(len(t), device="cuda"), t].sum().reshape(1) / max(1, len(t))
        out = {"loss": loss}
        if c["apart"] or not c["train"]:
            out["stats"] = torch.cat([top, torch.exp(lse - top)], 1)
        if not c["train"]:
            return out
        g = lp.exp_()
        g[torch.arange(len(t), device="cuda"), t] -= 1
        g /= max(1, len(t))
        return out | {"dx": torch.zeros_like(x).index_copy_(0, keep, g @ w), "dw": g.t() @ x[keep]}
    T, Hq, Hk, D = c["T"], c["Hq"], c["Hk"], c["D"]
    if c["op"] == "qk_rope":
        R = c["rotary"]
        i = torch.arange(R // 2, dtype=torch.float64, device="cuda")
        # Turning a pair is a product with exp(i angle).
        z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda").expand(T, R // 2),
                        d["positions"][:, None] * torch.exp(i * (-2.0 / R * math.log(c["base"]))))[:, None]

        def f(x, w):
            y = w * x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / D + EPS)
            r = y[..., :R]
            if c["interleaved"]:
                u = torch.complex(r[..., 0::2], r[..., 1::2]) * z
                r = torch.view_as_real(u).reshape(r.shape)
            else:
                u = torch.complex(r[..., :R // 2], r[..., R // 2:]) * z
                r = torch.cat([u.real, u.imag], -1)
            return torch.cat([r, y[..., R:]], -1)

        qkv, wq, wk = (d[k].requires_grad_() for k in ("qkv", "wq", "wk"))
        yq, yk = f(qkv[:, :Hq], wq), f(qkv[:, Hq:Hq + Hk], wk)
        out = {"yq": yq.detach(), "yk": yk.detach()}
        if c["train"]:
            out |= dict(zip(("dqkv", "dwq", "dwk"), torch.autograd.grad([yq, yk], [qkv, wq, wk], [d["dyq"], d["dyk"]])))
        return out
    qkv, do = d["qkv"], d["do"]
    o, lse = torch.zeros_like(do), torch.zeros(Hq, T, dtype=torch.float64, device="cuda")
    dqkv = torch.zeros_like(qkv)
    t0 = 0
    for L in _lengths(c):
        t1 = t0 + L
        x = qkv[t0:t1].clone().requires_grad_()
        q, k, v = (y.transpose(0, 1) for y in x.split([Hq, Hk, Hk], 1))
        k, v = (y.repeat_interleave(Hq // Hk, 0) for y in (k, v))
        z = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(D)
        if c["causal"]:
            z = z + torch.full((L, L), -math.inf, dtype=torch.float64, device="cuda").triu(1)
        y = torch.matmul(torch.softmax(z, -1), v).transpose(0, 1)
        o[t0:t1], lse[:, t0:t1] = y.detach(), torch.logsumexp(z.detach(), -1)
        if c["train"]:
            dqkv[t0:t1] = torch.autograd.grad(y, x, do[t0:t1])[0]
        t0 = t1
    return {"o": o, "lse": lse, "dqkv": dqkv} if c["train"] else {"o": o, "lse": lse}
