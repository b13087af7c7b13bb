"""A block's attention: what is measured of it.

Two operators.  Attention: softmax(scale q k^T) v of grouped heads without the
[queries, keys] weights in memory, and its gradients, which recompute them; its
form for few rows of queries over a long cache (single tokens, trees of drafted
tokens) is the same call (`hip.Attention`).  Head norms and rotation: the RMS
norm of each head of the queries and keys and the rotation by their positions
in one pass, and its gradients (`hip.HeadRotary`).

`own` false: the operators written out in elementary torch operations in f32.
`own` true: the calls a program makes of the framework.  Inputs, in either
case, are tensors on the GPU in their storage type; outputs and workspace are
taken anew in each call.

Sizes are the configurations' (the course GPT's 64 x 6 heads x 256 x 64, the
Llama-shaped 32 heads x 2048 x 128) and generic ones around them.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _attn(name, what, dtype, batch, heads, kv, tq, tk, d, kind, window=0, ragged=False):
    return {"name": name, "op": "attention", "what": what, "dtype": dtype, "batch": batch, "heads": heads, "kv": kv, "tq": tq,
            "tk": tk, "d": d, "kind": kind, "window": window, "ragged": ragged}


def _rot(name, what, dtype, batch, seq, heads, kv, d, rotary, norm, even=False, far=0):
    return {"name": name, "op": "rotary", "what": what, "dtype": dtype, "batch": batch, "seq": seq, "heads": heads, "kv": kv, "d": d,
            "rotary": rotary, "norm": norm, "even": even, "far": far}


def listed():
    return [
        # one layer of the course GPT's training step: value and gradients
        _attn("attention-course-step-f32", "step", "f32", 64, 6, 6, 256, 256, 64, "causal"),
        # the course GPT's next character after a full context: the smallest call
        _attn("attention-course-token-f32", "value", "f32", 1, 6, 6, 1, 256, 64, "all"),
        # one layer of the Llama-shaped forward: a prompt of 2048 tokens
        _attn("attention-prompt-bf16", "value", "bf16", 1, 32, 32, 2048, 2048, 128, "causal"),
        # a training step over four sequences with grouped heads: the largest
        _attn("attention-wide-step-bf16", "step", "bf16", 4, 32, 8, 4096, 4096, 128, "causal"),
        # serving: the next token of 32 sequences of unequal lengths
        _attn("attention-tokens-bf16", "value", "bf16", 32, 32, 8, 1, 8192, 128, "causal", ragged=True),
        # a tree of 24 drafted tokens for each of 8 sequences
        _attn("attention-drafts-f16", "value", "f16", 8, 32, 8, 24, 4096, 128, "tree", ragged=True),
        # sizes that are no multiple of anything, more keys than queries, a window
        _attn("attention-odd-vjp-f16", "vjp", "f16", 3, 10, 5, 777, 1021, 80, "causal", window=300, ragged=True),
        # documents packed into sequences, by a mask a sequence
        _attn("attention-packed-step-bf16", "step", "bf16", 2, 12, 12, 1024, 1024, 64, "documents"),
        # the Llama-shaped forward's rotation of its queries and keys
        _rot("rotary-prompt-bf16", "value", "bf16", 1, 2048, 32, 32, 128, 128, False),
        # a training step over 8192 tokens with normed heads
        _rot("rotary-wide-step-bf16", "step", "bf16", 2, 4096, 32, 8, 128, 128, True),
        # serving: single tokens at far positions
        _rot("rotary-tokens-f16", "value", "f16", 32, 1, 32, 8, 128, 128, True, far=500000),
        # odd sizes, half of a head rotated, neighbours paired
        _rot("rotary-odd-step-f32", "step", "f32", 3, 777, 10, 5, 80, 40, True, even=True, far=30000),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size of [lo, hi]: one in three as drawn (odd ones among them), the
    others whole eights or sixty-fours, as models have them."""
    v, step = _log(rng, lo, hi), rng.choice((1, 8, 64))
    return max(lo, min(hi, (v + step - 1) // step * step))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    kv = rng.choice([1, 2, 5, 6, 8, 12, 32])
    heads = kv * rng.choice([1, 1, 2, 4, 8])
    while heads > 64:
        heads //= 2
        kv = max(1, kv // 2)
    heads = heads // kv * kv
    d = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    if rng.random() < 0.4:
        while True:
            batch, seq = _log(rng, 1, 32), _size(rng, 1, 16384)
            if batch * seq * (heads + kv) * d <= 8192 * 40 * 128:
                break
        return {"op": "rotary", "what": rng.choice(["value", "step"]), "dtype": dtype, "batch": batch, "seq": seq, "heads": heads,
                "kv": kv, "d": d, "rotary": rng.choice([d, d, d // 2]), "norm": rng.random() < 0.6, "even": rng.random() < 0.3,
                "far": rng.choice([0, 0, 4000, 1000000])}
    use = rng.choice(["train", "train", "prompt", "tokens", "tree"])
    window, ragged, kind = 0, False, "causal"
    most = 4 * 32 * 4096 * 4096 / (4 if dtype == "f32" else 1)
    while True:
        batch = _log(rng, 1, 64)
        if use in ("train", "prompt"):
            tq = _size(rng, 17, 8192)
            tk = tq if use == "train" or rng.random() < 0.5 else tq + _size(rng, 1, 4096)
        else:
            tq = 1 if use == "tokens" else rng.randint(2, 64)
            tk = tq + _size(rng, 1, 32768)
        if batch * heads * tq * tk <= most and batch * tk * heads * d <= 1.1e9:
            break
    what = rng.choice(["step", "vjp"]) if use == "train" else "value"
    if use == "train":
        kind = rng.choice(["causal", "causal", "all", "documents"])
        if kind == "documents" and batch * tq * tk > 2e8:
            kind = "causal"
        ragged = kind != "documents" and rng.random() < 0.3
    elif use == "tree":
        kind, ragged = "tree", True
    else:
        ragged = rng.random() < 0.7
    if kind == "causal" and rng.random() < 0.25:
        window = _log(rng, 16, 4096)
    return {"op": "attention", "what": what, "dtype": dtype, "batch": batch, "heads": heads, "kv": kv, "tq": tq, "tk": tk, "d": d,
            "kind": kind, "window": window, "ragged": ragged}


# ---- inputs -------------------------------------------------------------------

def _lens(c):
    """The sequences' numbers of keys: all of them, or from a quarter on."""
    b, tq, tk = c["batch"], c["tq"], c["tk"]
    if not c["ragged"]:
        return [tk] * b
    return [max(1 if tq == tk else tq, tk - (tk * 3 // 4) * ((7 * i + 3) % b) // b) for i in range(b)]


def _first(c):
    """The first query's position in each sequence: the queries are its last
    keys, or, as many as the keys, stand beside them (and past its end, padded)."""
    return [0 if c["tq"] == c["tk"] else n - c["tq"] for n in _lens(c)]


def _attention_inputs(c, seed):
    """q, k ~ N(0, 1) and so scores ~ N(0, 1) after 1 / sqrt(d), v and the
    cotangent ~ N(0, 1), [batch, seq, heads, d] as the projections leave them;
    a cache's keys past a sequence's end hold what an earlier one left."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    b, h, kv, tq, tk, d, dt = c["batch"], c["heads"], c["kv"], c["tq"], c["tk"], c["d"], TORCH[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g).to(dt)

    s = {"q": normal(b, tq, h, d), "k": normal(b, tk, kv, d), "v": normal(b, tk, kv, d)}
    if c["ragged"]:
        s["lens"] = torch.tensor(_lens(c), device=DEV)
    if c["kind"] in ("causal", "tree"):
        s["first"] = torch.tensor(_first(c), device=DEV)
    if c["kind"] == "tree":
        # a drafted token follows one of those before it, and reads its
        # ancestors and itself
        m = torch.zeros(b, tq, tq, dtype=torch.bool)
        parent = (torch.rand(b, tq, generator=torch.Generator().manual_seed(seed)) * torch.arange(tq)).long()
        for i in range(tq):
            if i:
                m[:, i] = m[torch.arange(b), parent[:, i]]
            m[:, i, i] = True
        s["mask"] = m.to(DEV)
    if c["kind"] == "documents":
        starts = torch.rand(b, tq, device=DEV, generator=g) < 4 / tq
        doc = starts.long().cumsum(1)
        m = (doc[:, :, None] == doc[:, None, :]) & torch.ones(tq, tk, dtype=torch.bool, device=DEV).tril()
        s["mask"] = m.contiguous()
        s["first"] = torch.zeros(b, dtype=torch.int64, device=DEV)
    if c["what"] != "value":
        s["do"] = normal(b, tq, h, d)
    if c["what"] == "vjp":
        # the forward's outputs, as it leaves them
        f = _plain_attention({**c, "what": "value"}, s)
        s["o"], s["lse"] = f["o"], f["lse"]
    return s


def _rotary_inputs(c, seed):
    """Heads ~ N(0, 1) of unequal size, gains about one, positions from `far` on."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    b, n, h, kv, d, dt = c["batch"], c["seq"], c["heads"], c["kv"], c["d"], TORCH[c["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device=DEV, generator=g) * std

    s = {"q": (normal(b, n, h, d) * (0.5 + 0.1 * normal(b, n, h, 1).abs())).to(dt), "k": normal(b, n, kv, d).to(dt)}
    r = c["rotary"]
    s["freq"] = 1e4 ** (-2.0 * torch.arange(r // 2, device=DEV, dtype=torch.float64) / r)
    if c["far"]:
        s["at"] = torch.randint(0, c["far"], (b, 1), device=DEV, generator=g) + torch.arange(n, device=DEV)
    if c["norm"]:
        s["gq"], s["gk"] = (1.0 + normal(d, std=0.1)).to(dt), (1.0 + normal(d, std=0.1)).to(dt)
    if c["what"] == "step":
        s["dyq"], s["dyk"] = normal(b, n, h, d).to(dt), normal(b, n, kv, d).to(dt)
    return s


def _inputs(c, seed):
    return (_attention_inputs if c["op"] == "attention" else _rotary_inputs)(c, seed)


def prepare(case, seed):
    return {"case": dict(case), **_inputs(case, seed)}


# ---- the plain forms ------------------------------------------------------------

def _allowed(c, s):
    """bool [batch or 1, 1, tq, tk]: which keys a query reads."""
    b, tq, tk = c["batch"], c["tq"], c["tk"]
    j = torch.arange(tk, device=DEV)
    ok = torch.ones(1, 1, tq, tk, dtype=torch.bool, device=DEV)
    if c["ragged"]:
        ok = ok & (j < s["lens"][:, None, None, None])
    if c["kind"] == "causal":
        at = s["first"][:, None, None, None] + torch.arange(tq, device=DEV)[:, None]
        ok = ok & (j <= at)
        if c["window"]:
            ok = ok & (j > at - c["window"])
    if "mask" in s:
        m = s["mask"]
        at = j[None, :] - s["first"][:, None]
        cols = at.clamp(0, m.shape[-1] - 1)[:, None, :].expand(b, tq, tk)
        seen = torch.gather(m, 2, cols) & (at < m.shape[-1])[:, None, :]
        ok = ok & (seen | (at < 0)[:, None, :])[:, None]
    return ok


def _plain_attention(c, s):
    h, kv, dt = c["heads"], c["kv"], TORCH[c["dtype"]]
    scale = c["d"] ** -0.5
    q = s["q"].float().transpose(1, 2).contiguous()
    k, v = (s[n].float().transpose(1, 2).repeat_interleave(h // kv, 1).contiguous() for n in ("k", "v"))
    if c["ragged"]:
        past = torch.arange(c["tk"], device=DEV) >= s["lens"][:, None]
        v.masked_fill_(past[:, None, :, None], 0.0)
        k.masked_fill_(past[:, None, :, None], 0.0)
    z = q @ k.transpose(2, 3).contiguous()
    z.mul_(scale).masked_fill_(~_allowed(c, s), -math.inf)
    out = {}
    if c["what"] == "vjp":
        lse = s["lse"]
        p = torch.exp(z.sub_(torch.where(torch.isinf(lse), 0.0, lse)[..., None]))
        o = s["o"].float().transpose(1, 2)
    else:
        m = z.amax(-1, keepdim=True)
        m = torch.where(torch.isinf(m), 0.0, m)
        p = torch.exp(z.sub_(m))
        total = p.sum(-1, keepdim=True)
        p.div_(torch.where(total == 0, 1.0, total))
        o = p @ v
        out = {"o": o.to(dt).transpose(1, 2).contiguous(), "lse": (m + torch.log(total))[..., 0].contiguous()}
    del z
    if c["what"] != "value":
        do = s["do"].float().transpose(1, 2).contiguous()
        delta = (do * o).sum(-1, keepdim=True)
        dv = p.transpose(2, 3).contiguous() @ do
        ds = do @ v.transpose(2, 3).contiguous()
        ds.sub_(delta).mul_(p)
        del p
        dq = (ds @ k) * scale
        dk = (ds.transpose(2, 3).contiguous() @ q) * scale
        b, tk, d = c["batch"], c["tk"], c["d"]
        dk, dv = (x.view(b, kv, h // kv, tk, d).sum(2) for x in (dk, dv))
        out.update((n, x.to(dt).transpose(1, 2).contiguous()) for n, x in (("dq", dq), ("dk", dk), ("dv", dv)))
    return out


def _pairs(c, x):
    """The two elements of each rotated pair: r and r + rotary / 2, or neighbours."""
    r = c["rotary"]
    return (x[..., 0:r:2], x[..., 1:r:2]) if c["even"] else (x[..., :r // 2], x[..., r // 2:r])


def _joined(c, a, b, rest):
    r = torch.stack((a, b), -1).flatten(-2) if c["even"] else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def _plain_rotary(c, s):
    dt, r = TORCH[c["dtype"]], c["rotary"]
    at = s["at"] if "at" in s else torch.arange(c["seq"], device=DEV)[None]
    angle = (at.double()[..., None] * s["freq"])[:, :, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = {}
    for n in ("q", "k"):
        x = s[n].float()
        u = x
        if c["norm"]:
            rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
            g = s["g" + n].float()
            xn = x * rstd
            u = xn * g
        a, b = _pairs(c, u)
        out["y" + n] = _joined(c, a * cos - b * sin, b * cos + a * sin, u[..., r:]).to(dt)
        if c["what"] == "step":
            dy = s["dy" + n].float()
            da, db = _pairs(c, dy)
            du = _joined(c, da * cos + db * sin, db * cos - da * sin, dy[..., r:])
            if c["norm"]:
                out["dg" + n] = (du * xn).sum((0, 1, 2)).to(dt)
                dn = du * g
                du = rstd * (dn - xn * (dn * xn).mean(-1, keepdim=True))
            out["d" + n] = du.to(dt)
    return out


# ---- the framework's calls --------------------------------------------------------

def _own_attention(c, s):
    from presk_amd import hip
    hip.init(0)
    b, h, tq = c["batch"], c["heads"], c["tq"]
    cols = s["mask"].shape[-1] if "mask" in s else 0
    op = hip.Attention(c["dtype"], b, h, c["kv"], tq, c["tk"], c["d"], causal=c["kind"] == "causal", window=c["window"], mask_cols=cols)
    places = {n: s[n] for n in ("lens", "first", "mask") if n in s}
    qkv = {n: s[n] for n in ("q", "k", "v")}
    out, fwd = {}, s
    if c["what"] != "vjp":
        fwd = out = {"o": torch.empty_like(s["q"]), "lse": torch.empty(b, h, tq, device=DEV)}
        work = torch.empty(op.workspace("value"), dtype=torch.uint8, device=DEV)
        op.value(**qkv, **places, o=out["o"], lse=out["lse"], work=work)
    if c["what"] != "value":
        grads = {"d" + n: torch.empty_like(x) for n, x in qkv.items()}
        work = torch.empty(op.workspace("vjp"), dtype=torch.uint8, device=DEV)
        op.vjp(**qkv, **places, o=fwd["o"], lse=fwd["lse"], do=s["do"], **grads, work=work)
        out = {**out, **grads}
    return out


def _own_rotary(c, s):
    from presk_amd import hip
    hip.init(0)
    op = hip.HeadRotary(c["dtype"], c["batch"], c["seq"], c["heads"], c["kv"], c["d"], rotary=c["rotary"], norm=c["norm"], eps=1e-6,
                        pairs="even" if c["even"] else "half")
    given = {n: s[n] for n in ("q", "k", "freq", "at", "gq", "gk") if n in s}
    out = {"yq": torch.empty_like(s["q"]), "yk": torch.empty_like(s["k"])}
    op.value(**given, **out)
    if c["what"] == "step":
        grads = {"d" + n: torch.empty_like(s[n]) for n in ("q", "k", "gq", "gk") if n in s}
        work = torch.empty(op.workspace("vjp"), dtype=torch.uint8, device=DEV)
        op.vjp(**given, dyq=s["dyq"], dyk=s["dyk"], **grads, work=work)
        out.update(grads)
    return out


def run(state):
    c = state["case"]
    if own:
        return (_own_attention if c["op"] == "attention" else _own_rotary)(c, state)
    return (_plain_attention if c["op"] == "attention" else _plain_rotary)(c, state)


# ---- what a pass cannot do without ----------------------------------------------

def _read_keys(c):
    """(query, key) pairs that a head reads, over the batch."""
    n = 0
    for length, first in zip(_lens(c), _first(c)):
        if c["kind"] == "causal":
            for lo in range(0, c["tq"]):
                last = min(length, first + lo + 1)
                n += max(0, last - (max(0, first + lo + 1 - c["window"]) if c["window"] else 0))
        elif c["kind"] == "documents":
            # four documents a sequence on average
            n += c["tq"] * c["tk"] // 8
        else:
            n += c["tq"] * length
    return n


def work(case):
    c, e = case, BYTES[case["dtype"]]
    if c["op"] == "rotary":
        n, heads = c["batch"] * c["seq"], c["heads"] + c["kv"]
        x = e * n * heads * c["d"]
        step = c["what"] == "step"
        return {"bytes": x * ((5 if c["norm"] else 4) if step else 2) + 8 * n, "flops": n * heads * c["d"] * (24 if step else 8)}
    q, kv = e * c["batch"] * c["tq"] * c["heads"] * c["d"], e * sum(_lens(c)) * c["kv"] * c["d"]
    mask = c["batch"] * c["tq"] * (c["tk"] if c["kind"] == "documents" else c["tq"] if c["kind"] == "tree" else 0)
    rows = 4 * c["batch"] * c["heads"] * c["tq"]
    moved = {"value": 2 * q + 2 * kv, "vjp": 4 * q + 4 * kv, "step": 4 * q + 4 * kv}[c["what"]]
    flops = {"value": 4, "vjp": 10, "step": 14}[c["what"]] * _read_keys(c) * c["heads"] * c["d"]
    return {"bytes": moved + mask + rows, "flops": flops}


# ---- the same outputs in float64 --------------------------------------------------

def exact(case, seed):
    """By torch's reverse mode in float64, from the definitions."""
    s = _inputs(case, seed)
    return (_exact_attention if case["op"] == "attention" else _exact_rotary)(case, s)


def _exact_attention(c, s):
    """One sequence and one key head at a time, the keys a query may read looked up
    from the definition.  The gradients are those of the weights that the given
    sums of exponentials stand for: of softmax where they are its own."""
    b, h, kv, tq, d = c["batch"], c["heads"], c["kv"], c["tq"], c["d"]
    per, lens, first = h // kv, _lens(c), _first(c)
    out = {}
    if c["what"] != "vjp":
        out = {"o": torch.zeros(b, tq, h, d, dtype=torch.float64, device=DEV),
               "lse": torch.full((b, h, tq), -math.inf, dtype=torch.float64, device=DEV)}
    if c["what"] != "value":
        out.update(("d" + n, torch.zeros(s[n].shape, dtype=torch.float64, device=DEV)) for n in ("q", "k", "v"))
    for i in range(b):
        n = lens[i]
        key, query = torch.arange(n, device=DEV)[None, :], torch.arange(tq, device=DEV)[:, None]
        hidden = torch.zeros(tq, n, dtype=torch.bool, device=DEV)
        if c["kind"] == "causal":
            hidden |= key > query + first[i]
            if c["window"]:
                hidden |= key + c["window"] <= query + first[i]
        elif c["kind"] == "documents":
            hidden |= ~s["mask"][i][:, :n]
        elif c["kind"] == "tree":
            hidden[:, first[i]:] |= ~s["mask"][i][:, :n - first[i]]
        nothing = hidden.all(1)
        for g in range(kv):
            k = s["k"][i, :n, g].double().requires_grad_()
            v = s["v"][i, :n, g].double().requires_grad_()
            for a in range(g * per, (g + 1) * per):
                q = s["q"][i, :, a].double().requires_grad_()
                z = (q @ k.t() / math.sqrt(d)).masked_fill(hidden, -math.inf)
                if c["what"] != "vjp":
                    z = z.masked_fill(nothing[:, None], 0.0)
                    o = torch.softmax(z, -1).masked_fill(nothing[:, None], 0.0) @ v
                    out["o"][i, :, a] = o.detach()
                    out["lse"][i, a] = torch.logsumexp(z.detach(), -1).masked_fill(nothing, -math.inf)
                    if c["what"] == "value":
                        continue
                    grads = torch.autograd.grad((o * s["do"][i, :, a].double()).sum(), (q, k, v))
                else:
                    lse, do = s["lse"][i, a].double(), s["do"][i, :, a].double()
                    p = torch.exp(z - lse.masked_fill(nothing, 0.0)[:, None])
                    delta = (do * s["o"][i, :, a].double()).sum(-1)
                    with torch.no_grad():
                        dz = p * (do @ v.t() - delta[:, None])
                        grads = (dz @ k / math.sqrt(d), dz.t() @ q / math.sqrt(d), p.t() @ do)
                out["dq"][i, :, a] = grads[0]
                out["dk"][i, :n, g] += grads[1]
                out["dv"][i, :n, g] += grads[2]
    return out


def _exact_rotary(c, s):
    """The rotation as a product of complex numbers."""
    n, r = c["seq"], c["rotary"]
    at = s["at"].double() if "at" in s else torch.arange(n, device=DEV).double().expand(c["batch"], n)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), at[:, :, None, None] * s["freq"])
    out = {}
    for name in ("q", "k"):
        x = s[name].double().requires_grad_()
        leaves, u = [x], x
        if c["norm"]:
            g = s["g" + name].double().requires_grad_()
            leaves.append(g)
            u = g * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
        head = u[..., :r].unflatten(-1, (r // 2, 2) if c["even"] else (2, r // 2))
        first, second = head.unbind(-1 if c["even"] else -2)
        z = torch.complex(first, second) * turn
        y = torch.stack((z.real, z.imag), -1 if c["even"] else -2).flatten(-2)
        y = torch.cat((y, u[..., r:]), -1)
        out["y" + name] = y.detach()
        if c["what"] == "step":
            grads = torch.autograd.grad((y * s["dy" + name].double()).sum(), leaves)
            if c["norm"]:
                out["dg" + name] = grads[1]
            out["d" + name] = grads[0]
    return out
