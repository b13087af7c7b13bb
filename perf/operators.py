"""The losses of a large vocabulary: what is measured of them.

Three operators.  The head's loss: the softmax cross entropy of x . w against
one index a row without the [rows, vocab] logits in memory, and its gradients
(`hip.HeadLoss`).  Distillation: the divergence of a student's given logits
from the softmax of a teacher's top logits, and its gradient (`hip.Distill`).
The head's distillation: the same divergence through x . w (`hip.HeadLoss`
with `top`).

`own` false: the operators written out in elementary torch operations in f32.
`own` true: the calls a program makes of the framework.  Inputs, in either
case, are tensors on the GPU in their storage type; outputs and workspace are
taken anew in each call.

Sizes are the configurations' (the course GPT's 16384 x 384 x 65, the
Llama-shaped head of 4096 x 32000) and generic ones around them.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the course GPT's head and loss over its 65 characters: the mean loss
        # of a training step and its gradients
        {"name": "head-course-step-f32", "op": "head", "what": "step", "dtype": "f32", "rows": 16384, "d": 384,
         "vocab": 65, "tied": False, "top": 0, "t": 1.0},
        # the same head scoring one sequence of 256: the smallest call
        {"name": "head-course-score-f32", "op": "head", "what": "value", "dtype": "f32", "rows": 256, "d": 384,
         "vocab": 65, "tied": False, "top": 0, "t": 1.0},
        # the Llama-shaped head in a training step over 8192 tokens: the largest
        {"name": "head-wide-step-bf16", "op": "head", "what": "step", "dtype": "bf16", "rows": 8192, "d": 4096,
         "vocab": 32000, "tied": False, "top": 0, "t": 1.0},
        # the same head scoring a prompt of 2048 tokens (perplexity, reranking)
        {"name": "head-wide-score-bf16", "op": "head", "what": "value", "dtype": "bf16", "rows": 2048, "d": 4096,
         "vocab": 32000, "tied": False, "top": 0, "t": 1.0},
        # scoring the next token of eight sequences: the weight's bytes bound it
        {"name": "head-few-rows-bf16", "op": "head", "what": "value", "dtype": "bf16", "rows": 8, "d": 4096,
         "vocab": 32000, "tied": False, "top": 0, "t": 1.0},
        # sizes that are no multiple of anything, a scaled cotangent a row, as
        # reverse mode calls it with the forward's sums kept
        {"name": "head-odd-vjp-f16", "op": "head", "what": "vjp", "dtype": "f16", "rows": 1999, "d": 1021,
         "vocab": 50257, "tied": False, "top": 0, "t": 1.0},
        # a head tied to the embedding ([vocab, model]), in f32
        {"name": "head-tied-step-f32", "op": "head", "what": "step", "dtype": "f32", "rows": 2048, "d": 768,
         "vocab": 32000, "tied": True, "top": 0, "t": 1.0},
        # a student's head trained on the 64 largest logits of a teacher
        {"name": "head-distill-step-bf16", "op": "head", "what": "step", "dtype": "bf16", "rows": 4096, "d": 4096,
         "vocab": 32000, "tied": False, "top": 64, "t": 2.0},
        # a small tied student with odd sizes
        {"name": "head-distill-odd-f16", "op": "head", "what": "step", "dtype": "f16", "rows": 777, "d": 500,
         "vocab": 10007, "tied": True, "top": 20, "t": 1.5},
        # distillation of logits that the program has anyway, value and gradient
        {"name": "distill-step-bf16", "op": "distill", "what": "step", "dtype": "bf16", "rows": 8192, "vocab": 32000,
         "top": 64, "t": 2.0},
        # a few rows of a large vocabulary, the value alone
        {"name": "distill-few-rows-f32", "op": "distill", "what": "value", "dtype": "f32", "rows": 64, "vocab": 50257,
         "top": 20, "t": 1.0},
        # odd rows of an odd vocabulary, value and gradient
        {"name": "distill-odd-f16", "op": "distill", "what": "step", "dtype": "f16", "rows": 2047, "vocab": 50257,
         "top": 100, "t": 3.0},
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
    c = {"op": rng.choice(["head", "head", "distill"]), "what": rng.choice(["value", "step", "step", "vjp"]),
         "dtype": rng.choice(["f32", "bf16", "bf16", "f16"])}
    while True:
        c["rows"], c["vocab"] = _size(rng, 1, 16384), _size(rng, 33, 131072)
        if c["op"] == "head":
            c["d"] = _size(rng, 32, 4096)
            c["tied"] = rng.random() < 0.5
        most = 1.0e12 if c["dtype"] != "f32" else 1.0e11
        if c["rows"] * c["vocab"] <= 2.6e8 and c["rows"] * c["vocab"] * c.get("d", 1) <= most and c.get("d", 1) * c["vocab"] <= 1.4e8:
            break
    soft = c["op"] == "distill" or rng.random() < 0.4
    c["top"] = min(c["vocab"], _log(rng, 1, 256)) if soft else 0
    c["t"] = rng.choice([1.0, 1.5, 2.0, 4.0]) if soft else 1.0
    return c


# ---- inputs -------------------------------------------------------------------

def _inputs(c, seed):
    """Every input of a case: x ~ N(0, 1) and weights that make the logits
    ~ N(0, 2.5); logits given as such; indices uniform, one row in sixteen
    padding (-1); a teacher's slots at distinct indices, their logits falling
    from the first on, one slot in sixteen unused."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    n, v, k, dt = c["rows"], c["vocab"], c["top"], TORCH[c["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * std).to(dt)

    s = {}
    if c["op"] == "head":
        d = c["d"]
        s["x"] = normal(n, d)
        s["w"] = normal(*((v, d) if c["tied"] else (d, v)), std=2.5 * d ** -0.5)
    else:
        s["x"] = normal(n, v, std=2.5)
    padded = torch.rand(n, device=DEV, generator=g) < 1 / 16
    first = torch.randint(0, v, (n,), device=DEV, generator=g)
    if k:
        step = torch.arange(k, device=DEV) * (v // k)
        index = (first[:, None] + step) % v
        unused = torch.rand(n, k, device=DEV, generator=g) < 1 / 16
        s["index"] = index.masked_fill(unused | padded[:, None], -1).contiguous()
        fall = 6.0 * torch.log1p(torch.arange(k, device=DEV) * 1.0) / math.log(1.0 + max(k, 2))
        s["teacher"] = (12.0 - fall + torch.randn(n, k, device=DEV, generator=g) * 0.7).to(dt)
    else:
        s["index"] = first.masked_fill(padded, -1)
    if c["what"] == "vjp":
        # the forward's sums
        s["lse"] = torch.logsumexp(_logits(c, s) / c["t"], -1)
    if c["what"] == "vjp" or (c["what"] == "step" and c["dtype"] == "f16"):
        # a cotangent a row, at the loss scale that f16 gradients need (in
        # the other types a step takes the mean's)
        s["ct"] = min(1024.0, 65536.0 / n) * (1.0 + 0.25 * torch.randn(n, device=DEV, generator=g))
    return s


def _logits(c, s):
    """The student's logits in f32."""
    x = s["x"].float()
    if c["op"] != "head":
        return x
    w = s["w"].float()
    return x @ (w.t() if c["tied"] else w)


def prepare(case, seed):
    return {"case": dict(case), **_inputs(case, seed)}


# ---- the plain form -------------------------------------------------------------

def _plain(c, s):
    n, k, t, dt = c["rows"], c["top"], c["t"], TORCH[c["dtype"]]
    z = _logits(c, s) / t
    at = s["index"].reshape(n, -1)
    used = at >= 0
    if k:
        teacher = s["teacher"].float() / t
        used = used & (teacher > -math.inf)
        top = teacher.masked_fill(~used, -math.inf).amax(-1, keepdim=True)
        e = torch.exp(teacher - torch.where(torch.isinf(top), 0.0, top)).masked_fill(~used, 0.0)
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total == 0, 1.0, total)
        logp = teacher - top - torch.log(total)
    else:
        p, logp = used.float(), torch.zeros(n, 1, device=DEV)
    at = at.clamp_min(0)
    counted = used.any(-1)
    count = counted.sum().float().clamp_min(1.0)
    out = {}
    if c["what"] == "vjp":
        lse = s["lse"]
    else:
        m = z.amax(-1)
        lse = m + torch.log(torch.exp(z - m[:, None]).sum(-1))
        term = p * (logp - z.gather(1, at) + lse[:, None])
        loss = t * t * torch.where(p > 0, term, 0.0).sum(-1)
        out = {"loss": loss, "lse": lse, "mean": loss.sum() / count}
    if c["what"] != "value":
        coef = t * s["ct"] if "ct" in s else t / count
        dz = torch.exp(z - lse[:, None])
        dz.scatter_add_(1, at, -p)
        dz = dz * (coef * counted)[:, None]
        if c["op"] == "head":
            w, x = s["w"].float(), s["x"].float()
            out["dx"] = (dz @ (w if c["tied"] else w.t())).to(dt)
            out["dw"] = (dz.t() @ x if c["tied"] else x.t() @ dz).to(dt)
        else:
            out["dx"] = dz.to(dt)
    return out


# ---- the framework's calls --------------------------------------------------------

def _own(c, s):
    from presk_amd import hip
    n, what, x = c["rows"], c["what"], s["x"]
    hip.init(0)
    if c["op"] == "head":
        op = hip.HeadLoss(c["dtype"], n, c["d"], c["vocab"], tied=c["tied"], top=c["top"], temperature=c["t"])
    else:
        op = hip.Distill(c["dtype"], n, c["vocab"], c["top"], temperature=c["t"])
    bufs = {name: s[name] for name in ("x", "w", "index", "teacher", "lse", "ct") if name in s}
    out = {}
    if what != "vjp":
        out = {"loss": torch.empty(n, device=DEV), "lse": torch.empty(n, device=DEV), "mean": torch.empty(2, device=DEV)}
    if what != "value":
        out["dx"] = torch.empty_like(x)
        if c["op"] == "head":
            out["dw"] = torch.empty_like(s["w"])
    run = {"value": op.value, "vjp": op.vjp, "step": op.value_and_grad}[what]
    work = torch.empty(op.workspace(what), dtype=torch.uint8, device=DEV)
    run(**{**bufs, **out}, work=work, stream=torch.cuda.current_stream().cuda_stream)
    if "mean" in out:
        out["mean"] = out["mean"][0]
    return out


def run(state):
    return _own(state["case"], state) if own else _plain(state["case"], state)


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    c, e, n, v = case, BYTES[case["dtype"]], case["rows"], case["vocab"]
    grad = c["what"] != "value"
    small = n * (8 * max(c["top"], 1) + e * c["top"] + 8)
    if c["op"] == "distill":
        return {"bytes": e * n * v * (2 if grad else 1) + small, "flops": n * v * (8 if grad else 4)}
    d = c["d"]
    return {"bytes": e * (n * d + d * v) * (2 if grad else 1) + small, "flops": (6 if grad else 2) * n * d * v}


# ---- the same outputs in float64 --------------------------------------------------

def exact(case, seed):
    """By torch's reverse mode in float64, from the definition: a row's loss is
    T^2 times the divergence of softmax(z / T) from the target distribution."""
    c = case
    s = _inputs(c, seed)
    n, t = c["rows"], c["t"]
    leaves = [s["x"].double().requires_grad_()]
    z = leaves[0]
    if c["op"] == "head":
        w = s["w"].double().requires_grad_()
        leaves.append(w)
        z = z @ (w.t() if c["tied"] else w)
    logq = torch.log_softmax(z / t, -1)
    target = torch.zeros(n, c["vocab"], dtype=torch.float64, device=DEV)
    at = s["index"].reshape(n, -1)
    if c["top"]:
        p = torch.softmax((s["teacher"].double() / t).masked_fill(at < 0, -math.inf), -1).nan_to_num(0.0)
    else:
        p = (at >= 0).double()
    target.scatter_add_(1, at.clamp_min(0), p)
    counted = (at >= 0).any(-1)
    loss = t * t * (torch.special.xlogy(p, p).sum(-1) - (target * logq).sum(-1))
    mean = loss.sum() / counted.sum().clamp_min(1)
    out = {}
    if c["what"] != "vjp":
        out = {"loss": loss.detach(), "lse": torch.logsumexp(z.detach() / t, -1), "mean": mean.detach()}
    if c["what"] != "value":
        grads = torch.autograd.grad((loss * s["ct"].double()).sum() if "ct" in s else mean, leaves)
        out.update(zip(("dx", "dw"), grads))
    return out
