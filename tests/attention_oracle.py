"""Attention and head rotation from their definitions in float64 on the CPU, with
bounds of what rounding may add, for the tests of hip.Attention and
hip.HeadRotary."""
import math

import torch

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# half a step of a storage type, relative; and, of f16, half its smallest step
HALF = {t: torch.finfo(d).eps / 2 for t, d in TORCH.items()}
TINY = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}
F = 2.0 ** -24


def allowed(batch, tq, tk, causal=False, window=0, lens=None, first=None, mask=None):
    """bool [batch, tq, tk], one query and key at a time."""
    ok = torch.zeros(batch, tq, tk, dtype=torch.bool)
    cols = mask.shape[-1] if mask is not None else 0
    for b in range(batch):
        n = tk if lens is None else max(0, min(tk, int(lens[b])))
        f = int(first[b]) if first is not None else tk - (cols if mask is not None else tq)
        j = torch.arange(n)
        for i in range(tq):
            row = torch.ones(n, dtype=torch.bool)
            if causal:
                row = j <= f + i
                if window:
                    row = row & (j > f + i - window)
            if mask is not None:
                m = mask[b, i] if mask.ndim == 3 else mask[i]
                c = j - f
                row = (c < 0) | ((c < cols) & (m[c.clamp(0, cols - 1)] != 0))
            ok[b, i, :n] = row
    return ok


class Case:
    """q, k, v, do [batch, seq, heads, d] (storage types, CPU), as float64; the keys
    that no query reads are zeroed first, whatever they hold."""

    def __init__(self, dtype, q, k, v, ok, scale, do=None):
        self.dtype, self.scale = dtype, scale
        h, kv = q.shape[2], k.shape[2]
        self.per = h // kv
        unread = ~ok.any(1)                                      # [batch, tk]
        self.q = q.double().transpose(1, 2)
        zero = unread[:, :, None, None]
        self.k, self.v = (x.double().masked_fill(zero, 0.0).transpose(1, 2).repeat_interleave(self.per, 1) for x in (k, v))
        self.do = None if do is None else do.double().transpose(1, 2)
        self.ok = ok[:, None]
        self.s = (self.q @ self.k.transpose(2, 3)) * scale
        # the error of a score in f32, its products summed in any order
        self.es = F * (math.sqrt(q.shape[-1]) + 4) * scale * (self.q.abs() @ self.k.abs().transpose(2, 3)) + 4 * F * (self.s.abs() + 1)

    def value(self):
        z = self.s.masked_fill(~self.ok, -math.inf)
        none = ~self.ok.any(-1, keepdim=True)
        p = torch.softmax(z.masked_fill(none, 0.0), -1).masked_fill(~self.ok, 0.0)
        lse = torch.logsumexp(z, -1)
        o = p @ self.v
        u, f32 = HALF[self.dtype], self.dtype == "f32"
        worst = self.es.masked_fill(~self.ok, 0.0).amax(-1, keepdim=True)
        n = math.sqrt(z.shape[-1]) + 8
        weight = 0.0 if f32 else u
        eo = u * o.abs() + (p * (weight + worst + n * F + self.es)) @ self.v.abs() + worst * o.abs() + TINY[self.dtype] * (
            1 + self.ok.double() @ self.v.abs())
        el = worst[..., 0] + n * F + 4 * F * (lse.abs() + 1)
        return {"o": (o.transpose(1, 2), eo.transpose(1, 2) * 1.02 + 1e-30), "lse": (lse, el)}

    def vjp(self, o, lse):
        """From the forward's o and lse as they are stored."""
        o, lse = o.double().transpose(1, 2), lse.double()
        u, f32 = HALF[self.dtype], self.dtype == "f32"
        weight = 0.0 if f32 else u
        p = torch.exp(self.s - torch.where(torch.isinf(lse), 0.0, lse)[..., None]).masked_fill(~self.ok, 0.0)
        ep = p * (self.es + 4 * F * (lse.abs().nan_to_num(0.0, 0.0, 0.0)[..., None] + 1)) + TINY[self.dtype] / 256
        dp = self.do @ self.v.transpose(2, 3)
        delta = (self.do * o).sum(-1, keepdim=True)
        big = self.do.abs() @ self.v.abs().transpose(2, 3) + (self.do * o).abs().sum(-1, keepdim=True)
        ds = p * (dp - delta)
        n = math.sqrt(self.q.shape[-1]) + 8
        eds = (ep * (dp - delta).abs() + p * n * F * big + weight * ds.abs() + TINY[self.dtype]).masked_fill(~self.ok, 0.0)
        ep = (ep + weight * p).masked_fill(~self.ok, 0.0)
        out = {}
        m = math.sqrt(max(self.s.shape[-2:])) + 8

        def done(name, x, e, grouped):
            if grouped:
                x, e = (y.unflatten(1, (-1, self.per)).sum(2) for y in (x, e))
            e = e + u * x.abs() + TINY[self.dtype]
            out[name] = (x.transpose(1, 2), e.transpose(1, 2) * 1.02 + 1e-30)

        def product(w, ew, x):
            return w @ x, ew @ x.abs() + m * F * (w.abs() @ x.abs())

        dq, eq = product(ds, eds, self.k)
        done("dq", dq * self.scale, eq * self.scale, False)
        dk, ek = product(ds.transpose(2, 3), eds.transpose(2, 3), self.q)
        done("dk", dk * self.scale, ek * self.scale, True)
        dv, ev = product(p.transpose(2, 3), ep.transpose(2, 3), self.do)
        done("dv", dv, ev, True)
        return out


def check(name, got, want, bound):
    """Every element within its bound; infinities and NaN where they are."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite), f"{name}: finite where it should not be, or the reverse"
    same = ~finite
    assert torch.equal(got[same].nan_to_num(7.0), want[same].nan_to_num(7.0)), name
    over = ((got - want).abs() / bound)[finite]
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times its bound"
    return worst


def rotary(dtype, x, g, freq, at, rot, norm, eps, even, dy=None):
    """(y, its bound) or, with dy, {"dx", "dg"} of one tensor's heads [batch, seq,
    heads, d] in float64."""
    u = HALF[dtype]
    x = x.double()
    d = x.shape[-1]
    angle = at.double()[:, :, None, None] * freq.double()
    c, s = torch.cos(angle), torch.sin(angle)
    ea = 2.0 ** -52 * angle.abs() * 2 + 4 * F            # the angle's error, and its cosine's

    def parts(z):
        return (z[..., 0:rot:2], z[..., 1:rot:2]) if even else (z[..., :rot // 2], z[..., rot // 2:rot])

    def join(a, b, z):
        r = torch.stack((a, b), -1).flatten(-2) if even else torch.cat((a, b), -1)
        return torch.cat((r, z[..., rot:]), -1)

    def turn(z, sign):
        a, b = parts(z)
        return join(a * c - sign * b * s, b * c + sign * a * s, z)

    def spread(e, z):
        """The turn's error where z's elements have errors e."""
        (a, b), (za, zb) = parts(e), parts(z.abs())
        r = (a + b) + (za + zb) * (ea + 3 * F)
        return join(r, r, e)

    rstd = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) if norm else torch.ones_like(x[..., :1])
    n = x * rstd
    gd = torch.ones(d, dtype=torch.float64) if g is None else g.double()
    rel = (math.sqrt(d) + 8) * F if norm else 0.0
    if dy is None:
        v = n * gd
        y = turn(v, 1.0)
        return y, (u * y.abs() + spread(v.abs() * rel, v)) * 1.02 + TINY[dtype] + 1e-30
    dy = dy.double()
    du = turn(dy, -1.0)
    edu = spread(torch.zeros_like(dy), dy)
    out = {}
    if not norm:
        out["dx"] = (du, (u * du.abs() + edu) * 1.02 + TINY[dtype] + 1e-30)
        return out
    count = math.sqrt(x.shape[0] * x.shape[1] * x.shape[2]) + 16
    dg = (du * n).sum((0, 1, 2))
    edg = ((edu + du.abs() * (rel + 2 * F)) * n.abs()).sum((0, 1, 2)) + count * F * (du * n).abs().sum((0, 1, 2))
    out["dg"] = (dg, (u * dg.abs() + edg) * 1.02 + TINY[dtype] + 1e-30)
    dn = du * gd
    mean = (dn * n).mean(-1, keepdim=True)
    dx = rstd * (dn - n * mean)
    edn = edu * gd.abs() + dn.abs() * 2 * F
    em = (edn * n.abs() + (dn * n).abs() * (2 * rel + 4 * F)).mean(-1, keepdim=True) + rel * (dn * n).abs().mean(-1, keepdim=True)
    e = rstd * (edn + n.abs() * em + (n * mean).abs() * 2 * rel + 4 * F * (dn.abs() + (n * mean).abs())) + dx.abs() * rel
    out["dx"] = (dx, (u * dx.abs() + e) * 1.02 + TINY[dtype] + 1e-30)
    return out
