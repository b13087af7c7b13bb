"""The losses of a large vocabulary on the device against float64.

The reference is plain torch in float64, on the inputs as stored.  The bounds
follow the kernels' arithmetic, element by element:

  logits of a head  dz: 2 gamma_D sum |x w|, gamma_D = D 2^-24 (f32 sums of D
                    exact products in any order; f32 operands split in three
                    parts stay below it);
  u = z / T         du = dz / T + |u| 2^-22 (the factor's rounding and the fma's,
                    each half a step, and one more for the maximum's product);
  lse               the largest du of the row, V terms each within 2^-22 of its
                    exponential (v_exp_f32 1 ulp, its sum's roundings below
                    2^-24 a level of adding), so eL = max du + (8 + V / 256) 2^-24
                    + |lse| 2^-22;
  loss              T^2 (max du + eL + (k + 8) 2^-24 sum p |log p - u + lse|)
                    + half a step of the stored f32, the teacher's weights being
                    within (k + 8 + |u_t|) 2^-23 of theirs;
  cotangent         dq = q (exp(du + eL) - 1) + the weights' error, then |ct| T
                    times that, and one rounding to the storage type (r: half a
                    step) where it is stored, in a head's 16-bit products and in
                    an output; v_exp_f32 gives 0 below 2^-126, and a product
                    with ct T may end below it and count as 0 to the matrix
                    cores, so 2^-126 (1 + |ct| T) stands beside that: with
                    logits of hundreds whole columns have no larger q;
  dx, dw            sums of |d cotangent| |w| over the products, gamma of the sum's
                    length times sum |cotangent| |w|, and the output's rounding.
The bounds are sums of every error at its largest.
"""
import math

import pytest

torch = pytest.importorskip("torch")

from presk_amd import hip  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# the smallest step a stored value can be off by (subnormals: half of it)
TINY = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}
E24 = 2.0 ** -24


@pytest.fixture(autouse=True)
def device():
    hip.init(0)
    yield
    torch.cuda.synchronize()


class Guarded:
    """A buffer with 64 bytes of a pattern behind it (and, unless told
    otherwise, in it): nothing may be written past its end."""

    def __init__(self, *shape, dtype, fill=0xAB):
        n = math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
        self.raw = torch.full((n + 64,), fill, dtype=torch.uint8, device=DEV)
        self.raw[n:] = 0xCD
        self.t = self.raw[:n].view(dtype).reshape(shape)

    def intact(self):
        return bool((self.raw[-64:] == 0xCD).all())


class Case:
    def __init__(self, dtype, rows, vocab, d=0, tied=False, top=0, t=1.0, seed=0, pad=True, ct=None, std=2.5):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.dtype, self.rows, self.vocab, self.d, self.tied, self.top, self.t = dtype, rows, vocab, d, tied, top, t

        def normal(*shape, std=1.0):
            return (torch.randn(*shape, device=DEV, generator=g) * std).to(T[dtype])

        if d:
            self.x = normal(rows, d)
            self.w = normal(*((vocab, d) if tied else (d, vocab)), std=std * d ** -0.5)
        else:
            self.x, self.w = normal(rows, vocab, std=std), None
        k = max(top, 1)
        self.index = torch.randint(0, vocab, (rows, k), device=DEV, generator=g)
        self.teacher = None
        if top:
            self.teacher = normal(rows, top, std=2.0)
            if pad:
                self.index[torch.rand(rows, top, device=DEV, generator=g) < 0.2] = -1
        else:
            self.index = self.index[:, 0].contiguous()
        if pad and rows > 2:
            self.index[1::5] = -7
        scale = min(1024.0, 65536.0 / max(rows, 1)) if dtype == "f16" else 1.0
        self.ct = None
        if ct or (ct is None and dtype == "f16"):
            self.ct = scale * (1.0 + torch.rand(rows, device=DEV, generator=g))

    def op(self):
        if self.d:
            return hip.HeadLoss(self.dtype, self.rows, self.d, self.vocab, tied=self.tied, top=self.top, temperature=self.t)
        return hip.Distill(self.dtype, self.rows, self.vocab, self.top, temperature=self.t)

    def ins(self):
        b = {"x": self.x, "index": self.index, "teacher": self.teacher}
        return {**b, "w": self.w} if self.d else b

    def run(self, kind="step", dx=True, dw=True, stream=None, lse=None, mean=None, flag=None):
        """One call over guarded outputs and a guarded, poisoned workspace."""
        op, n = self.op(), self.rows
        out = {}
        if kind != "vjp":
            out = {m: Guarded(s, dtype=torch.float32) for m, s in (("loss", n), ("lse", n), ("mean", 2))}
        if kind != "value":
            if dx:
                out["dx"] = Guarded(*self.x.shape, dtype=T[self.dtype])
            if dw and self.d:
                out["dw"] = Guarded(*self.w.shape, dtype=T[self.dtype])
        work = Guarded(op.workspace(kind, "dx" in out, "dw" in out), dtype=torch.uint8, fill=0xFF)
        bufs = {m: b.t for m, b in out.items()}
        if kind == "vjp":
            bufs["lse"] = lse
            if self.ct is None:
                bufs["mean"] = mean
        if kind != "value":
            bufs["ct"] = self.ct
            bufs["flag"] = flag
        f = {"value": op.value, "vjp": op.vjp, "step": op.value_and_grad}[kind]
        torch.cuda.synchronize()
        f(**self.ins(), **bufs, work=work.t, stream=stream)
        torch.cuda.synchronize()
        for m, b in out.items():
            assert b.intact(), m
        assert work.intact(), "workspace"
        return {m: b.t for m, b in out.items()}

    # the definition and its bounds, in float64
    def exact(self):
        n, t, v = self.rows, self.t, self.vocab
        x = self.x.double()
        w = None
        if self.d:
            w = (self.w.t() if self.tied else self.w).double()
            z, dz = x @ w, 2 * self.d * E24 * (x.abs() @ w.abs())
        else:
            z, dz = x, torch.zeros_like(x)
        u = z / t
        du = dz / t + u.abs() * 4 * E24
        at = self.index.reshape(n, -1)
        used = at >= 0
        if self.top:
            tu = self.teacher.double() / t
            used = used & (tu > -math.inf)
            p = torch.softmax(tu.masked_fill(~used, -math.inf), -1).nan_to_num(0.0)
            ep = torch.where(p > 0, p * (self.top + 8 + tu.abs()) * 2 * E24, 0.0)
        else:
            p, ep = used.double(), torch.zeros(n, 1, dtype=torch.float64, device=DEV)
        counted = used.any(-1)
        at = at.clamp_min(0)
        lse = torch.logsumexp(u, -1)
        mdu = du.amax(-1)
        el = mdu + (8 + v / 256) * E24 + lse.abs() * 4 * E24
        logp = torch.where(p > 0, torch.log(p.clamp_min(1e-300)), 0.0)
        term = logp - u.gather(1, at) + lse[:, None]
        loss = t * t * (p * term).sum(-1)
        parts = (p * (logp.abs() + u.gather(1, at).abs() + lse.abs()[:, None])).sum(-1)
        eloss = t * t * (mdu + el + (p.shape[1] + 8) * E24 * parts + (ep * (1 + term.abs())).sum(-1)) + loss.abs() * E24
        count = counted.sum().double()
        r = {"loss": loss, "lse": lse, "mean": loss.sum() / count.clamp_min(1), "count": count}
        e = {"loss": eloss, "lse": el, "mean": (eloss.sum() + (loss.abs() * E24).sum()) / count.clamp_min(1) + 1e-30}
        ct = self.ct.double() if self.ct is not None else torch.ones(n, dtype=torch.float64, device=DEV) / count.clamp_min(1)
        coef = torch.where(counted, ct * t, 0.0)[:, None]
        q = torch.exp(u - lse[:, None])
        eg = q * torch.expm1(du + el[:, None] + 4 * E24) + q * 2 * E24
        g = q.scatter_add(1, at, -p)
        eg = (eg.scatter_add(1, at, ep + p * 2 * E24) + g.abs() * 4 * E24) * coef
        eg = eg + 2.0 ** -126 * (1.0 + coef)
        g = g * coef
        half, tiny = HALF[self.dtype], TINY[self.dtype]
        if not self.d:
            r["dx"], e["dx"] = g, eg + half * (g.abs() + eg) + tiny
            return r, e
        if self.dtype != "f32":
            # the cotangent in 16 bits (in f16 after a power of two that
            # leaves its largest at 2^14 or more: a step below 2^-38 of that)
            eg = eg + half * (g.abs() + eg) + (2.0 ** -38 * coef.amax() if self.dtype == "f16" else 0.0)
        for name, a, ea, b in (("dx", g, eg, w.t().contiguous()), ("dw", x.t().contiguous(), None, g)):
            if name == "dx":
                y, ey = a @ b, ea @ b.abs() + 2 * self.vocab * E24 * (a.abs() @ b.abs())
            else:
                y, ey = a @ b, a.abs() @ eg + 2 * n * E24 * (a.abs() @ b.abs())
            ey = ey + half * (y.abs() + ey) + tiny
            if name == "dw" and self.tied:
                y, ey = y.t(), ey.t()
            r[name], e[name] = y, ey
        return r, e

    def check(self, got, names=None):
        r, e = self.exact()
        for m in names or got:
            x = got[m].double()
            if m == "mean":
                assert float(x[1]) == float(r["count"]), m
                x = x[0]
            off = (x - r[m]).abs()
            bad = ~(off <= e[m])
            assert not bool(bad.any()), (m, int(bad.sum()), float((off / e[m]).nan_to_num(math.inf).max()), self.__dict__.get("name"))


def same(a, b, what):
    assert bool(torch.equal(a, b)), (what, int((a != b).sum()))


def name(c):
    return "-".join(str(x) for x in c)


# ---- a head, each type, layout and kind of target ----------------------------------

HEADS = [(dt, *s) for dt in ("f32", "bf16", "f16") for s in [
    # rows, d, vocab, tied, top, T
    (1, 1, 1, False, 0, 1.0), (1, 64, 2, False, 0, 1.0), (3, 8, 8, True, 0, 1.0), (5, 7, 65, False, 0, 1.0),
    (64, 64, 128, False, 0, 1.0), (64, 64, 128, True, 0, 1.0), (65, 72, 129, False, 0, 1.0), (129, 63, 257, True, 0, 1.0),
    (255, 65, 255, False, 0, 1.0), (257, 128, 1000, False, 0, 1.0), (257, 130, 1001, True, 0, 1.0), (300, 500, 2048, True, 0, 1.0),
    (7, 200, 5003, False, 0, 1.0), (2, 96, 50257, True, 0, 1.0), (700, 40, 33, False, 0, 1.0),
    (1, 16, 5, False, 3, 2.0), (33, 64, 640, False, 1, 1.0), (66, 100, 700, True, 4, 1.5), (130, 72, 1003, False, 5, 2.0),
    (140, 64, 4096, False, 64, 4.0), (20, 33, 65, True, 65, 1.0), (9, 64, 3001, False, 300, 0.5), (3, 40, 2000, True, 1024, 2.0),
    (520, 256, 3333, False, 20, 1.0),
]]


@pytest.mark.parametrize("c", HEADS, ids=name)
def test_head(c):
    dt, rows, d, vocab, tied, top, t = c
    k = Case(dt, rows, vocab, d=d, tied=tied, top=top, t=t, seed=rows + vocab)
    k.check(k.run("step"))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("top", [0, 6])
def test_head_value_then_vjp_equals_both(dt, tied, top):
    """The value alone, then the gradient from its lse, for the mean and for a
    cotangent a row, and one call that does both (of one piece, which adds a
    row's terms in another order), with either gradient left out (its products'
    sums may be cut elsewhere)."""
    for ct in (True, False):
        k = Case(dt, 200, 1100, d=96, tied=tied, top=top, seed=3, ct=ct)
        v = k.run("value")
        for got in (k.run("step"), v, k.run("vjp", lse=v["lse"], mean=v["mean"]), k.run("step", dw=False), k.run("step", dx=False)):
            k.check(got)


def test_head_value_and_grad_of_several_pieces_is_value_then_vjp():
    """16-bit storage, more logits than are kept: the same launches, the same bits."""
    k = Case("bf16", 40000, 28000, d=64, seed=3, ct=False)
    both, v = k.run("step"), k.run("value")
    g = k.run("vjp", lse=v["lse"], mean=v["mean"])
    for m, x in {**v, **g}.items():
        same(x, both[m], m)


# rows that make the vocabulary several pieces, the last one ragged
@pytest.mark.parametrize("dt,rows,d,vocab,tied,top", [
    ("bf16", 40000, 72, 3000, False, 0), ("f16", 40000, 64, 3001, True, 0), ("bf16", 30003, 40, 4097, True, 5),
    ("f32", 20000, 48, 4001, False, 0), ("f32", 20000, 40, 3900, True, 3),
], ids=str)
def test_head_in_several_pieces(dt, rows, d, vocab, tied, top):
    k = Case(dt, rows, vocab, d=d, tied=tied, top=top, seed=5)
    v = k.run("value")
    for got in (k.run("step"), v, k.run("vjp", lse=v["lse"], mean=v["mean"])):
        k.check(got)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_head_of_nearly_all_the_logits_that_are_kept(dt):
    """4.2 GB of f32 logits, whose byte offsets pass 2^31, in one piece."""
    k = Case(dt, 40000, 26000, d=72, seed=9)
    k.check(k.run("step"))


# more columns than a workgroup's registers hold of a row
@pytest.mark.parametrize("tied,top", [(False, 0), (True, 0), (True, 7), (False, 1000)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_head_of_long_rows(dt, tied, top):
    for rows in (3, 70):
        k = Case(dt, rows, 66001 if tied else 70003, d=40, tied=tied, top=top, seed=8)
        k.check(k.run("step"))


@pytest.mark.parametrize("dt,rows,d,vocab,tied", [("bf16", 2048, 1024, 8192, False), ("f16", 1999, 1021, 9001, False),
                                                  ("bf16", 2050, 1024, 8200, True), ("f32", 1024, 768, 8000, True)], ids=str)
def test_head_large(dt, rows, d, vocab, tied):
    k = Case(dt, rows, vocab, d=d, tied=tied, seed=6)
    k.check(k.run("step"))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_head_rows_that_do_not_count(dt):
    """All rows padding: a mean of 0 over 0 rows, losses and gradients 0; no
    rows at all: the same, and dw zeroed."""
    k = Case(dt, 50, 300, d=64, seed=1)
    k.index[:] = -1
    got = k.run("step")
    assert not got["loss"].any() and not got["mean"].any() and not got["dx"].any() and not got["dw"].any()
    r, e = k.exact()
    assert bool(((got["lse"].double() - r["lse"]).abs() <= e["lse"]).all())
    k = Case(dt, 0, 300, d=64, seed=1)
    got = k.run("step")
    assert not got["mean"].any() and not got["dw"].any()


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_head_index_outside_the_vocabulary(dt, top):
    """It makes its row's loss and cotangent NaN, and no other's."""
    k = Case(dt, 40, 300, d=64, top=top, seed=2, pad=False)
    good = k.run("step", dw=False)
    (k.index if not top else k.index[:, 1])[7] = 300
    (k.index if not top else k.index[:, 0])[9] = 1 << 40
    got = k.run("step")
    rows = torch.zeros(40, dtype=torch.bool, device=DEV)
    rows[7] = rows[9] = True
    assert bool(got["loss"][rows].isnan().all()) and bool(got["dx"][rows].isnan().all()) and bool(got["dw"].isnan().all())
    assert torch.equal(got["loss"][~rows], good["loss"][~rows]) and torch.equal(got["dx"][~rows], good["dx"][~rows])
    assert torch.equal(got["lse"], good["lse"]) and bool(got["mean"][0].isnan()) and float(got["mean"][1]) == 40.0


def test_head_large_logits():
    """Logits of hundreds: a sum that only the largest reaches."""
    for dt in ("f32", "bf16"):
        k = Case(dt, 100, 1000, d=64, seed=8, std=200.0)
        k.check(k.run("step"))


def test_head_f16_cotangents_past_its_range():
    """Cotangents of 1e6 a row: the piece's are scaled into f16, and outputs
    past its largest value are infinite and set the flag; those of 1e-6 reach dw
    where f16 could not hold them before the product."""
    k = Case("f16", 64, 256, d=64, seed=4, ct=True)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    k.ct[:] = 1e6
    got = k.run("step", flag=flag)
    assert int(flag) == 1 and bool(got["dx"].isinf().any())
    flag.zero_()
    k.ct[:] = 1e-6
    k.check(k.run("step", flag=flag))
    assert int(flag) == 0
    k.ct[:] = 0.0
    got = k.run("step", flag=flag)
    assert not got["dx"].any() and not got["dw"].any() and int(flag) == 0


# ---- given logits ------------------------------------------------------------------

GIVEN = [(dt, *s) for dt in ("f32", "bf16", "f16") for s in [
    (1, 1, 1, 1.0), (1, 2, 1, 2.0), (3, 7, 7, 1.0), (4, 64, 3, 1.0), (5, 65, 65, 3.0), (300, 257, 5, 1.0), (33, 1000, 64, 2.0),
    (33, 1024, 20, 1.0), (33, 1025, 65, 2.0), (9, 8191, 100, 1.0), (7, 8193, 1000, 0.7), (1100, 2049, 1024, 1.0), (2, 32000, 64, 4.0),
    (3, 32769, 2, 1.0), (2, 50257, 100, 1.0), (2, 65537, 33, 1.0), (1, 131072, 64, 1.0), (2, 131080, 64, 2.0), (1, 200003, 7, 1.0),
]]


@pytest.mark.parametrize("c", GIVEN, ids=name)
def test_distill(c):
    dt, rows, vocab, top, t = c
    k = Case(dt, rows, vocab, top=top, t=t, seed=rows + vocab)
    got = k.run("step")
    k.check(got)
    v = k.run("value")
    k.check(v)
    g = k.run("vjp", lse=v["lse"], mean=v["mean"])
    k.check(g)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [50, 1000, 5000, 140000])
def test_distill_infinite_and_missing_values(dt, vocab):
    """Logits of -inf (a masked vocabulary), NaN and infinities in rows that
    do not count, teachers' -inf, and a target whose logit is -inf."""
    k = Case(dt, 12, vocab, top=4, t=2.0, seed=9, pad=False, ct=True)
    k.x[:, vocab // 2 + 1::3] = -math.inf
    k.x[2], k.x[3, ::2], k.x[4, 0] = math.nan, math.inf, math.nan
    k.index[2:5] = -1
    k.teacher[5, :3] = -math.inf                 # one slot left
    k.teacher[6] = -math.inf                     # none
    k.index[7] = -1
    k.index[7, 2] = 1                            # one slot in use
    base = torch.arange(4, device=DEV)
    for r in (0, 1, 5, 8, 10, 11):
        k.index[r] = base + r
    k.index[9] = vocab // 2 + 1                  # all four name a -inf
    got = k.run("step")
    out = torch.zeros(12, dtype=torch.bool, device=DEV)
    out[2:5] = True
    out[6] = True
    assert not got["loss"][out].any() and not got["dx"][out].any()
    assert float(got["loss"][9]) == math.inf and float(got["mean"][1]) == 8.0
    keep = ~out
    keep[9] = False
    k2 = Case(dt, 12, vocab, top=4, t=2.0, seed=9, pad=False, ct=True)
    k2.x, k2.index, k2.teacher, k2.ct = k.x.clone(), k.index.clone(), k.teacher.clone(), k.ct
    k2.x[out], k2.index[out] = 0.0, -1
    k2.x[9], k2.index[9] = 0.0, -1
    # (float64's own -inf * 0 is kept out of the reference)
    k2.x = torch.where(k2.x == -math.inf, torch.full_like(k2.x, -6e4), k2.x)
    r, e = k2.exact()
    for m in ("loss", "lse", "dx"):
        off = (got[m].double() - r[m]).abs()
        bad = ~(off <= e[m] + (1e-4 if m == "lse" else 0.0)) if m != "dx" else ~(off <= e[m])
        bad = bad[keep]
        assert not bool(bad.any()), m
    # the row whose target has no probability: its cotangent is softmax - target
    q = torch.softmax(k.x[9].double() / 2.0, -1)
    want = (q - torch.zeros_like(q).index_fill_(0, torch.tensor([vocab // 2 + 1], device=DEV), 1.0)) * 2.0 * k.ct[9].double()
    assert bool(((got["dx"][9].double() - want).abs() <= (2 * HALF[dt] + 2.0 ** -18) * want.abs() + TINY[dt]).all())
    v = k.run("value")
    g = k.run("vjp", lse=v["lse"])
    assert torch.equal(g["dx"][out], got["dx"][out])


def test_distill_nan_reaches_its_row_alone():
    k = Case("f32", 6, 3000, top=3, seed=1, pad=False)
    k.x[1, 5] = math.nan
    k.teacher[3, 1] = math.nan
    k.index[4, 2] = 3000
    got = k.run("step")
    bad = torch.tensor([False, True, False, True, True, False], device=DEV)
    assert torch.equal(got["loss"].isnan(), bad)
    assert bool(got["dx"][bad].isnan().all()) and not bool(got["dx"][~bad].isnan().any())


@pytest.mark.parametrize("d", [0, 64])
def test_columns_named_twice_have_both_weights(d):
    for vocab in (40, 3000):
        k = Case("f32", 20, vocab, d=d, top=8, seed=4, pad=False)
        k.index[:, 4:] = k.index[:, :4]
        k.index[5] = 17
        k.check(k.run("step"))


def test_offsets_past_32_bits():
    """Given logits of 2.2 G elements: the last rows and the first."""
    rows, vocab, top = 68000, 32768, 3
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    ends = torch.cat([torch.arange(3), torch.arange(rows - 3, rows)]).to(DEV)
    x.zero_()
    x[ends] = torch.randn(6, vocab, device=DEV, generator=g).to(torch.bfloat16)
    k = Case("bf16", 6, vocab, top=top, seed=2, ct=True, pad=False)
    k.x = x[ends]
    index = torch.full((rows, top), -1, dtype=torch.int64, device=DEV)
    teacher = torch.zeros(rows, top, dtype=torch.bfloat16, device=DEV)
    ct = torch.zeros(rows, device=DEV)
    index[ends], teacher[ends], ct[ends] = k.index, k.teacher, k.ct
    op = hip.Distill("bf16", rows, vocab, top)
    dx, loss = torch.empty_like(x), torch.empty(rows, device=DEV)
    work = torch.empty(op.workspace("step"), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    op.value_and_grad(x, index, teacher, dx, loss=loss, ct=ct, work=work)
    torch.cuda.synchronize()
    k.check({"loss": loss[ends], "dx": dx[ends]})
    assert not loss[3:-3].any()


# ---- as they are used -----------------------------------------------------------------

def test_the_same_bits_twice_and_on_another_stream():
    for dt in ("bf16", "f32"):
        k = Case(dt, 333, 2000, d=200, top=9, seed=1)
        a = k.run("step")
        s = torch.cuda.Stream()
        b = k.run("step", stream=s.cuda_stream)
        for m in a:
            same(a[m], b[m], m)


def test_gradients_are_the_values_differences():
    """The mean's change along a direction of x and of w, in f32 from float64
    differences of the device's own losses: within the value's bound over the
    step and the second derivative's part (the step squared)."""
    k = Case("f32", 40, 200, d=48, top=5, t=2.0, seed=3)
    got = k.run("step")
    g = torch.Generator(device=DEV).manual_seed(5)
    for name, grad in (("x", got["dx"]), ("w", got["dw"])):
        base = getattr(k, name).clone()
        v = torch.randn(base.shape, device=DEV, generator=g)
        h = 2.0 ** -6
        vals, steps = [], []
        for s in (h, -h):
            setattr(k, name, (base + s * v).contiguous())
            steps.append(getattr(k, name).double() - base.double())
            vals.append(float(k.run("value")["mean"][0]))
            _, e = k.exact()
        setattr(k, name, base)
        slope = float((grad.double() * (steps[0] - steps[1])).sum())
        err = 2 * float(e["mean"]) + h ** 3 * float(v.double().norm()) ** 3
        # a third derivative of log sum exp along a unit direction is below 1;
        # the rows' directions here are v times the other factor
        assert abs(vals[0] - vals[1] - slope) <= err, (name, vals, slope, err)


def test_recorded_replayed_and_beside_each_other():
    """A head's loss and a distillation of the same sequence, recorded as one
    graph: replayed with new inputs in the same buffers, other work and
    synchronisations between, each replay equal to the eager call."""
    import ctypes
    lib = hip.lib()
    k, j = Case("bf16", 96, 700, d=128, seed=1, ct=False), Case("f16", 64, 5000, top=6, seed=2)
    ok, oj = k.op(), j.op()
    out, args = {}, {}
    for tag, c, op in (("k", k, ok), ("j", j, oj)):
        n = c.rows
        o = {"loss": torch.empty(n, device=DEV), "lse": torch.empty(n, device=DEV), "mean": torch.empty(2, device=DEV),
             "dx": torch.empty_like(c.x)}
        if c.d:
            o["dw"] = torch.empty_like(c.w)
        o["work"] = torch.empty(op.workspace("step"), dtype=torch.uint8, device=DEV)
        out[tag] = o
        args[tag] = op.args("step", **c.ins(), **o, **({"ct": c.ct} if c.ct is not None else {}))
    b = ctypes.c_void_p()
    hip.check(lib.presk_hip_batch_create(ctypes.byref(b)))
    try:
        hip.check(lib.presk_hip_batch_add_head_loss(b, ctypes.byref(args["k"]), 3))
        hip.check(lib.presk_hip_batch_add_distill(b, ctypes.byref(args["j"]), 3))
        hip.check(lib.presk_hip_batch_graph(b))
        for rep in range(3):
            for c, s in ((k, 11), (j, 12)):
                new = Case(c.dtype, c.rows, c.vocab, d=c.d, top=c.top, seed=s + 10 * rep, ct=c.ct is not None)
                for m in ("x", "w", "index", "teacher"):
                    if getattr(c, m) is not None:
                        getattr(c, m).copy_(getattr(new, m))
            torch.cuda.synchronize()
            hip.check(lib.presk_hip_batch_run(b, None))
            hip.sync()
            for tag, c in (("k", k), ("j", j)):
                eager = c.run("step")
                for m, x in eager.items():
                    same(out[tag][m], x, (rep, tag, m))
    finally:
        lib.presk_hip_batch_release(b)


def test_captured_by_the_caller():
    """The call captured by torch into a graph of its own, replayed."""
    k = Case("bf16", 96, 700, d=128, seed=1, ct=False)
    op = k.op()
    o = {"loss": torch.empty(96, device=DEV), "mean": torch.empty(2, device=DEV), "dx": torch.empty_like(k.x), "dw": torch.empty_like(k.w)}
    work = torch.empty(op.workspace("step"), dtype=torch.uint8, device=DEV)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        op.value_and_grad(**k.ins(), **o, work=work, stream=s.cuda_stream)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            op.value_and_grad(**k.ins(), **o, work=work, stream=s.cuda_stream)
    for rep in range(3):
        new = Case("bf16", 96, 700, d=128, seed=20 + rep, ct=False)
        for m in ("x", "w", "index"):
            getattr(k, m).copy_(getattr(new, m))
        for x in o.values():
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = k.run("step")
        for m, x in o.items():
            same(eager[m], x, (rep, m))


def test_the_bindings_own_workspace():
    k = Case("f32", 30, 100, d=16, seed=1)
    op, loss = k.op(), torch.empty(30, device=DEV)
    torch.cuda.synchronize()
    op.value(**k.ins(), loss=loss)
    hip.sync()
    same(loss, k.run("value")["loss"], "loss")


def test_the_bindings_own_workspace_captured_and_outgrown():
    """A captured call's workspace stays when a later call needs a larger one."""
    k = Case("bf16", 30, 3000, d=64, seed=1, ct=False)
    op, loss, s, graph = k.op(), torch.empty(30, device=DEV), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    want = k.run("value")["loss"]
    with torch.cuda.stream(s):
        op.value(**k.ins(), loss=loss, stream=s.cuda_stream)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            op.value(**k.ins(), loss=loss, stream=s.cuda_stream)
    first = op._work
    for _ in range(3):
        op.value_and_grad(**k.ins(), dx=torch.empty_like(k.x), dw=torch.empty_like(k.w))
        torch.cuda.synchronize()
        loss.zero_()
        graph.replay()
        torch.cuda.synchronize()
        same(loss, want, "loss")
    assert op._work is not first and first in op._outgrown
