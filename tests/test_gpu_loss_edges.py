"""The losses on the device where a mask is the type's lowest value, against
float64 under the bounds of tests/test_gpu_loss.py (its Case).

A row's loss and cotangent do not change when its logits, or its teacher's,
are all moved by one number, so the reference takes both below their row's
largest: a difference to the largest that the kernels take too, within half a
step of itself.  What lies 200 T or more below it (e^-200 of the largest: no
part of a sum in f32 or in the compared digits) stands at -200 T there, so that
the bounds, which grow with a logit, stay those of the others."""
import pytest

torch = pytest.importorskip("torch")

from presk_amd import hip  # noqa: E402
from tests.test_gpu_loss import DEV, E24, HALF, TINY, Case, T  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device():
    hip.init(0)
    yield
    torch.cuda.synchronize()


def below(x, t):
    x = x.double()
    return (x - x.amax(-1, keepdim=True)).clamp_min(-200.0 * t)


def reference(k, teacher_only=False):
    s = Case(k.dtype, k.rows, k.vocab, d=k.d, tied=k.tied, top=k.top, t=k.t, seed=0)
    s.index, s.ct = k.index, k.ct
    s.x, s.w = (k.x, k.w) if k.d else (below(k.x, k.t), None)
    s.teacher = below(k.teacher, k.t)
    return s.exact()


def check(got, r, e, names, rows=None):
    for m in names:
        off, bound = (got[m].double() - r[m]).abs(), e[m]
        bad = ~(off <= bound)
        if rows is not None:
            bad = bad[rows]
        assert not bool(bad.any()), (m, bad.nonzero()[:4].tolist())


LOW = [(dt, *s) for dt in ("f32", "bf16", "f16") for s in [
    # rows, vocab, top, T: each of the row kernels' widths, one chunk and several,
    # slots beside the sums and before them
    (12, 50, 4, 1.0), (12, 1000, 4, 2.0), (12, 5000, 4, 1.0), (12, 5000, 70, 1.0), (200, 5000, 4, 1.5), (12, 70000, 4, 1.0),
    (1100, 70000, 3, 1.0), (12, 140000, 5, 2.0), (12, 140000, 100, 1.0),
]]


@pytest.mark.parametrize("c", LOW, ids=str)
def test_distill_of_rows_and_slots_at_the_lowest_value(c):
    """Rows whose mask leaves nothing (softmax uniform), half masked rows, and
    teachers' slots of the lowest value, some and all of a row's."""
    dt, rows, vocab, top, t = c
    low = torch.finfo(T[dt]).min
    k = Case(dt, rows, vocab, top=top, t=t, seed=rows + vocab, pad=False, ct=True)
    k.index = torch.stack([torch.randperm(vocab // 2, device=DEV)[:top] if top <= vocab // 2 else torch.arange(top, device=DEV)
                           for _ in range(rows)]).contiguous()
    k.x[0], k.x[3] = low, low
    k.x[1, vocab // 2:] = low
    k.teacher[2], k.teacher[3] = low, low
    k.teacher[4, 1:] = low
    k.index[5] = -1
    k.x[5] = low
    r, e = reference(k)
    got = k.run("step")
    check(got, r, e, ("loss", "dx"))
    value = k.run("value")
    check(value, r, e, ("loss",))
    scale = k.x.double().amax(-1) / t
    for v in (got, value):
        off = (v["lse"].double() - (r["lse"] + scale)).abs()
        assert bool((off <= e["lse"] + (scale.abs() + r["lse"].abs()) * 4 * E24).all())
    # the gradient alone knows of a row its f32 lse, in which log V is lost
    # beside the lowest value of the wider types
    whole = torch.ones(rows, dtype=torch.bool, device=DEV)
    whole[0] = whole[3] = False
    g = k.run("vjp", lse=value["lse"])
    # (the lse is in the logits' own place, and half a step of it, of T's product
    # and of the difference to it moves an exponent)
    q, moved = torch.softmax(below(k.x, t) / t, -1), torch.expm1(8 * E24 * scale.abs())
    e["dx"] = e["dx"] + 2 * q * (moved * k.ct.double() * t)[:, None]
    check(g, r, e, ("dx",), whole)
    assert bool(g["dx"].isfinite().all())


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab", [(9, 300), (9, 5000), (300, 4000)])
def test_distill_of_a_target_at_the_lowest_value(dt, rows, vocab):
    """A masked column that the teacher wants: a loss of the logits' own size,
    not an infinity, where f32 holds it."""
    k = Case(dt, rows, vocab, top=1, t=1.0, seed=1, pad=False, ct=True)
    low = torch.finfo(T[dt]).min
    k.x[4, 7], k.index[4] = low, 7
    want = float(k.x[4].double().amax()) - low
    for kind in ("step", "value"):
        got = float(k.run(kind)["loss"][4])
        assert abs(got - want) <= want * 2.0 ** -10, (kind, got, want)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("top", [3, 6, 100, 300])
def test_head_of_a_teacher_at_the_lowest_value(dt, top):
    k = Case(dt, 70, 900, d=64, top=top, t=2.0, seed=top, ct=True)
    low = torch.finfo(T[dt]).min
    k.teacher[0], k.teacher[3, 1:] = low, low
    k.index[0] = torch.arange(top, device=DEV)
    r, e = reference(k)
    for kind in ("step", "value"):
        check(k.run(kind), r, e, ("loss", "lse") + (("dx", "dw") if kind == "step" else ()))


def test_a_call_without_a_stream_follows_torchs_current_one():
    """Inputs made on a side stream, late, and the outputs read there: the call
    that names no stream lies between."""
    n, v = 64, 2000
    k = Case("f32", n, v, top=4, seed=1, ct=False)
    want = k.run("value")["loss"]
    x, loss, op = torch.zeros_like(k.x), torch.empty(n, device=DEV), k.op()
    late = torch.randn(4096, 4096, device=DEV)
    op.value(k.x, k.index, k.teacher, loss=loss)
    torch.cuda.synchronize()
    for own in (True, False):
        work = None if own else torch.empty(op.workspace("value"), dtype=torch.uint8, device=DEV)
        x.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                torch.mm(late, late)
            x.copy_(k.x)
            op.value(x, k.index, k.teacher, loss=loss, work=work)
            got = loss.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want), own


def along(k, name):
    """A direction of x or w with rows (columns of a head's weights) of one
    length, against which each row's mean loss is steep, and the largest range
    that the logits / T of a row change by along it: (v, ranges)."""
    base = getattr(k, name).double().requires_grad_()
    x, w = (base, k.w) if name == "x" else (k.x, base)
    z = x.double()
    if k.d:
        z = z @ (w.t() if k.tied else w).double()
    p = torch.softmax((k.teacher.double() / k.t).masked_fill(k.index < 0, -torch.inf), -1).nan_to_num(0.0) if k.top else (k.index >= 0).double()[:, None]
    at = k.index.reshape(k.rows, -1).clamp_min(0)
    u = z / k.t
    # (the reference's direction alone; the loss itself is the device's)
    v, = torch.autograd.grad((p.sum(-1) * torch.logsumexp(u, -1) - (p * u.gather(1, at)).sum(-1)).sum(), base)
    v = v / v.norm(dim=-1, keepdim=True).clamp_min(1e-30)
    x, w = (v, k.w) if name == "x" else (k.x, v)
    a = x.double()
    if k.d:
        a = a @ (w.t() if k.tied else w).double()
    return v, (a.amax(-1) - a.amin(-1)) / k.t


@pytest.mark.parametrize("d,tied,top,t", [(48, False, 5, 2.0), (48, True, 3, 1.5), (48, False, 0, 1.0), (0, False, 5, 2.0)], ids=str)
def test_gradients_are_the_values_steep_differences(d, tied, top, t):
    """f(h) - f(-h) = 2 h f' + h^3 / 3 f''' of the mean f along a line of x or w,
    on which the logits are linear: f''' is T^2 times the mean of the third
    central moments of a row's change a / T under its softmax, at most R^3 /
    (6 sqrt 3) of a change of range R.  Beside it stand both values' errors and
    the gradient's own.  h leaves that an eighth of the difference or less, so a
    gradient of 0, of the other sign, or with a factor of T too many or too few
    is outside it."""
    k = Case("f32", 40, 200, d=d, tied=tied, top=top, t=t, seed=3, ct=False)
    got = k.run("step")
    _, e = k.exact()
    for name, grad in (("x", "dx"), ("w", "dw"))[:2 if d else 1]:
        v, ranges = along(k, name)
        h = 0.5 / float(ranges.max())
        base = getattr(k, name)
        vals, ends, off = [], [], 0.0
        for s in (h, -h):
            setattr(k, name, (base + s * v).float().contiguous())
            ends.append(getattr(k, name).double())
            vals.append(float(k.run("value")["mean"][0]))
            off += float(k.exact()[1]["mean"])
        setattr(k, name, base)
        step = ends[0] - ends[1]
        slope, change = float((got[grad].double() * step).sum()), vals[0] - vals[1]
        third = t * t * float((ranges ** 3).mean()) / (6 * 3 ** 0.5)
        err = off + h ** 3 / 3 * third + float((e[grad] * step.abs()).sum())
        print(name, "change", change, "slope", slope, "bound", err)
        assert abs(change - slope) <= err
        assert err <= abs(slope) / 8
        for wrong in (0.0, -slope) + ((slope / t, slope * t) if t != 1.0 else ()):
            assert abs(change - wrong) > err, wrong


def test_two_streams_at_once():
    """Calls in turn on two streams with nothing waited for between them, each
    object with the workspace that it keeps for its stream, one object on both
    among them: the bits of the calls alone."""
    cases = [Case("bf16", 500, 3000, d=256, seed=1, ct=False), Case("f16", 300, 9000, top=20, t=2.0, seed=2),
             Case("f32", 400, 1500, d=96, tied=True, top=7, seed=3, ct=False)]
    want = [k.run("step") for k in cases]
    ops, streams, rounds = [k.op() for k in cases], [torch.cuda.Stream() for _ in range(2)], 6
    outs = [[[{m: torch.empty_like(x) for m, x in w.items()} for w in want] for _ in streams] for _ in range(rounds)]
    torch.cuda.synchronize()
    for i in range(rounds):
        for s, made in zip(streams, outs[i]):
            with torch.cuda.stream(s):
                for k, op, o in zip(cases, ops, made):
                    op.value_and_grad(**k.ins(), **o, ct=k.ct)
    torch.cuda.synchronize()
    for i in range(rounds):
        for made in outs[i]:
            for w, o in zip(want, made):
                assert [m for m in w if not torch.equal(w[m], o[m])] == [], i


FINE = [(dt, *s) for dt in ("bf16", "f16") for s in [
    # rows, d, vocab, tied, top, T: one piece with a row in a workgroup's
    # registers, longer rows, and (the gradient alone) tiles of the products;
    # sizes that are and are not whole vectors
    (1, 64, 500, False, 0, 1.0), (3, 45, 1272, True, 0, 1.0), (3, 96, 770, False, 18, 2.0), (8, 200, 5003, False, 2, 1.0),
    (21, 1168, 400, False, 1, 2.0), (64, 320, 1347, False, 0, 1.0), (64, 40, 6656, True, 9, 1.5), (17, 40, 70003, False, 0, 1.0),
    (5, 72, 66001, True, 7, 1.0), (33, 4096, 640, False, 0, 1.0),
]]


@pytest.mark.parametrize("c", FINE, ids=str)
def test_few_rows_have_the_cotangents_f32_bits(c):
    """Gradients of at most 64 rows in 16-bit storage: the bounds of f32 storage,
    what two 16-bit parts leave of a cotangent (half a step of half a step; in
    f16 a part's own range ends 2^-38 below the largest), and the rounding of
    the outputs.  As a whole they are as far off as that rounding alone."""
    dt, rows, d, vocab, tied, top, t = c
    k = Case(dt, rows, vocab, d=d, tied=tied, top=top, t=t, seed=rows + vocab, pad=rows > 2, ct=True)
    k.dtype = "f32"
    r, e = k.exact()
    k.dtype = dt
    x, w = k.x.double(), (k.w.t() if tied else k.w).double().contiguous()
    at = k.index.reshape(rows, -1)
    p = torch.softmax((k.teacher.double() / t).masked_fill(at < 0, -torch.inf), -1).nan_to_num(0.0) if top else (at >= 0).double()
    coef = torch.where((at >= 0).any(-1), k.ct.double() * t, 0.0)[:, None]
    g = (torch.softmax(x @ w / t, -1).scatter_add(1, at.clamp_min(0), -p) * coef).abs()
    left = HALF[dt] ** 2 * g + (2.0 ** -38 * coef.amax() if dt == "f16" else 0.0)
    more = {"dx": left @ w.t().abs().contiguous(), "dw": x.t().abs().contiguous() @ left}
    if tied:
        more["dw"] = more["dw"].t()
    lse = k.run("value")["lse"]
    for got in (k.run("step"), k.run("vjp", lse=lse), k.run("step", dw=False), k.run("step", dx=False)):
        for m in {"dx", "dw"} & set(got):
            y, ey = r[m], e[m] + more[m]
            off = (got[m].double() - y).abs()
            bound = ey + HALF[dt] * (y.abs() + ey) + TINY[dt]
            assert bool((off <= bound).all()), (m, float((off / bound).max()))
            rounded = float((y.to(T[dt]).double() - y).norm())
            assert float(off.norm()) <= 1.1 * rounded, (m, float(off.norm()) / rounded)
