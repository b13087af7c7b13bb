"""hip.Attention on the device against float64 (tests/attention_oracle.py), within
what the roundings that it makes may add."""
import math

import pytest

torch = pytest.importorskip("torch")

from presk_amd import hip  # noqa: E402
from tests import attention_oracle as A  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda"


def tensors(dtype, batch, heads, kv, tq, tk, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(A.TORCH[dtype])  # noqa: E731
    return n(batch, tq, heads, d), n(batch, tk, kv, d), n(batch, tk, kv, d), n(batch, tq, heads, d)


def put(x, layout="bshd"):
    if x is None:
        return None
    x = x.to(DEV)
    return x.transpose(1, 2).contiguous() if layout == "bhsd" else x


def run(dtype, q, k, v, do, layout="bshd", scale=None, causal=False, window=0, lens=None, first=None, mask=None, grad=True):
    """The operator's value and gradients against float64."""
    hip.init(0)
    b, tq, h, d = q.shape
    tk, kv = k.shape[1], k.shape[2]
    op = hip.Attention(dtype, b, h, kv, tq, tk, d, causal=causal, window=window, mask_cols=0 if mask is None else mask.shape[-1], scale=scale,
                       layout=layout)
    Q, K, V, DO = (put(x, layout) for x in (q, k, v, do))
    where = {n: x.to(DEV) for n, x in (("lens", lens), ("first", first), ("mask", mask)) if x is not None}
    o = torch.full_like(Q, 9.0)
    lse = torch.full((b, h, tq), 9.0, device=DEV)
    op.value(Q, K, V, o, lse=lse, **where)
    back = (lambda x: x.transpose(1, 2)) if layout == "bhsd" else (lambda x: x)
    ok = A.allowed(b, tq, tk, causal, window, lens, first, mask)
    case = A.Case(dtype, q, k, v, ok, op.scale, do)
    worst = {n: A.check(n, back(g) if n == "o" else g, *case.value()[n]) for n, g in (("o", o), ("lse", lse))}
    if grad:
        grads = {n: torch.full_like(x, 9.0) for n, x in (("dq", Q), ("dk", K), ("dv", V))}
        op.vjp(Q, K, V, o, lse, DO, **grads, **where)
        want = case.vjp(back(o).cpu(), lse.cpu())
        worst.update((n, A.check(n, back(g), *want[n])) for n, g in grads.items())
    torch.cuda.synchronize()
    print({n: round(w, 3) for n, w in worst.items()}, flush=True)


# batch, heads, key heads, queries, keys, head
SIZES = [(1, 1, 1, 1, 1, 64), (2, 4, 2, 5, 77, 64), (1, 3, 1, 33, 65, 128), (2, 2, 2, 128, 128, 64), (1, 2, 1, 200, 131, 80),
         (2, 6, 3, 129, 300, 128), (3, 5, 5, 64, 64, 8), (1, 8, 2, 1, 700, 128), (1, 2, 2, 17, 31, 96)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_against_float64(dtype, causal, size):
    run(dtype, *tensors(dtype, *size, seed=sum(size)), causal=causal)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("size", [(1, 2, 1, 70, 150, 256), (1, 2, 2, 1, 400, 200), (2, 4, 1, 40, 33, 136)], ids=str)
def test_wide_heads(dtype, size):
    run(dtype, *tensors(dtype, *size), causal=size[3] <= size[4])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d", [1, 3, 20, 33, 65, 101])
def test_heads_that_are_no_whole_vectors(dtype, d):
    run(dtype, *tensors(dtype, 2, 4, 2, 37, 90, d), causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [(5, 20, 20, 300, 300, 64), (3, 14, 7, 1000, 1000, 128), (5, 4, 1, 300, 2000, 64), (1, 7, 7, 640, 2600, 128),
                                  (9, 16, 2, 55, 600, 80)], ids=str)
def test_all_workgroups_on_the_chip_at_once(dtype, size):
    """A number of tiles, or of their shares of the keys, that the XCDs do not divide:
    each is some workgroup's."""
    run(dtype, *tensors(dtype, *size, seed=3), causal=True, grad=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["all", "causal", "window", "lengths", "mask", "dk", "dv"])
@pytest.mark.parametrize("d", [20, 64, 128, 200])
def test_few_keys_and_many_rows(dtype, kind, d):
    """Keys' gradients that one workgroup a tile would leave CUs idle for: in parts
    of the rows, of which some may have none."""
    if dtype == "f32" and d > 128:
        pytest.skip("f32 heads end at 128")
    b, h, kv, tq, tk = 2, 6, 2, 610, 200
    q, k, v, do = tensors(dtype, b, h, kv, tq, tk, d, seed=d)
    g = torch.Generator().manual_seed(d)
    if kind in ("dk", "dv"):
        hip.init(0)
        op = hip.Attention(dtype, b, h, kv, tq, tk, d)
        Q, K, V, DO = (x.to(DEV) for x in (q, k, v, do))
        o, lse = torch.empty_like(Q), torch.empty(b, h, tq, device=DEV)
        op.value(Q, K, V, o, lse=lse)
        both = {"dk": torch.empty_like(K), "dv": torch.empty_like(V)}
        op.vjp(Q, K, V, o, lse, DO, **both)
        alone = torch.full_like(K, 9.0)
        op.vjp(Q, K, V, o, lse, DO, **{kind: alone})
        assert torch.equal(alone, both[kind])
        return
    more = {"all": {}, "causal": {"causal": True, "first": torch.tensor([0, -300])}, "window": {"causal": True, "window": 50, "first": torch.tensor([-400, 0])},
            "lengths": {"lens": torch.tensor([0, 131])}, "mask": {"mask": torch.rand(tq, tk, generator=g) < 0.3}}[kind]
    run(dtype, q, k, v, do, **more)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
def test_windows(dtype, window):
    run(dtype, *tensors(dtype, 1, 4, 2, 150, 210, 64), causal=True, window=window)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["all", "causal", "window"])
def test_sequences_of_unequal_lengths(dtype, kind):
    """Lengths of nothing, of one key and past the end; queries before the
    first key, and past the last."""
    q, k, v, do = tensors(dtype, 6, 4, 2, 40, 170, 64)
    lens = torch.tensor([0, 1, 170, 1000, 63, -5])
    first = torch.tensor([0, -20, 130, 200, 23, 7])
    for b, n in enumerate(lens.clamp(0, 170).tolist()):
        # what lies past a sequence's end is not read
        k[b, n:], v[b, n:] = math.nan, math.inf
    run(dtype, q, k, v, do, causal=kind != "all", window=25 if kind == "window" else 0, lens=lens, first=first)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("size", [(2, 4, 2, 100, 100, 64), (2, 2, 2, 45, 333, 128)], ids=str)
def test_masks_of_all_keys(dtype, shared, size):
    """Rows and columns that are masked whole, and a mask that every sequence
    shares."""
    q, k, v, do = tensors(dtype, *size)
    mask = torch.rand(size[0], size[3], size[4], generator=torch.Generator().manual_seed(1)) < 0.4
    mask[:, 3] = False
    mask[:, :, 40:] = mask[:, :, 40:] & (torch.arange(40, size[4]) % 7 > 2)
    mask[:, 7:20, :70] = True
    run(dtype, q, k, v, do, mask=mask[1] if shared else mask)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("per", [1, 4])
def test_trees_of_drafted_tokens(dtype, per):
    """A mask over the last keys of a cache, as bytes; what lies past it is not
    read."""
    b, tq, tk = 4, 13, 500
    q, k, v, do = tensors(dtype, b, 2 * per, 2, tq, tk, 64)
    lens = torch.tensor([13, 500, 77, 300])
    parent = (torch.rand(b, tq, generator=torch.Generator().manual_seed(2)) * torch.arange(tq)).long()
    mask = torch.zeros(b, tq, tq, dtype=torch.uint8)
    for i in range(tq):
        if i:
            mask[:, i] = mask[torch.arange(b), parent[:, i]]
        mask[:, i, i] = 255
    run(dtype, q, k, v, do, lens=lens, first=lens - tq, mask=mask)
    run(dtype, q, k, v, do, first=torch.tensor([0, 400, -3, 480]), mask=mask)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_heads_before_rows(dtype):
    run(dtype, *tensors(dtype, 2, 6, 2, 50, 81, 64), layout="bhsd", causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_slices_of_packed_projections(dtype):
    """Queries, keys, values and their gradients side by side in one buffer's rows."""
    hip.init(0)
    b, n, h, kv, d = 2, 90, 4, 2, 64
    q, k, v, do = tensors(dtype, b, h, kv, n, n, d)
    packed = torch.cat((q, k, v), 2).to(DEV)
    cut = lambda x: x.split((h, kv, kv), 2)  # noqa: E731
    Q, K, V = cut(packed)
    grads = torch.full_like(packed, 9.0)
    dq, dk, dv = cut(grads)
    op = hip.Attention(dtype, b, h, kv, n, n, d, causal=True)
    o, lse = torch.empty_like(do, device=DEV), torch.empty(b, h, n, device=DEV)
    op.value(Q, K, V, o, lse=lse)
    op.vjp(Q, K, V, o, lse, do.to(DEV), dq=dq, dk=dk, dv=dv)
    case = A.Case(dtype, q, k, v, A.allowed(b, n, n, True), op.scale, do)
    A.check("o", o, *case.value()["o"])
    want = case.vjp(o.cpu(), lse.cpu())
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        A.check(name, got, *want[name])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_start_anywhere(dtype):
    """Addresses and strides that are no multiples of 16 bytes, beside ones that are."""
    hip.init(0)
    b, n, h, d = 2, 70, 3, 64
    q, k, v, do = tensors(dtype, b, h, h, n, n, d)

    def odd(x):
        wide = torch.full((b, n + 1, h, d + 3), 9.0, dtype=x.dtype, device=DEV)
        y = wide[:, 1:, :, 1:d + 1]
        y.copy_(x)
        return y, wide

    op = hip.Attention(dtype, b, h, h, n, n, d, causal=True)
    (Q, _), (K, _), (DO, _) = odd(q), odd(k), odd(do)
    (o, ow), (dq, qw), (dv, vw) = odd(q), odd(q), odd(v)
    lse, dk, V = torch.empty(b, h, n, device=DEV), torch.empty_like(k, device=DEV), v.to(DEV)
    op.value(Q, K, V, o, lse=lse)
    op.vjp(Q, K, V, o, lse, DO, dq=dq, dk=dk, dv=dv)
    case = A.Case(dtype, q, k, v, A.allowed(b, n, n, True), op.scale, do)
    A.check("o", o, *case.value()["o"])
    want = case.vjp(o.cpu(), lse.cpu())
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        A.check(name, got, *want[name])
    for wide in (ow, qw, vw):
        assert (wide[..., 0] == 9).all() and (wide[..., d + 1:] == 9).all() and (wide[:, 0] == 9).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_keys_that_the_batch_shares(dtype):
    """Stride 0 over the batch: a prefix of all sequences."""
    hip.init(0)
    b, tq, tk, h, d = 3, 9, 140, 2, 64
    q, k, v, do = tensors(dtype, b, h, h, tq, tk, d)
    k, v = k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1)
    op = hip.Attention(dtype, b, h, h, tq, tk, d)
    o, lse = torch.empty_like(q, device=DEV), torch.empty(b, h, tq, device=DEV)
    op.value(q.to(DEV), k[:1].to(DEV).expand_as(k), v[:1].to(DEV).expand_as(v), o, lse=lse)
    case = A.Case(dtype, q, k, v, A.allowed(b, tq, tk), op.scale, do)
    A.check("o", o, *case.value()["o"])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scores_far_apart(dtype):
    """Scores of thousands, and a scale of its own: the weights are one key's."""
    q, k, v, do = tensors(dtype, 1, 2, 2, 40, 100, 64)
    run(dtype, q * 8, k * 8, v, do, scale=2.0, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scores_that_are_equal(dtype):
    """Weights of 1 / keys each."""
    q, k, v, do = tensors(dtype, 1, 2, 2, 40, 1500, 64)
    run(dtype, q * 0, k, v, do)


def test_no_queries_and_no_keys():
    hip.init(0)
    for tq, tk in ((0, 5), (5, 0), (0, 0)):
        q, k, v, do = (x.to(DEV) for x in tensors("bf16", 2, 2, 2, tq, tk, 64))
        op = hip.Attention("bf16", 2, 2, 2, tq, tk, 64)
        o, lse = torch.full_like(q, 9.0), torch.full((2, 2, tq), 9.0, device=DEV)
        op.value(q, k, v, o, lse=lse)
        dq, dk, dv = torch.full_like(q, 9.0), torch.full_like(k, 9.0), torch.full_like(v, 9.0)
        op.vjp(q, k, v, o, lse, do, dq=dq, dk=dk, dv=dv)
        assert (o == 0).all() and (lse == -math.inf).all() and (dq == 0).all() and (dk == 0).all() and (dv == 0).all()


def test_a_gradient_alone():
    """Any of the three by itself is the one that comes with the others."""
    hip.init(0)
    q, k, v, do = (x.to(DEV) for x in tensors("bf16", 1, 4, 2, 100, 130, 64))
    op = hip.Attention("bf16", 1, 4, 2, 100, 130, 64, causal=True)
    o, lse = torch.empty_like(q), torch.empty(1, 4, 100, device=DEV)
    op.value(q, k, v, o, lse=lse)
    like = {"dq": q, "dk": k, "dv": v}
    all_ = {n: torch.empty_like(x) for n, x in like.items()}
    op.vjp(q, k, v, o, lse, do, **all_)
    for n, x in like.items():
        one = torch.full_like(x, 9.0)
        op.vjp(q, k, v, o, lse, do, **{n: one})
        assert torch.equal(one, all_[n])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients_by_differences(dtype):
    """Of sum(o * do) along a random direction, from float32 values."""
    hip.init(0)
    b, tq, tk, h, kv, d = 1, 20, 50, 4, 2, 32
    q, k, v, do = (x.float() for x in tensors(dtype, b, h, kv, tq, tk, d))
    dirs = [x.double() for x in tensors("f32", b, h, kv, tq, tk, d, seed=5)[:3]]
    ok = A.allowed(b, tq, tk, True)

    def f(t):
        c = A.Case("f32", *(x.double() + t * y for x, y in zip((q, k, v), dirs)), ok, d ** -0.5)
        return float((c.value()["o"][0] * do.double()).sum())

    slope = (f(1e-4) - f(-1e-4)) / 2e-4
    ty = A.TORCH[dtype]
    Q, K, V, DO = (x.to(ty).to(DEV) for x in (q, k, v, do))
    op = hip.Attention(dtype, b, h, kv, tq, tk, d, causal=True)
    o, lse = torch.empty_like(Q), torch.empty(b, h, tq, device=DEV)
    op.value(Q, K, V, o, lse=lse)
    grads = [torch.empty_like(x) for x in (Q, K, V)]
    op.vjp(Q, K, V, o, lse, DO, *grads)
    got = sum(float((g.cpu().double() * y).sum()) for g, y in zip(grads, dirs))
    # the gradient's own roundings, independent: a few half steps of its terms'
    # root mean square, and the differences' 1e-6
    terms = math.sqrt(sum(float((g.cpu().double() * y).square().sum()) for g, y in zip(grads, dirs)))
    assert abs(got - slope) <= 16 * A.HALF[dtype] * terms + 1e-6 * (1 + abs(slope)), (got, slope, terms)


def test_a_captured_call_replays():
    """A captured value and gradient over lengths and masks that change."""
    hip.init(0)
    b, tq, tk, h, kv, d = 2, 6, 300, 4, 2, 64
    q, k, v, do = (x.to(DEV) for x in tensors("bf16", b, h, kv, tq, tk, d))
    mask = torch.ones(b, tq, tq, dtype=torch.bool, device=DEV).tril()
    lens, first = torch.tensor([40, 50], device=DEV), torch.tensor([34, 44], device=DEV)
    op = hip.Attention("bf16", b, h, kv, tq, tk, d, mask_cols=tq)
    o, lse = torch.empty_like(q), torch.empty(b, h, tq, device=DEV)
    grads = [torch.empty_like(x) for x in (q, k, v)]
    works = [torch.empty(op.workspace(n), dtype=torch.uint8, device=DEV) for n in ("value", "vjp")]

    def call(o, lse, grads, works):
        op.value(q, k, v, o, lse=lse, lens=lens, first=first, mask=mask, work=works[0])
        op.vjp(q, k, v, o, lse, do, *grads, lens=lens, first=first, mask=mask, work=works[1])

    call(o, lse, grads, works)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(o, lse, grads, works)
    for step in range(4):
        lens.add_(50), first.add_(50)
        mask[:, step + 1, step] = False
        q.mul_(1.1)
        for x in (o, lse, *grads):
            x.fill_(9.0)
        graph.replay()
        got = [x.clone() for x in (o, lse, *grads)]
        again = [torch.empty_like(x) for x in got]
        call(again[0], again[1], again[2:], [torch.empty_like(w) for w in works])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, again)), step


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_captured_shares_and_parts(dtype):
    """Keys in shares, their gradients in parts beside the queries', single tokens:
    two graphs of them that share one workspace, replayed in turn with eager calls
    between, over inputs that change."""
    hip.init(0)
    b, h, kv, tq, tk, d = 1, 8, 2, 300, 2100, 64
    q, k, v, do = (x.to(DEV) for x in tensors(dtype, b, h, kv, tq, tk, d))
    lens, first = torch.tensor([1200], device=DEV), torch.tensor([900], device=DEV)
    op, one = hip.Attention(dtype, b, h, kv, tq, tk, d, causal=True), hip.Attention(dtype, b, h, kv, 1, tk, d, causal=True)
    need = max(op.workspace("value"), op.workspace("vjp"), one.workspace("value"))
    rows = 4 * b * h * tq
    assert op.workspace("value") > 64 * rows and op.workspace("vjp") > 2 * rows + 4 * 2 * b * kv * tk * d     # (shares, parts)
    work = torch.empty(need, dtype=torch.uint8, device=DEV)

    def call(outs, work, i):
        o, lse, dq, dk, dv, o1 = outs
        if i == 0:
            op.value(q, k, v, o, lse=lse, lens=lens, first=first, work=work)
            op.vjp(q, k, v, o, lse, do, dq=dq, dk=dk, dv=dv, lens=lens, first=first, work=work)
        else:
            one.value(q[:, -1:], k, v, o1, lens=lens, first=last, work=work)

    def outs():
        return [torch.empty_like(q), torch.empty(b, h, tq, device=DEV), *(torch.empty_like(x) for x in (q, k, v)), torch.empty_like(q[:, -1:])]

    last = lens - 1
    mine, graphs = outs(), []
    for i in (0, 1):
        call(mine, work, i)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            call(mine, work, i)
    for step in range(3):
        lens.add_(300), first.add_(300), last.add_(300)
        k.mul_(1.1)
        for x in mine:
            x.fill_(9.0)
        graphs[0].replay(), graphs[1].replay()
        again = outs()
        for i in (0, 1):
            call(again, torch.empty_like(work), i)
        torch.cuda.synchronize()
        assert [n for n, x, y in zip(("o", "lse", "dq", "dk", "dv", "o1"), mine, again) if not torch.equal(x, y)] == [], step


def test_two_streams():
    """Calls of one object on two streams with no wait between them."""
    hip.init(0)
    ins = [[x.to(DEV) for x in tensors("bf16", 2, 4, 1, 1, 2000, 128, seed=s)] for s in (1, 2)]
    op = hip.Attention("bf16", 2, 4, 1, 1, 2000, 128)
    alone = []
    for q, k, v, _ in ins:
        o = torch.empty_like(q)
        op.value(q, k, v, o)
        alone.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    outs = [[torch.empty_like(i[0]) for _ in range(8)] for i in ins]
    torch.cuda.synchronize()
    for r in range(8):
        for s, (q, k, v, _), o in zip(streams, ins, outs):
            with torch.cuda.stream(s):
                op.value(q, k, v, o[r])
    torch.cuda.synchronize()
    for o, want in zip(outs, alone):
        assert all(torch.equal(x, want) for x in o)


def test_f16_gradients_that_overflow_set_the_flag():
    hip.init(0)
    q, k, v, do = (x.to(DEV) for x in tensors("f16", 1, 2, 2, 40, 40, 64))
    op = hip.Attention("f16", 1, 2, 2, 40, 40, 64)
    o, lse = torch.empty_like(q), torch.empty(1, 2, 40, device=DEV)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    grads = [torch.empty_like(x) for x in (q, k, v)]
    op.value(q, k, v, o, lse=lse, flag=flag)
    op.vjp(q, k, v, o, lse, do, *grads, flag=flag)
    assert int(flag) == 0
    op.vjp(q, k, v, o, lse, (do.float() * 0 + 60000).half(), *grads, flag=flag)
    assert int(flag) == 1


def test_f16_weights_cotangents_that_overflow_set_the_flag():
    """p (do . v - do . o) past f16, whose sums would not be: two keys of opposite
    values, so that the cotangents are half of 64 * 4000, times keys of 0.01."""
    hip.init(0)
    q, do = torch.zeros(1, 4, 1, 64), torch.full((1, 4, 1, 64), 4000.0)
    v = torch.ones(1, 2, 1, 64)
    v[:, 1] = -1
    q, k, v, do = (x.half().to(DEV) for x in (q, torch.full((1, 2, 1, 64), 0.01), v, do))
    op = hip.Attention("f16", 1, 1, 1, 4, 2, 64)
    o, lse, flag = torch.empty_like(q), torch.empty(1, 1, 4, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    op.value(q, k, v, o, lse=lse, flag=flag)
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    op.vjp(q, k, v, o, lse, do / 16, dq=dq, dk=dk, dv=dv, flag=flag)
    assert int(flag) == 0 and bool(torch.isfinite(dq).all())
    op.vjp(q, k, v, o, lse, do, dq=dq, flag=flag)
    assert int(flag) == 1
    flag.zero_()
    op.vjp(q + 1, k, v, o, lse, do, dk=dk, flag=flag)
    assert int(flag) == 1


def test_a_long_cache():
    """Keys whose elements lie past 2^31 elements and 2^32 bytes: the last ones'
    rows alone are read, by a window."""
    hip.init(0)
    tk, kv, d, w = 1 << 20, 17, 128, 200
    k = torch.zeros(1, tk, kv, d, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(3)
    kl, vl = (torch.randn(1, w, kv, d, generator=g).bfloat16() for _ in range(2))
    k[:, -w:], v[:, -w:] = kl.to(DEV), vl.to(DEV)
    q = torch.randn(1, 3, kv, d, generator=g).bfloat16()
    op = hip.Attention("bf16", 1, kv, kv, 3, tk, d, causal=True, window=w - 2)
    o = torch.empty_like(q, device=DEV)
    op.value(q.to(DEV), k, v, o)
    case = A.Case("bf16", q, kl, vl, A.allowed(1, 3, w, True, w - 2), op.scale)
    A.check("o", o, *case.value()["o"])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("stride", [0, 1, 2 ** 26, 2 ** 40])
@pytest.mark.parametrize("tq, tk", [(1, 5), (1, 300), (70, 1)])
def test_one_row_whose_stride_says_nothing(dtype, causal, stride, tq, tk):
    """A length of one leaves a tensor's row stride free: that of an expanded tensor is
    0, and a large one times a tile's row numbers would pass 32 bits."""
    hip.init(0)
    b, h, kv, d = 2, 4, 2, 64
    q, k, v, do = tensors(dtype, b, h, kv, tq, tk, d)

    def far(x):
        x = x.to(DEV)
        return x.as_strided(x.shape, (x.stride(0), stride, d, 1)) if x.shape[1] == 1 else x

    op = hip.Attention(dtype, b, h, kv, tq, tk, d, causal=causal)
    Q, K, V, DO = map(far, (q, k, v, do))
    o, dq, dk, dv = (far(torch.full_like(x, 9.0)) for x in (q, q, k, v))
    lse = torch.empty(b, h, tq, device=DEV)
    op.value(Q, K, V, o, lse=lse)
    op.vjp(Q, K, V, o, lse, DO, dq=dq, dk=dk, dv=dv)
    case = A.Case(dtype, q, k, v, A.allowed(b, tq, tk, causal), op.scale, do)
    A.check("o", o, *case.value()["o"])
    want = case.vjp(o.cpu(), lse.cpu())
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        A.check(name, got, *want[name])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_cotangent_that_is_shared(dtype):
    """One query's, of one row for all sequences and heads by expansion."""
    hip.init(0)
    b, h, kv, tk, d = 3, 4, 2, 200, 64
    q, k, v, _ = tensors(dtype, b, h, kv, 1, tk, d)
    do = torch.linspace(-1, 2, d).to(A.TORCH[dtype]).expand(b, 1, h, d)
    op = hip.Attention(dtype, b, h, kv, 1, tk, d)
    Q, K, V = (x.to(DEV) for x in (q, k, v))
    o, lse = torch.empty_like(Q), torch.empty(b, h, 1, device=DEV)
    op.value(Q, K, V, o, lse=lse)
    grads = {n: torch.empty_like(x) for n, x in (("dq", Q), ("dk", K), ("dv", V))}
    op.vjp(Q, K, V, o, lse, do[0, 0, 0].to(DEV).expand(b, 1, h, d), **grads)
    want = A.Case(dtype, q, k, v, A.allowed(b, 1, tk), op.scale, do).vjp(o.cpu(), lse.cpu())
    for n, g in grads.items():
        A.check(n, g, *want[n])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["all", "causal", "window", "lengths", "mask"])
@pytest.mark.parametrize("d", [64, 128])
def test_more_workgroups_than_cus(dtype, kind, d):
    """528 tiles of queries and of keys: the kernels of four waves, each gradient's a
    launch of its own."""
    b, h, n = 33, 8, 130
    q, k, v, do = tensors(dtype, b, h, h, n, n, d, seed=d)
    g = torch.Generator().manual_seed(d)
    lens = torch.randint(0, n + 1, (b,), generator=g)
    mask = torch.rand(b, n, n, generator=g) < 0.3
    mask[::3, 32:, 32:96] = False                    # (whole blocks without any)
    more = {"all": {}, "causal": {"causal": True}, "window": {"causal": True, "window": 50, "first": torch.randint(-40, 40, (b,), generator=g)},
            "lengths": {"lens": lens, "causal": True, "first": lens - n}, "mask": {"mask": mask}}[kind]
    run(dtype, q, k, v, do, **more)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [(14, 64, 8, 40, 40, 128), (14, 64, 8, 40, 40, 64), (1, 40, 2, 3400, 130, 64), (1, 40, 2, 3400, 130, 128),
                                  (2, 12, 4, 2100, 70, 96)], ids=str)
def test_the_queries_gradient_after_the_keys(dtype, size):
    """Few tiles of keys, whose kernel has eight waves, and many of queries."""
    run(dtype, *tensors(dtype, *size, seed=5), causal=size[3] == size[4])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_a_grouped_step(dtype):
    """Heads in groups of four, over 256 tiles of either, head after head."""
    run(dtype, *tensors(dtype, 9, 32, 8, 400, 400, 64, seed=2), causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [(4, 2, 1, 1, 6000, 64), (2, 8, 2, 3, 9000, 128), (1, 3, 1, 5, 5000, 80)], ids=str)
def test_many_shares_of_the_keys(dtype, size):
    """More than 16 shares of a sequence's keys, which a workgroup's waves join; some
    sequences have fewer, and none."""
    lens = torch.tensor([size[4], 300, 0, 4500])[:size[0]]
    run(dtype, *tensors(dtype, *size, seed=7), lens=lens, grad=False)
    run(dtype, *tensors(dtype, *size, seed=8), grad=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_more_shares_than_a_waves_lanes(dtype):
    """274 shares, 64 times 4 and the rest."""
    run(dtype, *tensors(dtype, 1, 2, 1, 1, 70000, 64, seed=9), grad=False)
    run(dtype, *tensors(dtype, 1, 2, 1, 2, 70000, 64, seed=10), causal=True, grad=False)


def sum_error(rows, d, lse, value=False):
    """What f32 sums over `rows` random terms p x may be off by, root mean square over
    that of the sums, and half as much again; in half steps (2^-24) of them:
    the sums: one rounding every 32 rows, 0.41 on average of a partial one's, which
    grow as a random walk's: 0.41 sqrt(rows / 32 / 2);
    a matrix instruction: a step at most, 0.82 on average, six every 16 elements of a
    score and of a cotangent, and as many every 16 of the 32 rows;
    a number between 2^e and 2^(e + 1): 0.58 2^e.  p = exp2(s log2 e - lse log2 e) has
    that difference's, times ln 2, and lse's: in log 2 and times ln 2, as it is
    stored, and times log2 e again, and of the weights' sum, whose partial ones grow
    evenly, 0.41 sqrt(keys / 32 / 3).  The value has the sum's and the difference's."""
    product, block = 0.82 * math.sqrt(6 * d / 16 / 2), 0.82 * math.sqrt(12 / 2)
    step = lambda x: 0.58 * 2.0 ** math.floor(math.log2(x))  # noqa: E731
    log2 = step(lse / math.log(2)) * math.log(2)
    weights = 0.41 * math.sqrt(math.exp(lse) / 32 / 3)
    terms = [product, block, log2, weights] + ([] if value else [product, log2, step(lse), log2])
    return 1.5 * A.F * math.sqrt(0.41 ** 2 * rows / 32 / 2 + sum(x * x for x in terms))


def off(got, want):
    return float((got.double() - want).square().mean().sqrt() / want.square().mean().sqrt())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv", [128, 129])
def test_f32_sums_over_a_groups_rows(d, kv):
    """Keys' and values' gradients over 4 x 4096 rows, by eight waves and by four."""
    hip.init(0)
    per, tq, tk = 4, 4096, 256
    g = torch.Generator(DEV).manual_seed(d + kv)
    q, k, v, do = (torch.randn(1, n, h, d, generator=g, device=DEV) for n, h in ((tq, per * kv), (tk, kv), (tk, kv), (tq, per * kv)))
    op = hip.Attention("f32", 1, per * kv, kv, tq, tk, d)
    o, lse = torch.empty_like(q), torch.empty(1, per * kv, tq, device=DEV)
    op.value(q, k, v, o, lse=lse)
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    op.vjp(q, k, v, o, lse, do, dk=dk, dv=dv)
    for head in (0, kv - 1):
        x, y = (t[0, :, head * per:(head + 1) * per].double().transpose(0, 1) for t in (q, do))
        kd, vd = k[0, :, head].double(), v[0, :, head].double()
        p = torch.softmax(x @ kd.T * op.scale, -1)
        dp = y @ vd.T
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * op.scale
        worst = {"dv": off(dv[0, :, head], sum(p[n].T @ y[n] for n in range(per))), "dk": off(dk[0, :, head], sum(ds[n].T @ x[n] for n in range(per)))}
        print({n: f"{e:.3g}" for n, e in worst.items()}, flush=True)
        assert max(worst.values()) <= sum_error(per * tq, d, math.log(tk) + 0.5), worst


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [256, 264])
def test_f32_sums_over_many_keys(d, heads):
    """The value and the queries' gradient over 16384 keys."""
    hip.init(0)
    kv, tq, tk = 8, 128, 16384
    g = torch.Generator(DEV).manual_seed(d + heads)
    q, k, v, do = (torch.randn(1, n, h, d, generator=g, device=DEV) for n, h in ((tq, heads), (tk, kv), (tk, kv), (tq, heads)))
    op = hip.Attention("f32", 1, heads, kv, tq, tk, d)
    o, lse, dq = torch.empty_like(q), torch.empty(1, heads, tq, device=DEV), torch.empty_like(q)
    op.value(q, k, v, o, lse=lse)
    op.vjp(q, k, v, o, lse, do, dq=dq)
    for head in (0, heads - 1):
        x, y, kd, vd = (t[0, :, n].double() for t, n in ((q, head), (do, head), (k, head * kv // heads), (v, head * kv // heads)))
        p = torch.softmax(x @ kd.T * op.scale, -1)
        dp = y @ vd.T
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * op.scale
        worst = {"o": off(o[0, :, head], p @ vd), "dq": off(dq[0, :, head], ds @ kd)}
        print({n: f"{e:.3g}" for n, e in worst.items()}, flush=True)
        assert worst["o"] <= sum_error(tk, d, math.log(tk) + 0.5, value=True), worst
        assert worst["dq"] <= sum_error(tk, d, math.log(tk) + 0.5), worst


@pytest.mark.parametrize("n", [40, 400])
def test_f32_small_elements(n):
    """Three bf16 parts are all of an element down to 2^-110; below, the last is a
    multiple of bf16's smallest step, 2^-133, of which half may be lost."""
    hip.init(0)
    g = torch.Generator().manual_seed(n)
    v = torch.randn(1, 1, 60, 64, generator=g, dtype=torch.float64) * 2.0 ** -torch.arange(100, 130, 0.5, dtype=torch.float64)[None, None, :, None]
    v = v.float().transpose(1, 2).contiguous()                  # [1, 60 keys, 1, 64]
    q = torch.zeros(1, n, 1, 64)
    k = torch.zeros(1, 60, 1, 64)
    i = torch.arange(n) % 60
    first = torch.tensor([0])
    mask = torch.zeros(n, 60, dtype=torch.bool)
    mask[torch.arange(n), i] = True                             # query i reads one key
    op = hip.Attention("f32", 1, 1, 1, n, 60, 64, mask_cols=60)
    o = torch.empty(1, n, 1, 64, device=DEV)
    op.value(q.to(DEV), k.to(DEV), v.to(DEV), o, first=first.to(DEV), mask=mask.to(DEV))
    want = v[0, i, 0].double()
    err = (o.cpu()[0, :, 0].double() - want).abs()
    print(float((err / (2.0 ** -134 + 2.0 ** -24 * want.abs())).max()))
    assert (err <= 2.0 ** -134 + 2.0 ** -24 * want.abs()).all()


F16_SIZES = [(1, 4, 2, 1024, 1024, 64), (33, 8, 8, 130, 130, 64), (33, 4, 4, 200, 200, 128), (1, 2, 1, 300, 600, 200), (14, 8, 1, 40, 90, 96)]


def f16_gradients(size, do, q=None, k=None, causal=True, last=0):
    """The largest root mean square error of f16's gradients, over that of rounding the
    exact ones to f16.  (Without a head's first element: where the scores hang on
    that one, the cotangents' roundings are times it; `last`: of that many rows.)"""
    hip.init(0)
    q0, k0, v, _ = tensors("f16", *size)
    q, k = q0 if q is None else q, k0 if k is None else k
    op = hip.Attention("f16", *size, causal=causal)
    Q, K, V, DO = (x.to(DEV) for x in (q, k, v, do))
    o, lse = torch.empty_like(Q), torch.empty(size[0], size[1], size[3], device=DEV)
    op.value(Q, K, V, o, lse=lse)
    grads = {n: torch.empty_like(x) for n, x in (("dq", Q), ("dk", K), ("dv", V))}
    op.vjp(Q, K, V, o, lse, DO, **grads)
    want = A.Case("f16", q, k, v, A.allowed(size[0], size[3], size[4], causal), op.scale, do).vjp(o.cpu(), lse.cpu())
    rms = lambda x: float(x.square().mean().sqrt())  # noqa: E731
    out = {}
    for n, g in grads.items():
        x = want[n][0]
        A.check(n, g, *want[n])
        out[n] = rms((g.cpu().double() - x)[:, -last:, :, 1:]) / rms((x.half().double() - x)[:, -last:, :, 1:])
    print({n: round(e, 2) for n, e in out.items()}, flush=True)
    return max(out.values())


@pytest.mark.parametrize("power", [0, -10, -13])
@pytest.mark.parametrize("size", F16_SIZES, ids=str)
def test_f16_gradients_of_small_cotangents(size, power):
    """A mean loss's: the weights' cotangents, rounded to f16, add as much as the
    gradients' own rounding does, whose errors are then 1.41 times those alone (and a
    tenth for the sample), not what f16 has left at that size."""
    do = (tensors("f16", *size)[3].float() * 2.0 ** power).half()
    worst = f16_gradients(size, do)
    assert worst <= 1.41 * 1.1


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("size", F16_SIZES, ids=str)
def test_f16_gradients_of_cotangents_far_apart(size, turned):
    """From 2^-20 to 2^6 along the rows, either way."""
    do = tensors("f16", *size)[3].float()
    power = torch.linspace(-20, 6, size[3])
    do = (do * torch.exp2(power.flip(0) if turned else power)[None, :, None, None]).half()
    worst = f16_gradients(size, do)
    assert worst <= 1.41 * 1.1


@pytest.mark.parametrize("size", [(2, 4, 2, 1001, 1000, 64), (9, 8, 8, 1001, 1000, 128), (1, 2, 1, 601, 600, 200)], ids=str)
def test_f16_gradients_of_low_scores(size):
    """Scores of -32 and less: a lane without a row or a key, beside the last ones of
    them, has scores of 0 in their place and weights of 10^13, which say nothing of
    the others' size."""
    q, k, _, do = tensors("f16", *size)
    q[..., 0], k[..., 0] = 16, -16 * (size[5] / 64) ** 0.5
    worst = f16_gradients(size, (do.float() * 2.0 ** -12).half(), q, k, False, last=8)
    assert worst <= 1.41 * 1.1


def test_captured_calls_take_their_own_workspace():
    """A first call while its stream is captured, without one of the caller's."""
    hip.init(0)
    b, n, h, kv, d = 2, 70, 4, 2, 64
    q, k, v, do = (x.to(DEV) for x in tensors("bf16", b, h, kv, n, n, d))
    freq, g = torch.from_numpy(hip.rotary_frequencies(d)).to(DEV), torch.ones(d, dtype=torch.bfloat16, device=DEV)

    def ops():
        return hip.Attention("bf16", b, h, kv, n, n, d, causal=True), hip.HeadRotary("bf16", b, n, h, kv, d, norm=True)

    def call(op, rot, outs):
        o, lse, dq, dk, dv, tq, tk, dg = outs
        op.value(q, k, v, o, lse=lse)
        op.vjp(q, k, v, o, lse, do, dq=dq, dk=dk, dv=dv)
        rot.vjp(freq, dq, tq, dyk=dk, dk=tk, q=q, k=k, gq=g, gk=g, dgq=dg)

    def outs():
        return [torch.empty_like(q), torch.empty(b, h, n, device=DEV), *(torch.empty_like(x) for x in (q, k, v, q, k, g))]

    captured, eager, mine = ops(), ops(), outs()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(*captured, mine)
    for step in range(3):
        q.mul_(1.1)
        for x in mine:
            x.fill_(9.0)
        graph.replay()
        again = outs()
        call(*eager, again)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(mine, again)), step


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_single_tokens_of_packed_projections(dtype):
    """One token a sequence, rotated in place and then read where the projection left
    it, its gradients side by side in one buffer."""
    hip.init(0)
    b, h, kv, d = 5, 4, 2, 64
    q, k, v, do = tensors(dtype, b, h, kv, 1, 1, d)
    packed, grads = torch.cat((q, k, v), 2).to(DEV), torch.full((b, 1, h + 2 * kv, d), 9.0, dtype=q.dtype, device=DEV)
    (Q, K, V), (dq, dk, dv) = (x.split((h, kv, kv), 2) for x in (packed, grads))
    freq, at = torch.from_numpy(hip.rotary_frequencies(d)), torch.arange(b)[:, None] * 100
    hip.HeadRotary(dtype, b, 1, h, kv, d).value(Q, freq.to(DEV), Q, k=K, yk=K, at=at.to(DEV))
    for x, y in ((q, Q), (k, K)):
        A.check("y", y, *A.rotary(dtype, x, None, freq, at, d, False, 0.0, False))
    assert torch.equal(V.cpu(), v)
    q, k = Q.cpu(), K.cpu()
    op = hip.Attention(dtype, b, h, kv, 1, 1, d, causal=True)
    o, lse = torch.empty(b, 1, h, d, dtype=q.dtype, device=DEV), torch.empty(b, h, 1, device=DEV)
    op.value(Q, K, V, o, lse=lse)
    op.vjp(Q, K, V, o, lse, do.to(DEV), dq=dq, dk=dk, dv=dv)
    case = A.Case(dtype, q, k, v, A.allowed(b, 1, 1, True), op.scale, do)
    A.check("o", o, *case.value()["o"])
    want = case.vjp(o.cpu(), lse.cpu())
    for name, got in (("dq", dq), ("dk", dk), ("dv", dv)):
        A.check(name, got, *want[name])
