"""hip.HeadRotary on the device against float64 (tests/attention_oracle.py)."""
import pytest

torch = pytest.importorskip("torch")

from presk_amd import hip  # noqa: E402
from tests import attention_oracle as A  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda"


def tensors(dtype, batch, seq, heads, kv, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(A.TORCH[dtype])  # noqa: E731
    return (n(batch, seq, heads, d), n(batch, seq, kv, d), n(batch, seq, heads, d), n(batch, seq, kv, d),
            (1 + 0.2 * n(d).float()).to(A.TORCH[dtype]), (1 + 0.2 * n(d).float()).to(A.TORCH[dtype]))


def run(dtype, batch, seq, heads, kv, d, rot=None, norm=True, pairs="half", at=None, gains=True, layout="bshd"):
    hip.init(0)
    q, k, dyq, dyk, gq, gk = tensors(dtype, batch, seq, heads, kv, d, seed=d + seq)
    op = hip.HeadRotary(dtype, batch, seq, heads, kv, d, rotary=rot, norm=norm, pairs=pairs, layout=layout)
    freq = torch.from_numpy(hip.rotary_frequencies(op.rotary))
    swap = (lambda x: x.transpose(1, 2).contiguous()) if layout == "bhsd" else (lambda x: x)
    Q, K, DYQ, DYK = (swap(x.to(DEV)) for x in (q, k, dyq, dyk))
    given = {"freq": freq.to(DEV), "at": None if at is None else at.to(DEV)}
    if norm and gains:
        given.update(gq=gq.to(DEV), gk=gk.to(DEV))
    yq, yk = torch.full_like(Q, 9.0), torch.full_like(K, 9.0)
    op.value(Q, yq=yq, k=K if kv else None, yk=yk if kv else None, **given)
    dq, dk = torch.full_like(Q, 9.0), torch.full_like(K, 9.0)
    dg = {n: torch.full((d,), 9.0, dtype=Q.dtype, device=DEV) for n in ("dgq", "dgk")} if norm else {}
    op.vjp(dyq=DYQ, dq=dq, dyk=DYK if kv else None, dk=dk if kv else None, **given, **dg,
           **({"q": Q, "k": K if kv else None} if norm else {}))
    where = torch.arange(seq).expand(batch, seq) if at is None else at
    worst = {}
    for n, x, g, dy, y, dx in (("q", q, gq, dyq, yq, dq), ("k", k, gk, dyk, yk, dk))[:2 if kv else 1]:
        g = g if norm and gains else None
        spec = (dtype, x, g, freq, where, op.rotary, norm, op.eps, pairs == "even")
        worst["y" + n] = A.check("y" + n, swap(y), *A.rotary(*spec))
        want = A.rotary(*spec, dy=dy)
        worst["d" + n] = A.check("d" + n, swap(dx), *want["dx"])
        if norm:
            worst["dg" + n] = A.check("dg" + n, dg["dg" + n], *want["dg"])
    print({n: round(w, 3) for n, w in worst.items()}, flush=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 64), (2, 33, 4, 2, 128), (1, 7, 3, 0, 80), (1, 5, 32, 8, 128), (3, 10, 5, 5, 96),
                                  (1, 3, 2, 1, 256), (2, 4, 2, 2, 32), (1, 3, 7, 1, 16)], ids=str)
def test_against_float64(dtype, norm, size):
    run(dtype, *size, norm=norm)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pairs", ["half", "even"])
@pytest.mark.parametrize("d, rot", [(128, 64), (80, 40), (64, 0), (96, 2), (65, 20), (33, 32), (1, 0), (255, 254), (250, 6), (40, 24)])
def test_parts_of_heads(dtype, pairs, d, rot):
    run(dtype, 2, 9, 3, 2, d, rot=rot, pairs=pairs)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_far_positions(dtype):
    at = torch.tensor([[0, 1, 131071, 1000003, -17], [5, 77777, 2 ** 24 + 1, 10 ** 8 + 7, 3]])
    run(dtype, 2, 5, 4, 2, 128, at=at)
    run(dtype, 2, 5, 4, 2, 64, at=at, norm=False, pairs="even")


def test_a_norm_without_gains():
    run("bf16", 2, 9, 4, 2, 128, gains=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_heads_before_rows(dtype):
    run(dtype, 2, 30, 4, 2, 64, layout="bhsd")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_tokens(dtype):
    """More than one of them a wave, whose gains' gradients are one sum."""
    run(dtype, 3, 1500, 6, 3, 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place(dtype):
    """The outputs may be the inputs, slices of a packed projection among them."""
    hip.init(0)
    b, n, h, kv, d = 2, 21, 4, 2, 64
    q, k, dyq, dyk, gq, gk = (x.to(DEV) for x in tensors(dtype, b, n, h, kv, d))
    freq = torch.from_numpy(hip.rotary_frequencies(d)).to(DEV)
    op = hip.HeadRotary(dtype, b, n, h, kv, d, norm=True)
    yq, yk, dq, dk = (torch.empty_like(x) for x in (q, k, q, k))
    op.value(q, freq, yq, k=k, yk=yk, gq=gq, gk=gk)
    op.vjp(freq, dyq, dq, dyk=dyk, dk=dk, q=q, k=k, gq=gq, gk=gk)
    packed, grads = torch.cat((q, k), 2), torch.cat((dyq, dyk), 2)
    (pq, pk), (pdq, pdk) = packed.split((h, kv), 2), grads.split((h, kv), 2)
    op.vjp(freq, pdq, pdq, dyk=pdk, dk=pdk, q=pq, k=pk, gq=gq, gk=gk)
    op.value(pq, freq, pq, k=pk, yk=pk, gq=gq, gk=gk)
    for got, want in ((pq, yq), (pk, yk), (pdq, dq), (pdk, dk)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_start_anywhere(dtype):
    hip.init(0)
    b, n, h, d = 2, 9, 3, 64
    q, _, _, _, gq, _ = tensors(dtype, b, n, h, 0, d)
    wide = torch.full((b, n, h, d + 3), 9.0, dtype=q.dtype, device=DEV)
    Q = wide[..., 1:d + 1]
    Q.copy_(q)
    op = hip.HeadRotary(dtype, b, n, h, 0, d, norm=True)
    freq = torch.from_numpy(hip.rotary_frequencies(d))
    op.value(Q, freq.to(DEV), Q, gq=gq.to(DEV))
    A.check("yq", Q, *A.rotary(dtype, q, gq, freq, torch.arange(n).expand(b, n), d, True, op.eps, False))
    assert (wide[..., 0] == 9).all() and (wide[..., d + 1:] == 9).all()


def test_no_tokens():
    hip.init(0)
    for b, n in ((0, 4), (4, 0)):
        x = torch.empty(b, n, 2, 64, dtype=torch.bfloat16, device=DEV)
        freq = torch.from_numpy(hip.rotary_frequencies(64)).to(DEV)
        op = hip.HeadRotary("bf16", b, n, 2, 2, 64, norm=True)
        op.value(x, freq, torch.empty_like(x), k=x, yk=torch.empty_like(x))
        dgq, dgk = (torch.full((64,), 9.0, dtype=x.dtype, device=DEV) for _ in range(2))
        op.vjp(freq, x, torch.empty_like(x), dyk=x, dk=torch.empty_like(x), q=x, k=x, dgq=dgq, dgk=dgk)
        assert (dgq == 0).all() and (dgk == 0).all()


def test_a_captured_call_replays():
    hip.init(0)
    q, k, dyq, dyk, gq, gk = (x.to(DEV) for x in tensors("bf16", 2, 40, 4, 2, 128))
    freq = torch.from_numpy(hip.rotary_frequencies(128)).to(DEV)
    at = torch.arange(40, device=DEV).expand(2, 40).contiguous()
    op = hip.HeadRotary("bf16", 2, 40, 4, 2, 128, norm=True)
    outs = [torch.empty_like(x) for x in (q, k, q, k, gq, gk)]

    def call(yq, yk, dq, dk, dgq, dgk, work):
        op.value(q, freq, yq, k=k, yk=yk, at=at, gq=gq, gk=gk)
        op.vjp(freq, dyq, dq, dyk=dyk, dk=dk, q=q, k=k, at=at, gq=gq, gk=gk, dgq=dgq, dgk=dgk, work=work)

    work = torch.empty(op.workspace("vjp"), dtype=torch.uint8, device=DEV)
    call(*outs, work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(*outs, work)
    for step in range(3):
        at.add_(1000), q.mul_(1.1)
        for x in outs:
            x.fill_(9.0)
        graph.replay()
        got = [x.clone() for x in outs]
        again = [torch.empty_like(x) for x in outs]
        call(*again, torch.empty_like(work))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, again)), step


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("size", [(1, 3, 3, 1, 64), (2, 33, 4, 2, 128), (1, 5, 7, 8, 64), (2, 9, 3, 2, 33)], ids=str)
def test_a_norm_without_eps(dtype, eps, size):
    """Lanes beyond the last head have no elements, whose norm would be infinite."""
    hip.init(0)
    b, n, h, kv, d = size
    q, k, dyq, dyk, gq, gk = tensors(dtype, *size, seed=d)
    rot = d // 2 * 2
    op = hip.HeadRotary(dtype, b, n, h, kv, d, rotary=rot, norm=True, eps=eps)
    freq = torch.from_numpy(hip.rotary_frequencies(rot))
    Q, K, DYQ, DYK, GQ, GK = (x.to(DEV) for x in (q, k, dyq, dyk, gq, gk))
    yq, yk, dq, dk = (torch.full_like(x, 9.0) for x in (Q, K, Q, K))
    dgq, dgk = torch.full_like(GQ, 9.0), torch.full_like(GK, 9.0)
    op.value(Q, freq.to(DEV), yq, k=K, yk=yk, gq=GQ, gk=GK)
    op.vjp(freq.to(DEV), DYQ, dq, dyk=DYK, dk=dk, q=Q, k=K, gq=GQ, gk=GK, dgq=dgq, dgk=dgk)
    at = torch.arange(n).expand(b, n)
    for x, g, dy, y, dx, dg in ((q, gq, dyq, yq, dq, dgq), (k, gk, dyk, yk, dk, dgk)):
        spec = (dtype, x, g, freq, at, rot, True, eps, False)
        A.check("y", y, *A.rotary(*spec))
        want = A.rotary(*spec, dy=dy)
        A.check("dx", dx, *want["dx"])
        A.check("dg", dg, *want["dg"])


@pytest.mark.parametrize("pairs", ["half", "even"])
@pytest.mark.parametrize("d", [2, 64])
def test_an_angle_of_2_30_radians(pairs, d):
    """Is right to 2^-23 of its f64 product's: whole turns are taken off without loss, so
    that what is left is f32's rounding of the angle (2^-25 at most), of its cosine
    or sine (2^-25) and of their series."""
    hip.init(0)
    n = 4096
    g = torch.Generator().manual_seed(d)
    at = (2 ** 30 - torch.randint(0, 2 ** 28, (2, n), generator=g)).contiguous()
    freq = 1.0 - torch.rand(d // 2, generator=g, dtype=torch.float64) * 0.2
    x = torch.zeros(2, n, 1, d)
    first = x[..., 0::2] if pairs == "even" else x[..., :d // 2]
    first += 1.0
    op = hip.HeadRotary("f32", 2, n, 1, 0, d, pairs=pairs)
    y = torch.empty_like(x, device=DEV)
    op.value(x.to(DEV), freq.to(DEV), y, at=at.to(DEV))
    y = y.cpu().double()
    angle = at.double()[:, :, None, None] * freq
    c, s = (y[..., 0::2], y[..., 1::2]) if pairs == "even" else (y[..., :d // 2], y[..., d // 2:])
    worst = max(float((c - torch.cos(angle)).abs().max()), float((s - torch.sin(angle)).abs().max()))
    print(f"{worst:.3g}", flush=True)
    assert worst <= 2.0 ** -23
