"""Programs whose attention is a step (gpt.build(fused_attention=True),
llama.build(fused_attention=True)) on the device, against the same programs of
nests in the interpreter's order; and a block's operators run together, as a
training step and as a cache that grows."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from presk_amd import configs, gpt, hip, llama  # noqa: E402
from presk_amd.program import Program, nbytes  # noqa: E402
from tests import attention_oracle as AO  # noqa: E402
from tests import fmt  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda"


def run(p, host):
    p.compile()
    configs.load_inputs(p, host)
    p.prepare()
    p.run()
    hip.sync()
    p.check_overflow()


def replays(p, outs):
    """As one graph the same bits, three times over poisoned outputs."""
    eager = {o: p.bufs.download(o).tobytes() for o in outs}
    p.record()
    for rep in range(3):
        for o in outs:
            p.bufs.dev[o].upload(np.full(p.bufs.dev[o].nbytes, 0x5A + rep, np.uint8))
        hip.sync()
        p.run()
        hip.sync()
        assert [o for o in outs if p.bufs.download(o).tobytes() != eager[o]] == [], rep
    p.check_overflow()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fused_head", [False, True])
def test_gpt_step(dt, fused_head):
    """Loss and every gradient within the bands that a FAST step is held to
    against EXACT (f32 1e-5 and 1e-4 of a gradient's largest value, bf16 2e-2
    and 6e-2; f16 between them)."""
    s = gpt.TINY
    host = gpt.host_inputs(s)
    ref, _, rn = gpt.build(s, dt, train=True, mode=hip.EXACT)
    run(ref, host)
    p, _, names = gpt.build(s, dt, train=True, fused_head=fused_head, fused_attention=True)
    run(p, host)
    loss = p.bufs.download(names["loss"])
    loss = float(loss.view(np.float32)[0]) if fused_head else float(fmt.decode(loss, dt)[0])
    want = float(fmt.decode(ref.bufs.download(rn["loss"]), dt)[0])
    assert abs(loss - want) <= {"f32": 1e-5, "f16": 5e-3, "bf16": 2e-2}[dt] * abs(want)
    assert set(names["grads"]) == set(rn["grads"])
    grads = {n: fmt.decode(p.bufs.download(b), dt).astype(np.float64) for n, b in names["grads"].items()}
    refs = {n: fmt.decode(ref.bufs.download(b), dt).astype(np.float64) for n, b in rn["grads"].items()}
    floor = 1e-3 * max(np.max(np.abs(r)) for r in refs.values())
    for n, r in refs.items():
        err = np.max(np.abs(grads[n] - r)) / max(np.max(np.abs(r)), floor)
        assert err < {"f32": 1e-4, "f16": 3e-2, "bf16": 6e-2}[dt], (n, err)
    replays(p, [names["loss"], "b0.om", "b1.att.dk"] + list(names["grads"].values()))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gpt_value(dt):
    s = gpt.TINY
    host = gpt.host_inputs(s)
    ref, _, rn = gpt.build(s, dt, train=False, mode=hip.EXACT)
    run(ref, host)
    p, _, names = gpt.build(s, dt, train=False, fused_attention=True)
    run(p, host)
    a, b = (fmt.decode(x.bufs.download(n["logits"]), dt).astype(np.float64) for x, n in ((p, names), (ref, rn)))
    assert np.max(np.abs(a - b)) <= {"f32": 1e-5, "bf16": 3e-2}[dt] * np.max(np.abs(b))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_llama_logits(dt):
    """Grouped heads, their rotation in one step."""
    s = llama.TINY
    host = llama.host_inputs(s)
    ref, _, rn = llama.build(s, dt, mode=hip.EXACT)
    run(ref, host)
    p, _, names = llama.build(s, dt, fused_attention=True)
    run(p, host)
    a, b = (fmt.decode(x.bufs.download(n["logits"]), dt).astype(np.float64) for x, n in ((p, names), (ref, rn)))
    assert np.max(np.abs(a - b)) <= {"f32": 2e-5, "bf16": 6e-2}[dt] * np.max(np.abs(b))
    replays(p, [names["logits"], "b0.o", "b1.rot.k"])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_steps_are_the_calls(dtype):
    """Every kind of step, its optional buffers among them, bit for bit what the
    same calls give by themselves, over inputs that change between a graph's replays."""
    b, n, h, kv, d, cols = 2, 24, 4, 2, 64, 24
    att = dict(dtype=dtype, batch=b, heads=h, kv_heads=kv, q_len=n, k_len=n, head_dim=d, mask_cols=cols)
    rot = dict(dtype=dtype, batch=b, seq=n, heads=h, kv_heads=kv, head_dim=d, rotary=32, norm=True, pairs="even")
    qkv = {"q": "yq", "k": "yk", "v": "v", "mask": "mask", "lens": "lens", "first": "first"}
    p = Program("heads", hip.FAST)
    p.add_head_rotary("value", {"q": "q", "k": "k", "freq": "freq", "at": "at", "gq": "gq", "gk": "gk", "yq": "yq", "yk": "yk"}, **rot)
    p.add_attention("value", {**qkv, "o": "o", "lse": "lse"}, **att)
    p.add_attention("vjp", {**qkv, "o": "o", "lse": "lse", "do": "do", "dq": "dyq", "dk": "dyk", "dv": "dv"}, **att)
    p.add_head_rotary("vjp", {"q": "q", "k": "k", "freq": "freq", "at": "at", "gq": "gq", "gk": "gk", "dyq": "dyq", "dyk": "dyk", "dq": "dq", "dk": "dk",
                              "dgq": "dgq", "dgk": "dgk"}, **rot)

    def inputs(seed):
        g = np.random.default_rng(seed)
        f = lambda *s: g.standard_normal(s).astype(np.float32)  # noqa: E731
        return {"q": f(b, n, h, d), "k": f(b, n, kv, d), "v": f(b, n, kv, d), "do": f(b, n, h, d), "gq": 1 + 0.1 * f(d), "gk": 1 + 0.1 * f(d),
                "freq": hip.rotary_frequencies(32), "at": g.integers(0, 10000, (b, n)), "mask": g.random((b, n, cols)) < 0.6,
                "lens": g.integers(1, n + 1, b), "first": g.integers(-3, 4, b)}

    p.compile()
    configs.load_inputs(p, inputs(1))
    p.prepare()
    outs = [st.bufs[a] for st in p.ops for a in st.writes()]
    for seed in (1, 2, 3, 4):
        if seed == 2:
            p.record()
        for name, arr in configs.storage_inputs(p, inputs(seed)).items():
            p.bufs.upload(name, arr)
        for o in outs:
            p.bufs.dev[o].upload(np.full(p.bufs.dev[o].nbytes, 0x40 + seed, np.uint8))
        hip.sync()
        p.run()
        hip.sync()
        mine = {}
        for st in p.ops:
            specs, writes = st.specs(), st.writes()
            bufs = {a: mine[x] if x in mine else p.bufs.dev[x] for a, x in st.bufs.items() if a not in writes}
            for a in writes:
                bufs[a] = mine[st.bufs[a]] = hip.DeviceBuffer(nbytes(*specs[a]))
            getattr(getattr(hip, st.name)(**st.sizes), st.kind)(**bufs)
            hip.sync()
        assert [o for o in outs if p.bufs.dev[o].download(np.uint8).tobytes() != mine[o].download(np.uint8).tobytes()] == [], seed
    p.check_overflow()


def block(x, w, gq, gk, mask, freq, h, kv, d):
    """A block's attention in float64 torch, from the definitions."""
    b, n, _ = x.shape
    qkv = (x @ w).view(b, n, h + 2 * kv, d)
    q, k, v = qkv.split((h, kv, kv), 2)
    turn = torch.polar(torch.ones((), dtype=torch.float64), torch.arange(n).double()[:, None, None] * freq)

    def head(z, g):
        z = g * z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6)
        z = torch.complex(z[..., :d // 2], z[..., d // 2:]) * turn
        return torch.cat((z.real, z.imag), -1)

    q, k = head(q, gq).transpose(1, 2), head(k, gk).transpose(1, 2).repeat_interleave(h // kv, 1)
    p = torch.softmax((q @ k.transpose(2, 3) / math.sqrt(d)).masked_fill(~mask, -math.inf), -1)
    return (p @ v.transpose(1, 2).repeat_interleave(h // kv, 1)).transpose(1, 2).reshape(b, n, h * d), qkv


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_blocks_training_step(dtype):
    """Norms, rotation and attention of a packed projection and all their
    gradients, against float64 reverse mode from the definitions: each of the four
    stages keeps a sum of at most 100 terms to 20 half steps of its type, so the whole
    to 100 of the largest value."""
    hip.init(0)
    b, n, h, kv, d, model = 2, 70, 4, 2, 64, 32
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, gq, gk, do = r(b, n, model), r(model, (h + 2 * kv) * d) * model ** -0.5, 1 + 0.1 * r(d), 1 + 0.1 * r(d), r(b, n, h * d)
    ty = AO.TORCH[dtype]
    freq = torch.from_numpy(hip.rotary_frequencies(d))
    packed = (x @ w).view(b, n, h + 2 * kv, d).to(ty)
    leaves = [packed.double().requires_grad_(), gq.to(ty).double().requires_grad_(), gk.to(ty).double().requires_grad_()]
    eye = torch.eye((h + 2 * kv) * d, dtype=torch.float64)
    mask = torch.ones(n, n, dtype=torch.bool).tril()
    o64, _ = block(leaves[0].reshape(b, n, -1), eye, leaves[1], leaves[2], mask, freq, h, kv, d)
    do = do.to(ty)
    want = torch.autograd.grad((o64 * do.double()).sum(), leaves)
    P, F, GQ, GK, DO = packed.to(DEV), freq.to(DEV), gq.to(ty).to(DEV), gk.to(ty).to(DEV), do.to(DEV).view(b, n, h, d)
    q, k, v = P.split((h, kv, kv), 2)
    rot = hip.HeadRotary(dtype, b, n, h, kv, d, norm=True)
    att = hip.Attention(dtype, b, h, kv, n, n, d, causal=True)
    yq, yk, o = torch.empty(b, n, h, d, dtype=ty, device=DEV), torch.empty(b, n, kv, d, dtype=ty, device=DEV), torch.empty(b, n, h, d, dtype=ty, device=DEV)
    lse = torch.empty(b, h, n, device=DEV)
    grads = torch.empty_like(P)
    dq, dk, dv = grads.split((h, kv, kv), 2)
    dgq, dgk = torch.empty_like(GQ), torch.empty_like(GK)
    rot.value(q, F, yq, k=k, yk=yk, gq=GQ, gk=GK)
    att.value(yq, yk, v, o, lse=lse)
    att.vjp(yq, yk, v, o, lse, DO, dq=dq, dk=dk, dv=dv)
    rot.vjp(F, dq, dq, dyk=dk, dk=dk, q=q, k=k, gq=GQ, gk=GK, dgq=dgq, dgk=dgk)
    tol = 100 * AO.HALF[dtype]
    for name, got, ref in (("o", o.view(b, n, -1), o64.detach()), ("packed", grads, want[0]), ("dgq", dgq, want[1]), ("dgk", dgk, want[2])):
        err = float((got.cpu().double() - ref).abs().max() / ref.abs().max())
        print(name, err / AO.HALF[dtype], flush=True)
        assert err <= tol, (name, err)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_cache_that_grows(dtype):
    """A prompt, then single tokens, then a tree of drafts, each over a cache with
    room left (never read: NaN) whose keys are turned as they are written: what one
    call over all of them gives, within the bounds of both."""
    hip.init(0)
    b, h, kv, d, room = 2, 4, 2, 64, 200
    ty = AO.TORCH[dtype]
    g = torch.Generator().manual_seed(2)
    n, drafts = 45, 5
    total = n + 4 + drafts
    q, k, v = (torch.randn(b, total, x, d, generator=g).to(ty) for x in (h, kv, kv))
    Q, K, V = q.to(DEV), k.to(DEV), v.to(DEV)
    F = torch.from_numpy(hip.rotary_frequencies(d)).to(DEV)
    cache_k, cache_v = (torch.full((b, room, kv, d), math.nan, dtype=ty, device=DEV) for _ in range(2))
    tree = torch.eye(drafts, dtype=torch.bool) | (torch.arange(drafts) == 0)        # the first draft, and four that follow it
    got, turned = [], []
    done = 0
    for m, kind in [(n, "causal"), (1, "causal"), (1, "causal"), (2, "causal"), (drafts, "tree")]:
        rot = hip.HeadRotary(dtype, b, m, h, kv, d)
        at = torch.arange(done, done + m, device=DEV).expand(b, m).contiguous()
        yq = torch.empty(b, m, h, d, dtype=ty, device=DEV)
        rot.value(Q[:, done:done + m], F, yq, k=K[:, done:done + m], yk=cache_k[:, done:done + m], at=at)
        cache_v[:, done:done + m] = V[:, done:done + m]
        lens, first = torch.full((b,), done + m, device=DEV), torch.full((b,), done, device=DEV)
        o = torch.empty_like(yq)
        op = hip.Attention(dtype, b, h, kv, m, room, d, causal=kind == "causal", mask_cols=drafts if kind == "tree" else 0)
        op.value(yq, cache_k, cache_v, o, lens=lens, first=first, **({"mask": tree.to(DEV)} if kind == "tree" else {}))
        got.append(o), turned.append(yq)
        done += m
    mask = torch.ones(total, total, dtype=torch.bool).tril()
    mask[-drafts:, -drafts:] = tree
    q, k, o = torch.cat(turned, 1).cpu(), cache_k[:, :total].cpu(), torch.cat(got, 1)
    case = AO.Case(dtype, q, k, v, mask.expand(b, -1, -1), d ** -0.5)
    AO.check("o", o, *case.value()["o"])
    whole = torch.empty_like(o)
    hip.Attention(dtype, b, h, kv, total, total, d, mask_cols=total).value(q.to(DEV), k.to(DEV), V, whole, mask=mask.to(DEV))
    AO.check("whole", whole, *case.value()["o"])
