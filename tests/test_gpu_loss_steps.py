"""Every kind of loss as a step of a program (Program.add_loss) on the device,
eagerly and as one graph, bit for bit what the same calls give by themselves
(which tests/test_gpu_loss.py holds against float64)."""
import numpy as np
import pytest

from presk_amd import configs, hip
from presk_amd.gpt import Builder
from presk_amd.program import Program, nbytes

pytestmark = pytest.mark.gpu

GIVEN = {"x": "z", "index": "zi", "teacher": "zt"}
TIED = {"x": "x", "w": "w", "index": "ti", "teacher": "tt"}
PLAIN = {"x": "x", "w": "v", "index": "y"}
# kind, rows, model, vocab, top, tied, T, buffers: a distillation of given
# logits; a tied head's distillation, its value, then its gradient from the
# value's lse and mean; a head's cross entropy, its value, then its gradient for
# a cotangent a row; both at once for the mean
STEPS = [
    ("step", 40, 0, 3001, 6, False, 2.0, {**GIVEN, "loss": "z.loss", "mean": "z.mean", "dx": "z.dx"}),
    ("value", 70, 72, 900, 9, True, 1.5, {**TIED, "loss": "t.loss", "lse": "t.lse", "mean": "t.mean"}),
    ("vjp", 70, 72, 900, 9, True, 1.5, {**TIED, "lse": "t.lse", "mean": "t.mean", "dx": "t.dx", "dw": "t.dw"}),
    ("value", 70, 72, 500, 0, False, 1.0, {**PLAIN, "lse": "p.lse"}),
    ("vjp", 70, 72, 500, 0, False, 1.0, {**PLAIN, "lse": "p.lse", "ct": "ct", "dx": "p.dx", "dw": "p.dw"}),
    ("step", 70, 72, 500, 0, False, 1.0, {**PLAIN, "loss": "q.loss", "mean": "q.mean", "dw": "q.dw"}),
]


def inputs(seed):
    g = np.random.default_rng(seed)
    ti = g.integers(0, 900, size=(70, 9))
    ti[g.random((70, 9)) < 0.2] = -1
    ti[5] = -1
    y = g.integers(0, 500, size=70)
    y[3::7] = -1
    f = lambda *s: g.standard_normal(s).astype(np.float32)  # noqa: E731
    return {"z": 2 * f(40, 3001), "zi": g.integers(0, 3001, size=(40, 6)), "zt": f(40, 6), "x": f(70, 72), "w": 0.3 * f(900, 72),
            "v": 0.3 * f(72, 500), "ti": ti, "tt": f(70, 9), "y": y, "ct": 1 + 0.1 * f(70)}


def alone(p, dtype):
    """The same calls over the program's own inputs, into buffers beside its."""
    out = {}

    def buffer(name, spec):
        if name in out:
            return out[name]
        return out.setdefault(name, hip.DeviceBuffer(nbytes(*spec)))

    for st, (kind, rows, model, vocab, top, tied, t, names) in zip(p.losses, STEPS):
        op = hip.HeadLoss(dtype, rows, model, vocab, tied, top, t) if model else hip.Distill(dtype, rows, vocab, top, t)
        writes, specs = st.writes(), st.specs()
        bufs = {a: out[b] if b in out else p.bufs.dev[b] if a not in writes else buffer(b, specs[a]) for a, b in names.items()}
        {"value": op.value, "vjp": op.vjp, "step": op.value_and_grad}[kind](**bufs)
        hip.sync()
    return {b: out[b].download(np.uint8).tobytes() for b in out}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_steps_are_the_calls(dtype):
    p = Program("losses", hip.FAST)
    for kind, rows, model, vocab, top, tied, t, names in STEPS:
        p.add_loss(kind, dtype, rows, vocab, names, model=model, top=top, tied=tied, temperature=t)
    p.compile()
    configs.load_inputs(p, inputs(1))
    p.prepare()
    p.run()
    hip.sync()
    outs = [b for st in p.losses for b in (st.bufs[a] for a in st.writes())]
    for seed in (None, 2, 3, 4):
        if seed is not None:
            # recorded once, then replayed over other inputs, its outputs poisoned
            if seed == 2:
                p.record()
            for name, arr in configs.storage_inputs(p, inputs(seed)).items():
                p.bufs.upload(name, arr)
            for b in outs:
                p.bufs.dev[b].upload(np.full(p.bufs.dev[b].nbytes, 0x50 + seed, np.uint8))
            hip.sync()
            p.run()
            hip.sync()
        want = alone(p, dtype)
        assert sorted(want) == sorted(outs)
        assert [b for b in outs if p.bufs.dev[b].download(np.uint8).tobytes() != want[b]] == [], seed
        values = p.bufs.download("z.mean").view(np.float32)
        assert np.isfinite(values).all() and values[1] == 40.0 and p.bufs.download("q.mean").view(np.float32)[1] == 60.0
    p.check_overflow()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_heads_of_one_program(dtype):
    """Each has its own outputs: those of a program with it alone."""
    from presk_amd.gpt import A
    got = []
    for heads in ((0, 1), (0,), (1,)):
        p = Program("heads", hip.FAST)
        b = Builder(p, dtype)
        b.input("x", A(("rows", 70), ("model", 72))), b.input("y", A(("rows", 70)), "idx")
        names = []
        for h in heads:
            b.input(f"w{h}", A(("model", 72), ("vocab", 500)))
            names.append(b.head_loss("x", f"w{h}", "y", "step", name=f"h{h}."))
        p.compile()
        host = inputs(1)
        configs.load_inputs(p, {"x": host["x"], "y": host["y"], "w0": host["v"], "w1": 0.5 * host["v"]})
        p.prepare()
        p.run()
        hip.sync()
        got.append([{k: p.bufs.dev[v].download(np.uint8).tobytes() for k, v in n.items()} for n in names])
    assert got[0] == got[1] + got[2] and got[0][0] != got[0][1]
