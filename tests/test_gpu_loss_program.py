"""Programs whose head and loss are one step (gpt.build(fused_head=True),
llama.build(score=True)) on the device, against the same programs with the
logits, in the interpreter's order."""
import numpy as np
import pytest

from presk_amd import configs, gpt, hip, llama
from tests import fmt

pytestmark = pytest.mark.gpu


def run(p, host):
    p.compile()
    configs.load_inputs(p, host)
    p.prepare()
    p.run()
    hip.sync()
    p.check_overflow()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_gpt_step(dt):
    """Loss and every gradient within the bands that a FAST step is held to
    against EXACT (f32 1e-5 and 1e-4 of a gradient's largest value, bf16 2e-2
    and 6e-2; f16 between them); as one graph the same bits, three times."""
    s = gpt.TINY
    host = gpt.host_inputs(s)
    ref, _, rn = gpt.build(s, dt, train=True, mode=hip.EXACT)
    run(ref, host)
    p, _, names = gpt.build(s, dt, train=True, fused_head=True)
    run(p, host)
    loss = p.bufs.download(names["loss"]).view(np.float32)
    want = float(fmt.decode(ref.bufs.download(rn["loss"]), dt)[0])
    assert loss[1] == s.B * s.T
    assert abs(float(loss[0]) - want) <= {"f32": 1e-5, "f16": 5e-3, "bf16": 2e-2}[dt] * abs(want)
    assert set(names["grads"]) == set(rn["grads"])
    grads = {n: fmt.decode(p.bufs.download(b), dt).astype(np.float64) for n, b in names["grads"].items()}
    refs = {n: fmt.decode(ref.bufs.download(b), dt).astype(np.float64) for n, b in rn["grads"].items()}
    floor = 1e-3 * max(np.max(np.abs(r)) for r in refs.values())
    for n, r in refs.items():
        err = np.max(np.abs(grads[n] - r)) / max(np.max(np.abs(r)), floor)
        assert err < {"f32": 1e-4, "f16": 3e-2, "bf16": 6e-2}[dt], (n, err)
    outs = [names["loss"], "ce", "d.xf"] + list(names["grads"].values())
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


def test_gpt_value_with_dropout_and_optimizer():
    """The forward alone; a step with dropout and the optimizer after it, whose
    updated head follows from the fused gradient."""
    s = gpt.TINY
    host = gpt.host_inputs(s)
    p, _, names = gpt.build(s, "f32", train=False, fused_head=True)
    run(p, host)
    q, _, qn = gpt.build(s, "f32", train=False)
    run(q, host)
    a, b = p.bufs.download(names["loss"]).view(np.float32)[0], fmt.decode(q.bufs.download(qn["loss"]), "f32")[0]
    assert abs(a - b) <= 1e-5 * abs(b)
    host.update(gpt.optimizer_inputs(s, 200, 1000))
    heads = []
    for fused in (True, False):
        p, _, names = gpt.build(s, "f32", train=True, dropout=0.2, optimizer=True, fused_head=fused)
        run(p, host)
        # AdamW divides a gradient by its own size: what may differ is a
        # gradient near 0, so the moment is compared, which is linear in it
        heads.append(fmt.decode(p.bufs.download(names["adamw"]["head"][1]), "f32").astype(np.float64))
    assert np.max(np.abs(heads[0] - heads[1])) <= 1e-4 * np.max(np.abs(heads[1]))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_llama_score(dt):
    """Each token's loss against the one of the logits that the forward
    stores (in bf16 rounded, so a logit is off by up to 2^-8 of itself there,
    and the states before them by the FAST band)."""
    s = llama.TINY
    host = llama.host_inputs(s)
    host["y"] = np.random.default_rng(3).integers(0, s.V, size=(s.B, s.T), dtype=np.int64)
    host["y"][0, 1] = -1
    p, _, names = llama.build(s, dt, score=True)
    run(p, host)
    q, _, qn = llama.build(s, dt, mode=hip.EXACT)
    run(q, host)
    z = fmt.decode(q.bufs.download(qn["logits"]), dt).astype(np.float64).reshape(-1, s.V)
    y = host["y"].ravel()
    top = z.max(-1)
    lse = top + np.log(np.exp(z - top[:, None]).sum(-1))
    want = np.where(y >= 0, lse - z[np.arange(len(y)), np.maximum(y, 0)], 0.0)
    got = p.bufs.download(names["ce"]).view(np.float32)
    tol = {"f32": 1e-5, "bf16": 5e-2}[dt] * np.max(np.abs(z)) * 2
    assert np.max(np.abs(got - want)) <= tol + 1e-5
    assert got[1] == 0.0
    mean = p.bufs.download(names["loss"]).view(np.float32)
    assert mean[1] == len(y) - 1 and abs(mean[0] - want.sum() / (len(y) - 1)) <= tol + 1e-5


def test_steps_in_a_program_are_checked():
    """A loss that reads a buffer of another type is refused (a mixed program
    gives it no conversion)."""
    from presk_amd.program import Program
    p = Program("t", hip.FAST)
    p.add_loss("value", "bf16", 8, 100, {"x": "x", "w": "w", "index": "y", "loss": "l"}, model=64)
    p.compile()
    p.declare("x", "f32", 8 * 64), p.declare("w", "bf16", 6400), p.declare("y", "i64", 8)
    with pytest.raises(ValueError, match="E7005"):
        p.prepare()
