"""Attention and head rotations as steps of a program, without a GPU: what they
refuse, what they read, and that a program without them is as it was."""
import numpy as np
import pytest

from presk_amd import configs, gpt, hip, llama
from presk_amd import lower as L
from presk_amd.gpt import A, Builder
from presk_amd.program import Program

SIZES = dict(dtype="f32", batch=2, heads=2, kv_heads=1, q_len=4, k_len=4, head_dim=8, causal=True)
QKV = {"q": "q", "k": "k", "v": "v"}


def program():
    p = Program("t", hip.FAST)
    p.add_attention("value", {**QKV, "o": "o", "lse": "s"}, **SIZES)
    return p


@pytest.mark.parametrize("kind, bufs, text", [
    ("value", {**QKV, "o": "o"}, "buffer o, attention's o, is another step's output"),
    ("vjp", {**QKV, "o": "o", "lse": "s", "do": "d", "dq": "g", "dk": "g"}, "buffer g, attention's dk, is another step's output"),
    ("step", {**QKV, "o": "p"}, "kind is 'step'"),
    ("value", {**QKV, "o": "p", "bias": "b"}, "no argument bias"),
])
def test_steps_that_are_refused(kind, bufs, text):
    p = program()
    with pytest.raises(ValueError, match=text):
        p.add_attention(kind, bufs, **SIZES)
    assert len(p.ops) == 1


def test_an_output_is_one_steps():
    p = program()
    with pytest.raises(ValueError, match="buffer o is an operator's output"):
        p.add(L.dot([gpt.O(A(8, 8), "real"), gpt.O(A(8, 8), "real")], "f32"), ["x", "w"], "o")
    with pytest.raises(ValueError, match="buffer s, a loss's dx, is another step's output"):
        p.add_loss("step", "f32", 8, 100, {"x": "x", "w": "w", "index": "y", "dx": "s"}, model=64)
    with pytest.raises(ValueError, match="buffer o, a rotation's yq"):
        p.add_head_rotary("value", {"q": "q", "freq": "f", "yq": "o"}, dtype="f32", batch=2, seq=4, heads=2, kv_heads=0, head_dim=8)


def test_what_the_steps_read():
    p = program()
    p.add_head_rotary("value", {"q": "o", "freq": "f", "at": "at", "yq": "r"}, dtype="f32", batch=2, seq=4, heads=2, kv_heads=0, head_dim=8)
    p.add_attention("value", {**QKV, "q": "r", "o": "z", "mask": "m", "lens": "n"}, **{**SIZES, "causal": False, "mask_cols": 4})
    assert dict(p.input_specs()) == {"q": ("f32", 128), "k": ("f32", 64), "v": ("f32", 64), "o": ("f32", 128), "f": ("f64", 4), "at": ("i64", 8),
                                     "r": ("f32", 128), "m": ("int8", 32), "n": ("i64", 2)}


def test_programs_that_are_refused():
    s = gpt.TINY
    with pytest.raises(ValueError, match="E7005.*FAST mode"):
        gpt.build(s, "f32", mode=hip.EXACT, fused_attention=True)
    with pytest.raises(ValueError, match="E7005.*dropout"):
        gpt.build(s, "f32", dropout=0.2, fused_attention=True)
    with pytest.raises(hip.HipError, match="E7005"):
        gpt.build(s, "e8m15", fused_attention=True)
    with pytest.raises(ValueError, match="E7005.*FAST mode"):
        llama.build(llama.TINY, "f32", mode=hip.EXACT, fused_attention=True)


def test_the_steps_of_the_models():
    """One a layer forward and one back, and no buffer of [seq, seq]."""
    s = gpt.TINY
    p, b, names = gpt.build(s, "f32", fused_attention=True)
    assert [(st.name, st.kind) for st in p.ops] == [("Attention", "value")] * s.L + [("Attention", "vjp")] * s.L
    assert sorted(names["grads"]) == sorted(gpt.build(s, "f32")[2]["grads"])
    assert not any(n.endswith((".scores", ".probs", "mask")) for n in b.axes)
    p, b, _ = llama.build(llama.TINY, "f32", fused_attention=True)
    assert [st.name for st in p.ops] == ["HeadRotary", "Attention"] * llama.TINY.L
    assert not any(n.endswith((".scores", ".probs", "mask")) for n in b.axes)


def test_views_and_axes():
    p = Program("t", hip.FAST)
    b = Builder(p, "bf16")
    b.input("flat", A(("n", 2 * 4 * 16))), b.input("kv", A(("batch", 2), ("seq", 4), ("model", 8)))
    q = b.view("flat", A(("batch", 2), ("seq", 4), ("model", 16)), "q")
    o, lse = b.attention(q, "kv", "kv", 2, 1, keep=True, name="o")
    assert p.ops[0].bufs == {"q": "flat", "k": "kv", "v": "kv", "o": "o", "lse": "o.lse"}
    assert [a.len for a in b.axes[o]] == [2, 4, 16] and [a.len for a in b.axes[lse]] == [2, 2, 4]
    grads = b.attention_vjp(q, "kv", "kv", o, lse, "do", 2, 1, name="g")
    assert grads == ("g.dq", "g.dk", "g.dv") and [[a.len for a in b.axes[g]] for g in grads] == [[2, 4, 16], [2, 4, 8], [2, 4, 8]]


def test_a_masks_host_values():
    """Anything but 0 is a key that is read, and a mask without a batch is every
    sequence's."""
    p = Program("t", hip.FAST)
    p.add_attention("value", {**QKV, "o": "o", "mask": "m"}, **{**SIZES, "causal": False, "mask_cols": 4})
    rng = np.random.default_rng(1)
    want = rng.random((2, 4, 4)) < 0.5
    for m in (want, want.astype(np.uint8) * 255, want * 256, want * 0.25, np.where(want, -1.0, 0.0)):
        got = configs.storage_inputs(p, {"m": m})["m"]
        assert got.dtype == np.uint8 and ((got != 0) == want.ravel()).all()
    got = configs.storage_inputs(p, {"m": want[0]})["m"]
    assert got.size == 32 and ((got.reshape(2, 4, 4) != 0) == want[0]).all()
