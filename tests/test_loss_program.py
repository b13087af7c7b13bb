"""Losses as steps of a program, without a GPU: what add_loss and a builder's
head_loss refuse, and what a program's steps read."""
import pytest

from presk_amd import gpt, hip
from presk_amd import lower as L
from presk_amd.gpt import A, Builder
from presk_amd.program import Program

HEAD = {"x": "x", "w": "w", "index": "y"}


def program():
    p = Program("t", hip.FAST)
    p.add_loss("step", "f32", 8, 100, {**HEAD, "loss": "l", "lse": "s", "mean": "m", "dx": "dx", "dw": "dw"}, model=64)
    return p


@pytest.mark.parametrize("kind,bufs,text", [
    ("step", {**HEAD, "mean": "m2", "dx": "dx"}, "buffer dx, a loss's dx, is another step's output"),
    ("value", {**HEAD, "loss": "l"}, "buffer l, a loss's loss, is another step's output"),
    ("value", {**HEAD, "loss": "a", "lse": "a"}, "buffer a, a loss's lse, is another step's output"),
    ("both", {**HEAD, "loss": "a"}, "kind 'both'"),
    ("value", {**HEAD, "loss": "a", "logits": "z"}, "no argument logits"),
])
def test_a_buffer_is_one_steps_output(kind, bufs, text):
    p = program()
    with pytest.raises(ValueError, match=text):
        p.add_loss(kind, "f32", 8, 100, bufs, model=64)
    assert len(p.losses) == 1


def test_launches_and_masks_count_too():
    p = program()
    low = L.dot([gpt.O(A(8, 64), "real"), gpt.O(A(64, 100), "real")], "f32")
    with pytest.raises(ValueError, match="buffer dx is a loss's output"):
        p.add(low, ["x", "w"], "dx")
    p.add(low, ["x", "w"], "z")
    with pytest.raises(ValueError, match="buffer z, a loss's dx"):
        p.add_loss("vjp", "f32", 8, 100, {**HEAD, "lse": "s", "mean": "m", "dx": "z"}, model=64)
    p.add_mask("drop", 0, 0.5, "f32", 512)
    with pytest.raises(ValueError, match="buffer drop, a loss's dx"):
        p.add_loss("vjp", "f32", 8, 100, {**HEAD, "lse": "s", "mean": "m", "dx": "drop"}, model=64)
    # what another step wrote may be read
    p.add_loss("vjp", "f32", 8, 100, {**HEAD, "lse": "s", "mean": "m", "dx": "again"}, model=64)


def test_two_heads_of_one_program():
    p = Program("t", hip.FAST)
    b = Builder(p, "f32")
    b.input("x", A(("batch", 2), ("seq", 4), ("model", 64))), b.input("w", A(("model", 64), ("vocab", 100)))
    b.input("y", A(("batch", 2), ("seq", 4)), "idx")
    first = b.head_loss("x", "w", "y", "step")
    with pytest.raises(ValueError, match="another step's output"):
        b.head_loss("x", "w", "y", "step")
    second = b.head_loss("x", "w", "y", "step", name="again.")
    assert not set(first.values()) & set(second.values()) and len(p.losses) == 2
    with pytest.raises(ValueError, match="kind 'vjp'"):
        b.head_loss("x", "w", "y", "vjp", name="third.")


def test_a_views_buffer_is_its_bases():
    p = Program("t", hip.FAST)
    b = Builder(p, "f32")
    b.input("x", A(("rows", 8), ("model", 64))), b.input("flat", A(("n", 6400))), b.input("ids", A(("b", 2), ("s", 4)), "idx")
    b.view("flat", A(("model", 64), ("vocab", 100)), "w"), b.view("ids", A(("rows", 8)), "y")
    b.head_loss("x", "w", "y", "value")
    assert [name for name, _ in p.input_specs()] == ["x", "flat", "ids"]
