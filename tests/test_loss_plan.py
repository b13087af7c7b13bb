"""The branches of a recorded sequence with losses among its steps, on the CPU
under AddressSanitizer and UndefinedBehaviorSanitizer: the spans that a loss
step gives the planner (presk_amd/csrc/loss_buffers.hpp) order it after what it
reads and before what overwrites that, and no other."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "presk_amd", "csrc")
VALUE, GRAD = 1, 2
F32, BF16 = 1, 2       # the conversions' type codes

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("plan") / "loss_plan")
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-fno-omit-frame-pointer",
           "-I", CSRC, "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "native", "loss_plan.cpp"),
           os.path.join(CSRC, "ir.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return out


class Memory:
    """Names to addresses, 1 MiB apart (0: null)."""

    def __init__(self):
        self.at = {}

    def __call__(self, name):
        return 0 if name is None else self.at.setdefault(name, (len(self.at) + 1) << 20)


ORDER = ("x", "w", "index", "teacher", "loss", "lse", "mean", "ct", "dx", "dw", "flag", "work")


def loss(mem, what, head=True, rows=8, model=64, vocab=100, top=0, **bufs):
    bufs = {"index": "y", "flag": "flag", **({"w": "w"} if head else {}), **bufs}
    ptrs = " ".join(str(mem(bufs.get(n))) for n in ORDER)
    return f"L {int(head)} {what} f32 {rows} {model if head else 0} {vocab} {top} {ptrs} 4096"


def convert(mem, src, dst, n):
    return f"C {mem(src)} {mem(dst)} {mem('flag')} {F32} {BF16} {n}"


def ordered(driver, tmp_path, lines, branches):
    """Every pair (i, j) of steps of which the plan runs i before j."""
    f = tmp_path / "seq.txt"
    f.write_text("\n".join(lines) + "\n")
    r = subprocess.run([driver, str(f), str(branches)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stderr[-3000:])
    plan = [[int(x) for x in ln.split()] for ln in r.stdout.splitlines()]
    assert len(plan) == len(lines)
    before = []
    for j, (lane, *waits) in enumerate(plan):
        mine = set()
        for i in waits + [i for i in range(j) if plan[i][0] == lane][-1:]:
            mine |= before[i] | {i}
        before.append(mine)
    return {(i, j) for j, s in enumerate(before) for i in s}


def sequences(mem):
    """(steps, the pairs that must be ordered, the pairs that need not be)."""
    step = dict(loss="l", mean="m", dx="dx", dw="dw", x="x", work="k1")
    value = dict(x="x", loss="l", lse="s", mean="m", work="k1")
    yield "a shared workspace", [loss(mem, 3, **step), loss(mem, 3, **{**step, "loss": "l2", "mean": "m2", "dx": "dx2", "dw": "dw2"})], {(0, 1)}, set()
    yield "nothing shared but inputs and the flag", [loss(mem, 3, **step), loss(
        mem, 3, **{**step, "loss": "l2", "mean": "m2", "dx": "dx2", "dw": "dw2", "work": "k2"})], set(), {(0, 1)}
    yield "a gradient from a value's sums", [
        loss(mem, VALUE, **value), loss(mem, GRAD, x="x", lse="s", mean="m", dx="dx", work="k2"),
        loss(mem, GRAD, x="x", lse="other", mean="m", dx="dx2", work="k3"), loss(mem, GRAD, x="x", lse="other", ct="c", dx="dx3", work="k4"),
    ], {(0, 1), (0, 2)}, {(1, 2), (0, 3)}
    yield "a cotangent that is read next", [loss(mem, 3, **step), convert(mem, "dx", "dx16", 8 * 64), convert(mem, "dw", "dw16", 6400),
                                            convert(mem, "m", "m16", 2), convert(mem, "l", "l16", 8)], {(0, 1), (0, 2), (0, 3), (0, 4)}, {(1, 2)}
    yield "inputs overwritten after", [loss(mem, VALUE, top=2, teacher="t", **value), convert(mem, "a", "x", 8 * 64), convert(mem, "a", "w", 10),
                                       convert(mem, "a", "t", 16), convert(mem, "a", "y", 8)], {(0, 1), (0, 2), (0, 3), (0, 4)}, set()
    yield "states made before", [convert(mem, "a", "x", 8 * 64), convert(mem, "b", "c", 8), loss(mem, GRAD, x="x", lse="s", ct="c", dx="dx", work="k1")], {
        (0, 2), (1, 2)}, {(0, 1)}
    yield "given logits", [convert(mem, "a", "z", 800), loss(mem, 3, head=False, top=2, x="z", teacher="t", dx="dz", loss="l", work="k1"),
                           convert(mem, "dz", "d16", 800)], {(0, 1), (1, 2)}, set()
    # (an output that this call does not write orders nothing)
    yield "a value that names a gradient", [loss(mem, VALUE, dx="dx", **value), convert(mem, "dx", "dx16", 512)], set(), {(0, 1)}


@pytest.mark.parametrize("n", range(8))
def test_the_plan_orders_what_meets(driver, tmp_path, n):
    mem = Memory()
    what, lines, must, free = list(sequences(mem))[n]
    for branches in (2, 4, 8):
        got = ordered(driver, tmp_path, lines, branches)
        assert must <= got, (what, branches, must - got)
    assert not free & got, (what, free & got)
    assert ordered(driver, tmp_path, lines, 1) == {(i, j) for j in range(len(lines)) for i in range(j)}
