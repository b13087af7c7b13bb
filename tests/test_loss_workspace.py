"""What a head's loss takes of workspace, term by term, as loss.hip's head
states it: past the 4 GiB of logits that a call of both keeps, and for the value
or the gradient alone, it grows with the vocabulary by the row sums'
partials and, with more than four slots a row, by the lists of their blocks."""
import pytest

from presk_amd import hip

MIB = 1 << 20
VOCABS = [32000, 128256, 1 << 20, (1 << 22) - 64]


def up(n, to):
    return -(-n // to) * to


def most(dtype, rows, model, vocab, top, kind):
    """An upper bound, in bytes."""
    half = dtype != "f32"
    b = 64 << 10                                    # each buffer's rounding to 256 bytes
    b += rows * (8 * top + 4 * 8)                   # slots, entropies; counts, lse, loss, factors
    if half and top > 4:
        b += 2 * rows * (up(vocab, 64) // 64 + 1)   # the slots' first of each 64 columns
    if kind != "vjp":
        # maximum, sum and target of a row's tile; in f32 of its piece
        tile = 128 if half else 256 if rows >= 1024 else 2048
        b += 12 * rows * (up(vocab, tile) // tile)
    if kind != "value" or not half:
        # a piece's cotangent, in f32 its logits: 128 MiB, or all of logits of 256 MiB
        piece = max(256 * up(rows, 64) * (2 if half else 4), 128 * MIB)
        if 4 * rows * up(vocab, 4) <= 256 * MIB:
            piece = max(piece, (2 if half else 4) * up(rows, 64) * up(vocab, 256))
        b += piece
    if kind != "value":
        b += 4 * rows * up(model, 4)                # dx summed over the pieces
    # a product's shares of k: a round of the CUs' tiles each, of both gradients
    return b + 2 * 64 * MIB


@pytest.mark.parametrize("kind", ["value", "vjp", "step"])
@pytest.mark.parametrize("top", [0, 4, 5, 64])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [8192, 65536, 1 << 20])
def test_the_terms(dtype, rows, top, kind):
    model = 256
    for vocab in VOCABS:
        if kind == "step" and 4 * rows * up(vocab, 4) <= 4096 * MIB:
            continue    # kept whole
        got = hip.HeadLoss(dtype, rows, model, vocab, top=top).workspace(kind)
        assert got <= most(dtype, rows, model, vocab, top, kind), (vocab, got / MIB, most(dtype, rows, model, vocab, top, kind) / MIB)


@pytest.mark.parametrize("top,kind,per", [(0, "value", 12), (4, "value", 12), (5, "value", 20), (64, "value", 20), (0, "vjp", 0), (64, "vjp", 8),
                                          (0, "step", 12), (64, "step", 20)])
def test_the_growth_with_the_vocabulary(top, kind, per):
    """Bytes a row and 256 columns (the tiles of many rows) in 16-bit storage."""
    rows, at = 65536, [1 << 20, 1 << 21]
    a, b = (hip.HeadLoss("bf16", rows, 256, v, top=top).workspace(kind) for v in at)
    assert abs((b - a) - per * rows * (at[1] - at[0]) // 256) <= 2 * MIB


def test_logits_that_are_kept():
    """Both in one call, up to 4 GiB of f32 logits: those and their 16-bit
    cotangent; in f32 the one is written over the other."""
    for dtype, bytes_ in (("bf16", 6), ("f16", 6), ("f32", 4)):
        need = hip.HeadLoss(dtype, 8192, 4096, 131072).workspace("step")
        assert bytes_ * 8192 * 131072 <= need <= bytes_ * 8192 * 131072 + 256 * MIB
