"""Why one product is enough to quantise a bf16 row (i8_quantize_kernel): over all pairs of bf16 mantissas, an element
times the moved reciprocal of the scale rounds to the integer nearest x / s, ties to even. Powers of two change nothing,
but where the scale is the smallest one, whose reciprocal is exact."""
import numpy as np


def quotients(top, x):
    """(the kernel's integers, whether each is nearest x / s with ties to even): numbers of 32 bits, exact in 64."""
    s = (np.float64(top) / 127).astype(np.float32)
    small = s < np.float32(2.0 ** -126)
    s = np.where(small, np.float32(2.0 ** -126), s)
    inverse = (1.0 / s.astype(np.float64)).astype(np.float32)  # rounded once more than 64 bits: the test below is of what it gives
    over = s.astype(np.float64) * 127 - top
    nudge = np.where(s == np.float32(2.0 ** -126), 0, np.sign(over)).astype(np.int32)
    moved = (inverse.view(np.int32) - nudge).view(np.float32).astype(np.float64)
    got = np.rint(x * moved)  # exact products; 1.5 * 2^23 more rounds them to integers, ties to even
    # x / s lies within half a step of `got`, and on a tie `got` is even: all products here are exact
    off = 2 * (np.abs(x) - np.abs(got) * s.astype(np.float64))
    return got, (np.abs(off) < s) | ((np.abs(off) == s) & (got % 2 == 0))


def test_every_pair_of_mantissas():
    m = np.arange(128, 256, dtype=np.float64)
    top, x, j = np.meshgrid(m, m, np.arange(0, 12), indexing="ij")
    x = x * 2.0 ** -j
    keep = x <= top
    for exponent in (-7, 0, 90, -118):
        got, right = quotients((top * 2.0 ** exponent)[keep], (x * 2.0 ** exponent)[keep])
        assert right.all() and (np.abs(got) <= 127).all()
        ties = np.abs(np.abs(x * 254 / top)[keep] % 2 - 1) < 1e-9
        assert ties.sum() > 100  # quotients of k + 1/2 but for the scale's rounding


def test_rows_of_the_smallest_numbers():
    """bf16 numbers down to 2^-133, with scales at and around the smallest."""
    top = np.concatenate([np.arange(1, 256) * 2.0 ** -133, np.arange(128, 256) * 2.0 ** -127, np.arange(128, 256) * 2.0 ** -120])
    for t in top:
        x = np.concatenate([np.arange(0, 256) * 2.0 ** e for e in (-133, -130, -127, -120)])
        x = x[x <= t]
        got, right = quotients(np.full(len(x), t), x)
        assert right.all() and (np.abs(got) <= 127).all()


def test_without_the_move_ties_go_wrong():
    """What the move is there for."""
    top, x = np.meshgrid(np.arange(128, 256, dtype=np.float64), np.arange(128, 256, dtype=np.float64) / 2, indexing="ij")
    s = (top / 127).astype(np.float32)
    got = np.rint(x * (1.0 / s.astype(np.float64)).astype(np.float32).astype(np.float64))
    off = 2 * (x - got * s.astype(np.float64))
    assert (np.abs(off) > s).any()
