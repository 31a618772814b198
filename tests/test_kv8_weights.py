"""The rounding of the attention weights over the 8-bit cache, on the CPU.

A weight is held as an integer of 32 bits (two halves where more rows share the pages) of the largest value of
softmax weight * value scale. This model of that rounding says how much of the output it costs when one position is
2^n times louder than the others but weighs next to nothing: its block's other positions are held as 0 and still have
the largest weights. Blocks whose scale is not within 2^8 below the reference are therefore added in fp32."""
import numpy as np
import pytest

import kv8_model as model

SPREAD = 8
FIXED = 4294967040.0


def emulate(p, values, exps, hide):
    """The output for softmax weights p (largest 1) of [positions], values [positions][dim] held with exps [blocks]."""
    e = np.repeat(exps, model.BLOCK)[:len(p)].astype(np.float64)
    if hide:
        ref = min(exps.max(), exps.min() + SPREAD)
        far = (e > ref) | (e < ref - SPREAD)
    else:
        ref, far = exps[0], np.zeros(len(p), bool)
    w = p * 2.0 ** (e - ref)
    top = w[~far].max() if not far.all() else 1.0
    held = np.where(far, w, np.rint(w / top * FIXED) / FIXED * top)
    codes = values / 2.0 ** e[:, None]
    return (held @ codes) * 2.0 ** ref / (held * 2.0 ** (ref - e)).sum()


def worst(louder, drop, hide, seed=0):
    """The error relative to the sum of the output's terms."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((64, 1, 32))
    x[5] *= 2.0 ** louder
    h = model.Held(1, 32)
    h.append(x)
    p = np.exp(-rng.exponential(1.0, 64))
    p /= p.max()
    p[5] = 2.0 ** -drop
    v = h.values()[:, 0]
    want, size = (p @ v) / p.sum(), (p @ np.abs(v)) / p.sum()
    return (np.abs(emulate(p, v, h.exps[:, 0], hide) - want) / size).max()


@pytest.mark.parametrize("louder,drop", [(0, 3), (4, 10), (8, 12), (14, 200), (20, 200), (28, 200), (34, 200), (40, 200),
                                         (20, 20), (40, 40), (40, 33), (70, 60)])
def test_a_loud_position_costs_the_others_nothing(louder, drop):
    # 64 weights, each off by 2^-33 of the largest at the bottom of the range (2^8), of terms that add up to an eighth
    # of the largest at least
    assert worst(louder, drop, True) <= 64 * 2.0 ** (SPREAD - 33) * 8


def test_the_model_sees_what_one_scale_for_all_would_cost():
    assert worst(20, 200, False) > 1e-5 and worst(28, 200, False) > 1e-3 and worst(40, 200, False) > 0.25
