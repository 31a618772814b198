"""Attention over the 8-bit cache where single elements are far from the rest: what the kernels hold in integers and
halves must keep the small ones. Against the 64-bit definition, by bounds of the sums that each output is made of."""
import numpy as np
import pytest

import kv8_model as model
from phonon_b200 import runtime as rt
from test_gpu_kv8 import Cache, dev, f64, rows

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def kind(dtype):
    return rt.ROWS_BF16 if dtype == torch.bfloat16 else rt.ROWS_F32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv_heads,group,dim,lengths,count", [
    (2, 1, 64, [40, 300], 1), (2, 4, 128, [40, 300], 1), (1, 3, 32, [70], 1), (2, 2, 64, [90], 2), (1, 2, 64, [90], 4),
    (2, 4, 128, [150], 3),
])
def test_quiet_channels_beside_a_loud_one(cuda_ok, kv_heads, group, dim, lengths, count, dtype):
    """One channel of q is 2^11 times the others and meets keys of 0: the scores are the quiet channels'. q is held in 31
    bits (22 in halves) of the row's largest, so that the quiet elements keep 19 and more, bf16's 8 all of them: the
    errors stay below the bound's dim / 8 + 10 steps of 2^-23, relative to the score's own terms."""
    rng = np.random.default_rng(dim + group)
    c = Cache(kv_heads, dim, lengths)
    keys = [rows(rng, n, kv_heads, dim, dtype) for n in lengths]
    for k in keys:
        k[..., 0] = 0
    values = [rows(rng, n, kv_heads, dim, dtype) for n in lengths]
    c.append(lengths, keys, values)
    q = rows(rng, count * len(lengths), kv_heads * group, dim, dtype)
    q[..., 0] = 2.0 ** 11 * q[..., 1:].abs().amax(-1)
    out = torch.empty_like(q)
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(c.batch(lengths, [count] * len(lengths)),
                   rt.kv8_query(q.data_ptr(), out.data_ptr(), kind(dtype), heads=kv_heads * group), ws)
    torch.cuda.synchronize()
    for i, n in enumerate(lengths):
        held = [model.Held(kv_heads, dim) for _ in range(2)]
        held[0].append(f64(keys[i]))
        held[1].append(f64(values[i]))
        part = slice(i * count, (i + 1) * count)
        want, size = model.attention(f64(q[part]), held[0].values(), held[1].values())
        bound = model.attention_bound(size, np.abs(held[1].values()).max(), want, dim, n, dtype == torch.bfloat16)
        assert (np.abs(f64(out[part]) - want) <= bound).all()


def sums(q, keys, values, window, exps, bf16, reference=None):
    """The 64-bit output of rows at the last positions, and per element how far a kernel that keeps its documented
    precision may be: by the terms that the element is a sum of, and not by the largest value of the sequence.

    Position k has the weight p_k (the row's largest is 1) and adds p_k v_k, off by its score's and weight's error as in
    model.attention_bound, relative to the position's own terms; the sum of weights likewise. Weights are rounded to a
    step: 2^-33 times the reference scale in bytes (2^-39 in halves), which is at most 2^8 above the smallest value
    scale of the sequence or 2^64 below the largest, times an integer of at most 127. bf16 rows: a weight in one half, 2^-12, and the output's
    rounding, 2^-8."""
    u = 2.0 ** -23
    rows_, heads, dim = q.shape
    length, kv_heads = keys.shape[:2]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for r in range(rows_):
        at = length - rows_ + r
        first = max(0, at - window + 1) if window else 0
        for h in range(heads):
            g = h * kv_heads // heads
            k, v = keys[first:at + 1, g], values[first:at + 1, g]
            s = (k @ q[r, h]) * dim ** -0.5
            off = (np.abs(k) @ np.abs(q[r, h])) * dim ** -0.5 * (dim / 8 + 10) * u + 4 * u + (len(s) / 16 + 128) * u
            p = np.exp(s - s.max())
            total = p.sum()
            out[r, h] = (p @ v) / total
            each = off[:, None] + (2.0 ** -12 if bf16 else 0.0)
            step = len(s) * 2.0 ** -33 * 127 * 2.0 ** (max(exps[:, g].min() + 8, exps[:, g].max() - 64) if reference is None else reference)
            bound[r, h] = ((p[:, None] * each * np.abs(v)).sum(0) + np.abs(out[r, h]) * (p @ off) + step) / total
            bound[r, h] *= 1 + off.max()
    return out, bound + (2.0 ** -8 if bf16 else u) * np.abs(out) + 1e-30


FORMS = [
    # kv_heads, group, dim, lengths, rows: byte products of one to four rows, halves of up to 8 and 16, 128 rows
    (2, 1, 64, [300, 60], 1), (2, 4, 128, [300, 60], 1), (1, 3, 32, [300, 60], 1), (1, 2, 64, [3000, 60], 2),
    (1, 2, 64, [300, 60], 4), (2, 1, 128, [300, 60], 7), (1, 3, 32, [300, 60], 9), (1, 2, 128, [300, 60], 9),
    (1, 2, 64, [300, 60], 20), (4, 1, 64, [600, 300] + [1000] * 8, 256), (4, 1, 128, [600, 300] + [1000] * 8, 256),
    (4, 1, 32, [600, 300] + [1000] * 10, 200),
]


def loud_position(kv_heads, group, dim, lengths, count, dtype, louder, drop, window, at):
    """One position's value is 2^louder times the others' and its weight 2^-drop of an ordinary one's; `at`: where, by
    sequence length. Its block's other positions are then held as 0 or nearly so. The first two sequences are checked."""
    rng = np.random.default_rng(dim + abs(louder) + drop)
    c = Cache(kv_heads, dim, lengths)
    keys = [rows(rng, n, kv_heads, dim, dtype) for n in lengths]
    values = [rows(rng, n, kv_heads, dim, dtype) for n in lengths]
    q = rows(rng, count * len(lengths), kv_heads * group, dim, dtype)
    q[..., 1] = 8.0
    for i, n in enumerate(lengths):
        keys[i][..., 1] = 0
        if i < 2:
            keys[i][at(n), :, 1] = -drop * np.log(2.0) / 8 * dim ** 0.5
            values[i][at(n)] *= 2.0 ** louder
    c.append(lengths, keys, values)
    out = torch.empty_like(q)
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(c.batch(lengths, [count] * len(lengths)),
                   rt.kv8_query(q.data_ptr(), out.data_ptr(), kind(dtype), heads=kv_heads * group, window=window), ws)
    torch.cuda.synchronize()
    for i, n in enumerate(lengths[:2]):
        held = [model.Held(kv_heads, dim) for _ in range(2)]
        held[0].append(f64(keys[i]))
        held[1].append(f64(values[i]))
        part = slice(i * count, (i + 1) * count)
        want, bound = sums(f64(q[part]), held[0].values(), held[1].values(), window, held[1].exps, dtype == torch.bfloat16)
        err = np.abs(f64(out[part]) - want)
        assert (err <= bound).all(), (i, (err / bound).max(), (err / np.maximum(np.abs(want), 1e-30)).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("louder,drop", [(6, 3), (20, 300), (40, 300), (20, 20), (40, 40), (40, 33), (75, 60), (-40, 5)])
@pytest.mark.parametrize("kv_heads,group,dim,lengths,count", FORMS)
def test_a_loud_position_among_quiet_ones(cuda_ok, kv_heads, group, dim, lengths, count, louder, drop, dtype):
    """Weights near 0, weights that make it as much as all the others, and a position far below them."""
    loud_position(kv_heads, group, dim, lengths, count, dtype, louder, drop, 0, lambda n: 21)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("louder", [20, 40, 75])
@pytest.mark.parametrize("kv_heads,group,dim,lengths,count", FORMS)
def test_a_loud_position_that_rows_do_not_see(cuda_ok, kv_heads, group, dim, lengths, count, louder, dtype):
    """Behind a window's first page: one row a sequence. Ahead of all rows but the last: more."""
    if count == 1:
        loud_position(kv_heads, group, dim, lengths, count, dtype, louder, 0, 20, lambda n: (n - 20) // 16 * 16)
    else:
        loud_position(kv_heads, group, dim, lengths, count, dtype, louder, 0, 0, lambda n: n - 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv_heads,group,dim,lengths,count", FORMS)
def test_value_scales_that_rise_and_fall(cuda_ok, kv_heads, group, dim, lengths, count, dtype):
    """Whole blocks louder and quieter, one after another and in long runs: the reference moves, up and down."""
    rng = np.random.default_rng(3 * dim + count)
    c = Cache(kv_heads, dim, lengths)
    keys = [rows(rng, n, kv_heads, dim, dtype) for n in lengths]
    values = []
    for i, n in enumerate(lengths):
        steps = rng.choice([0, 0, 3, 7, 9, 20, -9, -20, 70], n // 16 + 1) if i == 0 else np.linspace(-50, 50, n // 16 + 1).round()
        values.append(rows(rng, n, kv_heads, dim, dtype) * dev(2.0 ** np.repeat(steps, 16)[:n, None, None], torch.float32).to(dtype))
    c.append(lengths, keys, values)
    q = rows(rng, count * len(lengths), kv_heads * group, dim, dtype)
    out = torch.empty_like(q)
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(c.batch(lengths, [count] * len(lengths)),
                   rt.kv8_query(q.data_ptr(), out.data_ptr(), kind(dtype), heads=kv_heads * group), ws)
    torch.cuda.synchronize()
    for i, n in enumerate(lengths[:2]):
        held = [model.Held(kv_heads, dim) for _ in range(2)]
        held[0].append(f64(keys[i]))
        held[1].append(f64(values[i]))
        part = slice(i * count, (i + 1) * count)
        want, bound = sums(f64(q[part]), held[0].values(), held[1].values(), 0, held[1].exps, dtype == torch.bfloat16)
        assert (np.abs(f64(out[part]) - want) <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("count", [1, 9])
def test_references_that_move_within_a_warp(cuda_ok, count, dtype):
    """Sequences too long for one window of a warp's page ids, items enough that they are hardly split: the scales' range
    grows upwards in the first, downwards in the second.

    Splits and windows that hold loud blocks only have those for their reference, so that the step of a weight is 2^-33 of
    the loudest scale here: next to a position with weight 1 whose integer is 0 in some dim, one of weight 2^-24 keeps 9
    of its bits there (the whole output is 2^24 times what it adds)."""
    kv_heads, dim, lengths = 64, 32, [8000, 8000] + [100] * 8
    rng = np.random.default_rng(40 + count)
    c = Cache(kv_heads, dim, lengths)
    keys = [rows(rng, n, kv_heads, dim, dtype) for n in lengths]
    values = [rows(rng, n, kv_heads, dim, dtype) for n in lengths]
    at = np.arange(8000)
    for i, steps in enumerate((np.select([at < 3000, at < 4500], [0, 20], 40), np.select([at < 3000, at < 5000], [30, 27], 0))):
        values[i] = (values[i].float() * dev(2.0 ** steps[:, None, None].astype(np.float64), torch.float32)).to(dtype)
    c.append(lengths, keys, values)
    q = rows(rng, count * len(lengths), kv_heads, dim, dtype)
    out = torch.empty_like(q)
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(c.batch(lengths, [count] * len(lengths)),
                   rt.kv8_query(q.data_ptr(), out.data_ptr(), kind(dtype), heads=kv_heads), ws)
    torch.cuda.synchronize()
    some = [0, 31, 63]
    for i, n in enumerate(lengths[:2]):
        held = [model.Held(len(some), dim) for _ in range(2)]
        held[0].append(f64(keys[i])[:, some])
        held[1].append(f64(values[i])[:, some])
        part = slice(i * count, (i + 1) * count)
        want, bound = sums(f64(q[part])[:, some], held[0].values(), held[1].values(), 0, held[1].exps, dtype == torch.bfloat16,
                           held[1].exps.max())
        assert (np.abs(f64(out[part])[:, some] - want) <= bound).all(), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_loud_positions_in_splits_of_many_rows(cuda_ok, dim, dtype):
    """One chunk of 480 rows over 6000 positions: its splits see different scales and meet in the merge."""
    kv_heads, n, count = 4, 6000, 480
    rng = np.random.default_rng(dim)
    c = Cache(kv_heads, dim, [n])
    keys, values = rows(rng, n, kv_heads, dim, dtype), rows(rng, n, kv_heads, dim, dtype)
    values[::701] *= 2.0 ** 25
    values[3200:4000] *= 2.0 ** -18
    c.append([n], [keys], [values])
    q = rows(rng, count, kv_heads, dim, dtype)
    out = torch.empty_like(q)
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(c.batch([n], [count]), rt.kv8_query(q.data_ptr(), out.data_ptr(), kind(dtype), heads=kv_heads), ws)
    torch.cuda.synchronize()
    held = [model.Held(kv_heads, dim) for _ in range(2)]
    held[0].append(f64(keys))
    held[1].append(f64(values))
    last = 30
    want, bound = sums(f64(q[-last:]), held[0].values(), held[1].values(), 0, held[1].exps, dtype == torch.bfloat16)
    assert (np.abs(f64(out[-last:]) - want) <= bound).all()
