"""Causal attention over packed prompts against the formula in 64 bits."""
import math

import numpy as np
import pytest

from phonon_b200 import runtime as rt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {True: torch.bfloat16, False: torch.float32}


def formula(q, k, v, begin, window=0, scale=0.0, tol=None):
    """[rows][heads][dim] in 64 bits, on the device. With tol = (bits that a weight and the output keep are below 2^-8:
    True for bf16) also how far a result may be off, element by element."""
    heads, kvh, dim = q.shape[1], k.shape[1], q.shape[2]
    scale = scale or dim ** -0.5
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lim = torch.zeros_like(out)
    for b, e in zip(begin, begin[1:]):
        if e <= b:
            continue
        at = torch.arange(e - b, device=q.device)
        hidden = at[None] > at[:, None]
        if window:
            hidden |= at[None] <= at[:, None] - window
        for h in range(heads):
            c = h * kvh // heads
            x, y, z = q[b:e, h].double(), k[b:e, c].double(), v[b:e, c].double()
            score = (x @ y.t() * scale).masked_fill(hidden, -math.inf)
            p = torch.softmax(score, 1)
            p = torch.where(hidden, 0.0, p)
            # rows hidden from every row of the product may hold anything
            out[b:e, h] = p @ z
            if tol is not None:
                lim[b:e, h] = bound(x, y, z, p, out[b:e, h], hidden, scale, tol)
    return (out, lim) if tol is not None else out


def bound(x, y, z, p, out, hidden, scale, bf16):
    """u = 2^-23 a rounding or truncation to fp32. A score: at most dim + 12 of them relative to scale sum |q k| (products of
    three-slice operands leave 2 u of it); the exponent's own argument three of the score. A weight is off by what the scores
    of its row are, relatively (twice: the sum of weights too), by 4 u of its own and, bf16, by 2^-8. The sums over positions:
    at most one rounding for every 16 of them, and 64. The result is rounded once."""
    u = 2.0 ** -23
    terms = scale * (x.abs() @ y.abs().t()).masked_fill(hidden, 0.0).amax(1, keepdim=True)
    eps = 2 * ((x.shape[1] + 15) * u * terms + 4 * u) + (64 + p.shape[1] / 16) * u + (2.0 ** -8 if bf16 else 0.0)
    lim = (torch.expm1(eps) * (p @ z.abs())) * 1.01
    return lim + (2.0 ** -8 if bf16 else 2.0 ** -24) * (out.abs() + lim) + 1e-37


def rows_of(rng, rows, heads, kvh, dim, bf16, loud=1.0):
    """Queries, keys and values side by side, as a projection leaves them."""
    x = rng.standard_normal((max(rows, 1), heads + 2 * kvh, dim)).astype(np.float32)
    x[:, :heads + kvh] *= loud
    x[:, heads + kvh:] *= np.exp(rng.standard_normal((max(rows, 1), kvh, 1)))
    packed = torch.tensor(x).to(DTYPES[bf16]).cuda()
    return packed, packed[:, :heads], packed[:, heads:heads + kvh], packed[:, heads + kvh:]


def call(q, k, v, out, begin, rows=None, max_rows=None, bf16=False, **kw):
    lengths = np.diff(begin)
    device_begin = torch.tensor(begin, dtype=torch.int32, device=q.device)
    c = rt.PromptAttention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), device_begin.data_ptr(), len(begin) - 1,
                           q.shape[0] if rows is None else rows, max(1, int(lengths.max())) if max_rows is None else max_rows,
                           q.shape[1], k.shape[1], q.shape[2], rt.ROWS_BF16 if bf16 else rt.ROWS_F32, q_stride=q.stride(0),
                           k_stride=k.stride(0), v_stride=v.stride(0), out_stride=out.stride(0), **kw)
    c.keep = device_begin
    return c


def begins(lengths):
    return [int(x) for x in np.concatenate([[0], np.cumsum(lengths)])]


CASES = [  # lengths, heads, K/V heads, dim, window
    ([1], 1, 1, 32, 0), ([1, 0, 2, 1], 8, 8, 64, 0), ([128], 8, 8, 64, 0), ([127, 129], 2, 1, 128, 0),
    ([256, 255, 257, 3], 4, 4, 64, 0), ([700], 3, 3, 32, 0), ([1000, 31, 64, 65], 8, 2, 128, 0), ([513, 0, 0, 90], 7, 1, 64, 0),
    ([300, 5], 6, 2, 32, 0), ([77, 400], 24, 3, 128, 0), ([1537], 2, 2, 128, 0), ([600, 100], 16, 1, 64, 0),
    ([45, 260], 130, 1, 64, 0), ([90], 34, 2, 32, 0), ([900, 17], 8, 8, 64, 250), ([400, 300], 4, 2, 128, 1),
    ([1200], 3, 1, 64, 64), ([650, 129], 5, 5, 32, 127), ([2100], 1, 1, 64, 1000), ([500, 500], 4, 4, 128, 130),
]


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("lengths,heads,kvh,dim,window", CASES)
def test_against_the_formula(cuda_ok, lengths, heads, kvh, dim, window, bf16):
    rng = np.random.default_rng(sum(lengths) + heads)
    begin = begins(lengths)
    rows = begin[-1]
    packed, q, k, v = rows_of(rng, rows + 3, heads, kvh, dim, bf16)
    out = torch.full((rows + 3, heads, dim), 7.0, dtype=DTYPES[bf16], device="cuda")
    status = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
    call(q, k, v, out, begin, bf16=bf16, window=window)(status.data_ptr())
    torch.cuda.synchronize()
    assert not status.any() and (out[rows:] == 7).all()
    want, lim = formula(q, k, v, begin, window, tol=bf16)
    err = (out.double() - want).abs()[:rows]
    assert (err <= lim[:rows]).all(), (err / lim[:rows].clamp(min=1e-300)).max()
    # the typical error is far below the bound: bf16 about its rounding, fp32 a few times the plain form's in fp32
    typical = (err.norm() / want[:rows].norm().clamp(min=1e-30)).item()
    assert typical < (4e-3 if bf16 else 2e-6), typical


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_flat_and_peaked_rows(cuda_ok, scale, bf16):
    """Scores of +-hundreds (single keys take all) and of nearly nothing; a scale of the caller's."""
    rng = np.random.default_rng(3)
    begin = begins([800, 40])
    packed, q, k, v = rows_of(rng, 840, 4, 2, 64, bf16, loud=5.0 if scale == 1.0 else 1.0)
    out = torch.empty(840, 4, 64, dtype=DTYPES[bf16], device="cuda")
    call(q, k, v, out, begin, bf16=bf16, scale=scale)()
    torch.cuda.synchronize()
    want, lim = formula(q, k, v, begin, 0, float(np.float32(scale)), tol=bf16)
    assert ((out.double() - want).abs() <= lim).all()


@pytest.mark.parametrize("bf16", [True, False])
def test_scores_that_rise_and_fall_along_a_row(cuda_ok, bf16):
    """Maxima that move at every turn, and a first position far above the rest."""
    rng = np.random.default_rng(4)
    n, dim = 1500, 64
    packed, q, k, v = rows_of(rng, n, 2, 2, dim, bf16)
    ramp = torch.linspace(-40, 40, n, device="cuda").to(packed.dtype)
    q[..., 0] = 8.0
    k[:, 0, 0], k[:, 1, 0] = ramp, ramp.flip(0)
    out = torch.empty(n, 2, dim, dtype=packed.dtype, device="cuda")
    call(q, k, v, out, [0, n], bf16=bf16)()
    torch.cuda.synchronize()
    want, lim = formula(q, k, v, [0, n], tol=bf16)
    assert ((out.double() - want).abs() <= lim).all()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_what_a_row_does_not_see_does_not_matter(cuda_ok, dim, bf16):
    """Infinities and NaN behind the row, before its window, in other prompts and behind the last: the rows that do not see
    them are bit for bit what they are without; those that do are not finite, and only their prompts are named."""
    rng = np.random.default_rng(dim)
    begin, window = begins([300, 200, 150]), 100
    rows = 680
    packed, q, k, v = rows_of(rng, rows, 4, 2, dim, bf16)
    outs = []
    status = torch.zeros(3, dtype=torch.int32, device="cuda")
    for dirty in (False, True):
        if dirty:
            packed[650:] = float("nan")
            v[40, 0, 3], v[250, 1, 0], k[120, 1, 5] = float("inf"), float("nan"), float("-inf")
            k[290, 0, 0] = float("nan")
            q[30, 2, 1] = float("inf")
        out = torch.full((rows, 4, dim), 7.0, dtype=packed.dtype, device="cuda")
        status.zero_()
        call(q, k, v, out, begin, bf16=bf16, window=window)(status.data_ptr())
        torch.cuda.synchronize()
        assert (out[650:] == 7).all()
        outs.append(out)
    clean, dirty = outs
    assert clean[:650].isfinite().all() and status.tolist() == [rt.NON_FINITE, 0, 0]
    sees = torch.zeros(650, 4, dtype=torch.bool, device="cuda")
    for at, heads in ((40, (0, 1)), (250, (2, 3)), (290, (0, 1))):
        for h in heads:
            sees[at:min(at + window, 300), h] = True
    sees[30, 2] = True
    # (a score of -inf has weight 0, one of +inf has none that is a number)
    sign = torch.zeros(650, 4, dtype=torch.bool, device="cuda")
    sign[120:220, 2:] = q[120:220, 2:, 5] < 0
    maybe = torch.zeros(650, 4, dtype=torch.bool, device="cuda")
    maybe[120:220, 2:] = True
    same = (clean[:650] == dirty[:650]).all(-1)
    assert (same | sees | maybe).all()
    broken = ~dirty[:650].isfinite().all(-1)
    assert (broken[sees]).all() and (broken[sign & maybe]).all() and not broken[~(sees | maybe)].any()
    assert not broken[120:220, 2:][(q[120:220, 2:, 5] > 0)].any()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("length", [1, 40, 70, 200])
def test_values_that_are_not_finite_in_short_prompts(cuda_ok, length, dim, bf16):
    """The turns that a prompt ends in: every row from the value on sees it, whatever its place."""
    rng = np.random.default_rng(length)
    for bad in sorted({0, length // 2, length - 1}):
        packed, q, k, v = rows_of(rng, length, 2, 2, dim, bf16)
        v[bad, 0, dim - 1] = float("inf")
        k[bad, 1, 0] = float("nan")
        out = torch.empty(length, 2, dim, dtype=packed.dtype, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        call(q, k, v, out, [0, length], bf16=bf16)(status.data_ptr())
        torch.cuda.synchronize()
        assert status.tolist() == [rt.NON_FINITE]
        broken = ~out.isfinite().all(-1)
        assert not broken[:bad].any() and broken[bad:].all()


@pytest.mark.parametrize("bf16", [True, False])
def test_rows_of_bad_prompts_stay(cuda_ok, bf16):
    rng = np.random.default_rng(8)
    packed, q, k, v = rows_of(rng, 400, 2, 2, 64, bf16)
    # (of the first: 500 lies outside, and 400 before it)
    for begin, bad, kw in (([0, 100, 500, 400, 400], [1, 2, 3], {}), ([-5, 100, 200], [0], {}), ([0, 100, 50, 300], [1, 2], {}),
                           ([0, 150, 230], [0], dict(max_rows=149)), ([0, 200, 1 << 30], [1], {}),
                           ([300, 400, 0, 100], [1, 2], {}), ([390, 380], [0], {})):
        out = torch.full((400, 2, 64), 7.0, dtype=packed.dtype, device="cuda")
        status = torch.zeros(len(begin) - 1, dtype=torch.int32, device="cuda")
        call(q, k, v, out, begin, bf16=bf16, **({"max_rows": 400} | kw))(status.data_ptr())
        torch.cuda.synchronize()
        assert [i for i, s in enumerate(status.tolist()) if s] == bad and set(status.tolist()) <= {0, rt.INVALID}
        kept = torch.ones(400, dtype=torch.bool, device="cuda")
        for i, (b, e) in enumerate(zip(begin, begin[1:])):
            if i not in bad and e > b:
                kept[b:e] = False
                want, lim = formula(q[b:e], k[b:e], v[b:e], [0, e - b], tol=bf16)
                assert ((out[b:e].double() - want).abs() <= lim).all()
        assert (out[kept] == 7).all()


def test_thousands_of_short_prompts(cuda_ok):
    rng = np.random.default_rng(9)
    lengths = rng.integers(0, 4, 5000)
    begin = begins(lengths)
    packed, q, k, v = rows_of(rng, begin[-1], 2, 1, 32, True)
    out = torch.full((begin[-1], 2, 32), 7.0, dtype=torch.bfloat16, device="cuda")
    call(q, k, v, out, begin, bf16=True)()
    torch.cuda.synchronize()
    want, lim = formula(q.cpu(), k.cpu(), v.cpu(), begin, tol=True)
    assert ((out.double().cpu() - want).abs() <= lim).all()


@pytest.mark.parametrize("bf16", [True, False])
def test_in_place_on_two_streams_and_replayed(cuda_ok, bf16):
    """out in place of q inside the packed rows; two calls at once; a captured call over other rows and lengths."""
    rng = np.random.default_rng(10)
    sets, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for n in range(2):
        begin = begins([200 + 60 * n, 33])
        packed, q, k, v = rows_of(rng, begin[-1], 4, 4, 64, bf16)
        sets.append((begin, packed, q, k, v, packed.clone(), call(q, k, v, q, begin, bf16=bf16)))
    torch.cuda.synchronize()
    for stream, s in zip(streams, sets):
        s[-1](stream_ptr=stream.cuda_stream)
    torch.cuda.synchronize()
    for begin, packed, q, k, v, before, _ in sets:
        want, lim = formula(before[:, :4], k, v, begin, tol=bf16)
        assert ((q.double() - want).abs() <= lim).all() and (packed[:, 4:] == before[:, 4:]).all()
    begin, packed, q, k, v, before, _ = sets[0]
    out = torch.empty(begin[-1], 4, 64, dtype=packed.dtype, device="cuda")
    c = call(q, k, v, out, begin, max_rows=begin[-1], bf16=bf16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c(stream_ptr=torch.cuda.current_stream().cuda_stream)
    for new in ([0, 100, 233], [0, 0, 233], begin):
        packed.copy_(before.flip(0))
        c.keep.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want, lim = formula(q, k, v, new, tol=bf16)
        assert ((out.double() - want).abs() <= lim).all()


def test_rows_beyond_32_bits_of_elements(cuda_ok):
    """Prompts at both ends of an array of more than 2^31 elements."""
    rng = np.random.default_rng(11)
    rows, wide = 40000, 1 << 16
    big = torch.zeros(rows, wide, dtype=torch.bfloat16, device="cuda")
    _, q, k, v = rows_of(rng, 200, 2, 1, 64, True)
    at = rows - 200
    views = []
    for x, col in ((q, 0), (k, 1024), (v, 60000)):
        big[at:, col:col + x.shape[1] * 64] = x.reshape(200, -1)
        views.append(big[:, col:col + x.shape[1] * 64].unflatten(1, (-1, 64)))
    out = torch.empty(rows, 2, 64, dtype=torch.bfloat16, device="cuda")
    call(*views, out, [0, 70, at, rows], bf16=True, max_rows=rows)()
    torch.cuda.synchronize()
    want, lim = formula(q, k, v, [0, 200], tol=True)
    assert ((out[at:].double() - want).abs() <= lim).all() and (out[:70] == 0).all()


def test_refusals(cuda_ok):
    a = torch.zeros(8192, device="cuda")
    p = a.data_ptr()
    begin = torch.tensor([0, 4], dtype=torch.int32, device="cuda")

    def status(q=p, k=p + 4096, v=p + 8192, out=p + 12288, begin=begin.data_ptr(), prompts=1, rows=4, max_rows=4, heads=2, kv_heads=1,
               head_dim=32, **kw):
        try:
            rt.PromptAttention(q, k, v, out, begin, prompts, rows, max_rows, heads, kv_heads, head_dim, **kw)()
        except rt.CudaError as e:
            return e.status
        return rt.OK

    assert status() == rt.OK and status(rows=0) == rt.OK and status(out=p) == rt.OK
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(begin=None), dict(prompts=0), dict(max_rows=0),
               dict(heads=0), dict(kv_heads=0), dict(heads=3, kv_heads=2), dict(head_dim=48), dict(head_dim=256), dict(type=2),
               dict(scale=-1.0), dict(scale=float("nan")), dict(scale=2e30), dict(q=p + 8), dict(out=p + 12290),
               dict(q_stride=63), dict(q_stride=68), dict(k_stride=24), dict(v_stride=8), dict(out_stride=66),
               dict(out=p, out_stride=128), dict(out=p + 4096), dict(out=p + 8192), dict(window=(1 << 30) + 1),
               dict(rows=(1 << 30) + 1), dict(heads=1 << 17)):
        assert status(**kw) == rt.INVALID, kw
    assert status(prompts=1 << 24, rows=1 << 30, max_rows=1 << 30, heads=256, kv_heads=256) == rt.CAPACITY
    torch.cuda.synchronize()
