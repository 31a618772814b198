"""Attention over packed prompts where a CTA of the bf16 kernel has two row tiles: calls of enough positions. The tests of the
formula, of values that are not finite, of calls in place and at the same time, at such sizes."""
import numpy as np
import pytest

from launches import launches
from phonon_b200 import runtime as rt
from test_gpu_prompt import begins, call, formula, rows_of

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

LONG = [700] * 8 + [1001, 130]
CASES = [(LONG, 32, 8, 128, 0), (LONG, 32, 8, 128, 130), (LONG, 32, 8, 128, 1000), (LONG, 16, 16, 128, 1),
         ([3000] * 8, 8, 8, 64, 0), ([3000] * 8, 8, 8, 64, 250), ([1201, 31, 2000, 64, 1500, 900, 1700] * 2, 24, 8, 64, 0),
         ([1201, 31, 2000, 64, 1500, 900, 1700] * 2, 24, 8, 64, 90),
         ([900] * 20, 8, 8, 32, 0), ([900] * 20, 8, 8, 32, 100), ([555, 1, 0, 777, 1024] * 4, 20, 4, 32, 300)]


def has_two_tiles(c, begin, heads, kvh):
    """Whether the call has as many CTAs as blocks of two row tiles, and fewer than of one."""
    group = heads // kvh
    pack = group if group <= 32 else 1
    half, n, most = 128 // pack, len(begin) - 1, max(np.diff(begin))

    def ctas(tokens):
        return heads // pack * min(begin[-1] // tokens + n, n * -(-most // tokens))
    (name, grid), = launches(lambda stream: c(stream_ptr=stream))
    return "prompt_bf16_kernel" in name and grid == ctas(2 * half) < ctas(half)


def setup(seed, lengths, heads, kvh, dim):
    begin = begins(lengths)
    return (begin,) + rows_of(np.random.default_rng(seed), begin[-1], heads, kvh, dim, True)


@pytest.mark.parametrize("lengths,heads,kvh,dim,window", CASES)
def test_against_the_formula(cuda_ok, lengths, heads, kvh, dim, window):
    begin, packed, q, k, v = setup(dim + window, lengths, heads, kvh, dim)
    out = torch.full((begin[-1], heads, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    status = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
    c = call(q, k, v, out, begin, bf16=True, window=window)
    assert has_two_tiles(c, begin, heads, kvh)
    c(status.data_ptr())
    torch.cuda.synchronize()
    assert not status.any()
    want, lim = formula(q, k, v, begin, window, tol=True)
    err = (out.double() - want).abs()
    assert (err <= lim).all(), (err / lim.clamp(min=1e-300)).max()
    assert (err.norm() / want.norm()).item() < 4e-3


@pytest.mark.parametrize("lengths,heads,kvh,dim,window", CASES)
def test_what_a_row_does_not_see_does_not_matter(cuda_ok, lengths, heads, kvh, dim, window):
    """Values that are not finite in a prompt's first and second tiles, and after the last prompt: rows that do not see them are
    bit for bit what they are without, rows that do are not finite, and their prompts are named."""
    begin, packed, q, k, v = setup(dim + window + 1, lengths + [40], heads, kvh, dim)  # (the last 40 rows are no prompt's)
    begin = begin[:-1]
    out, again = (torch.full((begin[-1] + 40, heads, dim), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    status = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
    assert has_two_tiles(call(q, k, v, out, begin, rows=begin[-1], bf16=True, window=window), begin, heads, kvh)
    packed[begin[-1]:] = float("nan")
    marks = [(begin[i] + at, h) for i, at, h in ((0, 5, 0), (0, 300, kvh - 1), (2, 0, 0), (3, min(lengths[3] - 1, 650), 1)) if at < lengths[i]]
    sees = torch.zeros(begin[-1], heads, dtype=torch.bool, device="cuda")
    for row, h in marks:
        v[row, h, row % dim] = (float("inf"), float("nan"))[row % 2]
        end = next(e for e in begin if e > row)
        group = heads // kvh
        sees[row:min(row + window, end) if window else end, h * group:(h + 1) * group] = True
    call(q, k, v, again, begin, rows=begin[-1], bf16=True, window=window)(status.data_ptr())
    torch.cuda.synchronize()
    hit = {next(i for i in range(len(lengths)) if begin[i] <= row < begin[i + 1]) for row, _ in marks}
    assert status.tolist() == [rt.NON_FINITE if i in hit else 0 for i in range(len(lengths))]
    assert (again[begin[-1]:] == 7).all()
    same = (out == again).all(-1)[:begin[-1]]
    assert (same | sees).all() and not again[:begin[-1]].isfinite().all(-1)[sees].any()


@pytest.mark.parametrize("lengths,heads,kvh,dim,window", [CASES[0], CASES[5], CASES[10]])
def test_in_place_and_at_the_same_time(cuda_ok, lengths, heads, kvh, dim, window):
    """out in place of q on two streams at once, and one of the calls captured and replayed over other rows."""
    sets, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for n in range(2):
        begin, packed, q, k, v = setup(n, lengths, heads, kvh, dim)
        assert has_two_tiles(call(q, k, v, torch.empty_like(q), begin, bf16=True, window=window), begin, heads, kvh)
        sets.append((begin, packed, q, k, v, packed.clone(), call(q, k, v, q, begin, bf16=True, window=window)))
    torch.cuda.synchronize()
    for stream, s in zip(streams, sets):
        s[-1](stream_ptr=stream.cuda_stream)
    torch.cuda.synchronize()
    for begin, packed, q, k, v, before, _ in sets:
        want, lim = formula(before[:, :heads], k, v, begin, window, tol=True)
        assert ((q.double() - want).abs() <= lim).all() and (packed[:, heads:] == before[:, heads:]).all()
    begin, packed, q, k, v, before, c = sets[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c(stream_ptr=torch.cuda.current_stream().cuda_stream)
    packed.copy_(before.flip(0))
    before = packed.clone()
    graph.replay()
    torch.cuda.synchronize()
    want, lim = formula(before[:, :heads], k, v, begin, window, tol=True)
    assert ((q.double() - want).abs() <= lim).all()
