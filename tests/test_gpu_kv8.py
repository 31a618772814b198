"""The 8-bit paged K/V cache on the GPU: rows written and read back equal the
64-bit definition bit for bit; attention stays within the arithmetic's bound
of it. Every shape here is a place where one of them can go wrong: empty and
one-position sequences, ends inside a page, several rows at once, grouped
heads, windows, strides, bad tables, streams and captured calls."""
import numpy as np
import pytest

import kv8_model as model
from phonon_b200 import runtime as rt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def dev(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype, device="cuda")


def i32(a):
    return dev(a, torch.int32)


class Cache:
    """A cache with a page table of its own, shuffled, and spare pages."""

    def __init__(self, kv_heads, dim, lengths, seed=0, layers=1, spare=3):
        self.kv_heads, self.dim = kv_heads, dim
        pages = [-(-n // 16) for n in lengths]
        self.stride = max(1, max(pages))
        self.pool = sum(pages) + spare
        order = np.random.RandomState(seed).permutation(self.pool)
        table = np.full((len(lengths), self.stride), -1)
        at = 0
        for i, n in enumerate(pages):
            table[i, :n] = order[at:at + n]
            at += n
        self.table = i32(table)
        self.kv = rt.Kv8Cache(kv_heads, dim, self.pool, layers=layers)
        self.keep = []

    def batch(self, lengths, counts, max_rows=None, max_length=None):
        begin, length = i32(np.concatenate([[0], np.cumsum(counts)])), i32(lengths)
        self.keep += [begin, length]
        return rt.kv8_batch(len(lengths), length.data_ptr(), self.table.data_ptr(), self.stride,
                            max_length=self.stride * 16 if max_length is None else max_length,
                            rows=int(sum(counts)), row_begin_ptr=begin.data_ptr(),
                            max_rows=max(1, max(counts)) if max_rows is None else max_rows)

    def append(self, lengths, keys, values, layer=0, status=None, stream=0):
        """keys, values: a list of [rows][kv_heads][dim] per sequence"""
        counts = [len(k) for k in keys]
        k, v = torch.cat(keys).contiguous(), torch.cat(values).contiguous()
        self.keep += [k, v]
        kind = rt.ROWS_BF16 if k.dtype == torch.bfloat16 else rt.ROWS_F32
        self.kv.append(self.batch(lengths, counts), rt.kv8_rows(k.data_ptr(), v.data_ptr(), kind), layer=layer,
                       status_ptr=status, stream_ptr=stream)

    def read(self, lengths, counts=None, dtype=torch.float32, layer=0, status=None):
        counts = lengths if counts is None else counts
        out = [torch.full((sum(counts), self.kv_heads, self.dim), float("nan"), dtype=dtype, device="cuda")
               for _ in range(2)]
        kind = rt.ROWS_BF16 if dtype == torch.bfloat16 else rt.ROWS_F32
        self.kv.read(self.batch(lengths, counts), rt.kv8_rows(out[0].data_ptr(), out[1].data_ptr(), kind), layer=layer,
                     status_ptr=status)
        torch.cuda.synchronize()
        return [np.split(o.float().cpu().numpy(), np.cumsum(counts)[:-1]) for o in out]


def rows(rng, n, heads, dim, dtype=torch.float32):
    """Rows with a loudness of their own per position and head, so that scales rise inside blocks."""
    x = rng.standard_normal((n, heads, dim)) * np.exp(rng.standard_normal((n, heads, 1)))
    return dev(x, torch.float32).to(dtype)


def f64(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------- write, read back
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv_heads,dim", [(8, 64), (1, 32), (3, 128)])
def test_written_in_pieces_reads_back_exactly(cuda_ok, kv_heads, dim, dtype):
    rng = np.random.default_rng(kv_heads * dim)
    pieces = [[0, 1, 1, 1, 13, 1, 1], [16, 16, 0, 1, 0, 0, 31], [5, 40, 3, 1, 1, 1, 1], [1, 0, 0, 0, 0, 0, 0],
              [0, 0, 0, 0, 0, 0, 0]]
    final = [sum(p) for p in pieces]
    c = Cache(kv_heads, dim, final)
    held = [[model.Held(kv_heads, dim) for _ in pieces] for _ in range(2)]
    lengths = [0] * len(pieces)
    for step in range(len(pieces[0])):
        counts = [p[step] for p in pieces]
        new = [[rows(rng, n, kv_heads, dim, dtype) for n in counts] for _ in range(2)]
        for w in range(2):
            for h, r in zip(held[w], new[w]):
                h.append(f64(r))
        lengths = [a + b for a, b in zip(lengths, counts)]
        c.append(lengths, *new)
        for got, want in zip(c.read(lengths), held):
            for g, h in zip(got, want):
                np.testing.assert_array_equal(g, h.values().astype(np.float32))
    # the last positions only, from inside a block, in bf16 (integers of 8 bits: exact)
    counts = [min(n, 7) for n in lengths]
    for got, want in zip(c.read(lengths, counts, torch.bfloat16), held):
        for g, h, n in zip(got, want, counts):
            np.testing.assert_array_equal(g, h.values()[len(h.codes) - n:].astype(np.float32))


def test_extreme_and_non_finite_values(cuda_ok):
    c = Cache(2, 64, [16, 16, 16, 5])
    x = np.zeros((16, 2, 64), np.float32)
    x[3, 0] = 3e38          # above 127 * 2^64: held as the largest
    x[4, 1] = 1e-40         # below the smallest scale's half step: 0
    tie = np.zeros((16, 2, 64), np.float32)
    tie[0] = 127.0
    tie[1, :, :8] = [0.5, 1.5, 2.5, -0.5, -1.5, 126.5, 127.0, -127.0]
    edge = np.zeros((16, 2, 64), np.float32)
    edge[0, 0, 0], edge[0, 1, 0] = 127.0, np.nextafter(np.float32(127.0), np.float32(200.0))
    bad = np.ones((5, 2, 64), np.float32)
    bad[1, 0, 3], bad[2, 1, 5] = np.nan, -np.inf
    all_rows = [x, tie, edge, bad]
    lengths = [16, 16, 16, 5]
    status = torch.zeros(4, dtype=torch.int32, device="cuda")
    c.append(lengths, [dev(r) for r in all_rows], [dev(-r) for r in all_rows], status=status.data_ptr())
    got = c.read(lengths)
    for sign, side in zip((1, -1), got):
        for g, r in zip(side, all_rows):
            h = model.Held(2, 64)
            h.append(sign * r.astype(np.float64))
            np.testing.assert_array_equal(g, h.values().astype(np.float32))
    assert status.tolist() == [0, 0, 0, rt.NON_FINITE]
    # a bad element costs nothing but itself
    assert got[0][3][1, 0, 3] == 0 and got[0][3][2, 1, 5] == 0 and (np.abs(got[0][3]) == 1).sum() == 5 * 128 - 2


def test_strided_rows_layers_and_untouched_memory(cuda_ok):
    rng = np.random.default_rng(3)
    c = Cache(4, 32, [20, 33], layers=3)
    packed = dev(rng.standard_normal((53, 3, 4, 32)), torch.float32)  # [q | k | v] rows of a projection
    c.keep.append(packed)
    batch = c.batch([20, 33], [20, 33])
    c.kv.append(batch, rt.kv8_rows(packed[:, 1].data_ptr(), packed[:, 2].data_ptr(), stride=3 * 128), layer=1)
    want = [[model.Held(4, 32) for _ in range(2)] for _ in range(2)]
    for w in range(2):
        for i, part in enumerate((packed[:20, 1 + w], packed[20:, 1 + w])):
            want[w][i].append(f64(part))
    out = torch.full((60, 3, 4, 32), 7.0, device="cuda")
    c.kv.read(batch, rt.kv8_rows(out[:, 1].data_ptr(), out[:, 2].data_ptr(), stride=3 * 128), layer=1)
    torch.cuda.synchronize()
    assert (out[:, 0] == 7).all() and (out[53:] == 7).all()
    for w in range(2):
        ref = np.concatenate([h.values() for h in want[w]]).astype(np.float32)
        np.testing.assert_array_equal(out[:53, 1 + w].cpu().numpy(), ref)
    for layer in (0, 2):  # the other layers still hold nothing
        assert all((g == 0).all() for side in c.read([20, 33], layer=layer) for g in side)


# ------------------------------------------------------------------ attention
CASES = [
    # kv_heads, group, dim, lengths, rows, window
    (8, 1, 64, [1, 2, 15, 16, 17, 0, 64, 250, 1000], 1, 0),
    (8, 1, 64, [4000], 1, 0),
    (2, 4, 64, [77, 1, 0, 513], 1, 0),
    (1, 8, 128, [300, 16], 1, 0),
    (2, 7, 128, [95, 33], 1, 40),
    (3, 1, 32, [1, 16, 31, 200], 1, 17),
    (2, 3, 32, [70, 9], 5, 0),
    (8, 1, 64, [40, 256, 300], 16, 250),
    (2, 5, 64, [33, 100], 9, 0),
    (2, 2, 128, [50, 130, 3], 20, 0),
    (1, 1, 64, [700], 300, 0),
    (1, 12, 64, [64, 65], 3, 1),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv_heads,group,dim,lengths,count,window", CASES)
def test_attention_against_the_definition(cuda_ok, kv_heads, group, dim, lengths, count, window, dtype):
    rng = np.random.default_rng(dim + count + len(lengths))
    c = Cache(kv_heads, dim, lengths)
    new = [[rows(rng, n, kv_heads, dim, dtype) for n in lengths] for _ in range(2)]
    c.append(lengths, *new)
    held = [[model.Held(kv_heads, dim) for _ in lengths] for _ in range(2)]
    for w in range(2):
        for h, r in zip(held[w], new[w]):
            if len(r):
                h.append(f64(r))
    heads = kv_heads * group
    counts = [count] * len(lengths)  # more rows than positions in the short ones: those see nothing
    q = rows(rng, sum(counts) + 2, heads, dim, dtype)
    out = torch.full_like(q, 9.0)
    kind = rt.ROWS_BF16 if dtype == torch.bfloat16 else rt.ROWS_F32
    status = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
    ws = rt.Kv8Workspace(c.kv)
    for _ in range(2):  # the second call finds the scratch as the first left it
        c.kv.attention(c.batch(lengths, counts),
                       rt.kv8_query(q.data_ptr(), out.data_ptr(), kind, heads=heads, window=window), ws,
                       status_ptr=status.data_ptr())
    torch.cuda.synchronize()
    assert (out[sum(counts):] == 9).all() and not status.any()
    got = f64(out)
    for i, n in enumerate(lengths):
        k, v = held[0][i].values(), held[1][i].values()
        part = got[i * count:(i + 1) * count]
        want, size = model.attention(f64(q[i * count:(i + 1) * count]), k, v, window)
        biggest = np.abs(v).max() if n else 0.0
        bound = model.attention_bound(size, biggest, want, dim, n, dtype == torch.bfloat16)
        assert (np.abs(part - want) <= bound).all(), (i, n, (np.abs(part - want) / bound).max())
        assert (part[:max(0, count - n)] == 0).all()


def test_attention_in_place_strided_scaled_and_one_row_form(cuda_ok):
    rng = np.random.default_rng(8)
    lengths = [37, 5, 120]
    c = Cache(2, 64, lengths)
    new = [[rows(rng, n, 2, 64) for n in lengths] for _ in range(2)]
    c.append(lengths, *new)
    held = [[model.Held(2, 64) for _ in lengths] for _ in range(2)]
    for w in range(2):
        for h, r in zip(held[w], new[w]):
            h.append(f64(r))
    packed = rows(rng, 3, 8, 64)  # the first 4 heads are the queries and receive the output
    before = packed.clone()
    length = i32(lengths)
    batch = rt.kv8_batch(3, length.data_ptr(), c.table.data_ptr(), c.stride, max_length=120)
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(batch, rt.kv8_query(packed.data_ptr(), packed.data_ptr(), heads=4, scale=0.25, q_stride=512,
                                       out_stride=512), ws)
    torch.cuda.synchronize()
    assert torch.equal(packed[:, 4:], before[:, 4:])
    for i, n in enumerate(lengths):
        want, size = model.attention(f64(before[i:i + 1, :4]), held[0][i].values(), held[1][i].values(), scale=0.25)
        bound = model.attention_bound(size, np.abs(held[1][i].values()).max(), want, 64, n, False)
        assert (np.abs(f64(packed[i:i + 1, :4]) - want) <= bound).all()


def test_values_of_very_different_blocks(cuda_ok):
    """Blocks whose value scales differ by 2^60, the loud one with a small weight, and scores over the whole range
    of the exponential: the weights are scaled by the blocks' scales inside the kernel."""
    rng = np.random.default_rng(9)
    n = 64
    k = rng.standard_normal((n, 1, 64))
    k[16:32] *= 30.0
    v = rng.standard_normal((n, 1, 64)) * np.repeat([1.0, 2.0 ** -30, 2.0 ** 30, 1e-3], 16)[:, None, None]
    c = Cache(1, 64, [n])
    c.append([n], [dev(k, torch.float32)], [dev(v, torch.float32)])
    hk, hv = model.Held(1, 64), model.Held(1, 64)
    hk.append(f64(dev(k, torch.float32)))
    hv.append(f64(dev(v, torch.float32)))
    q = rows(rng, n, 1, 64)
    out = torch.empty_like(q)
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(c.batch([n], [n]), rt.kv8_query(q.data_ptr(), out.data_ptr(), heads=1), ws)
    torch.cuda.synchronize()
    want, size = model.attention(f64(q), hk.values(), hv.values())
    # a row's error is bounded by the largest value among the keys it sees
    biggest = np.maximum.accumulate(np.abs(hv.values()).max((1, 2)))[:, None, None]
    bound = model.attention_bound(size, 1.0, 0 * want, 64, n, False) * biggest + 2.0 ** -23 * np.abs(want)
    assert (np.abs(f64(out) - want) <= bound).all()


# ------------------------------------------------- what the kernels must refuse
def test_bad_lengths_rows_and_pages_are_flagged(cuda_ok):
    rng = np.random.default_rng(11)
    lengths = [40, 40, 40, 40]
    c = Cache(2, 64, lengths)
    new = [[rows(rng, n, 2, 64) for n in lengths] for _ in range(2)]
    c.append(lengths, *new)
    good = c.read(lengths)
    q = rows(rng, 4, 4, 64)
    ws = rt.Kv8Workspace(c.kv)

    def attend(lengths, max_length=48, q=q):
        out = torch.full_like(q, 9.0)
        status = torch.zeros(4, dtype=torch.int32, device="cuda")
        c.kv.attention(c.batch(lengths, [1, 1, 1, 1], max_length=max_length),
                       rt.kv8_query(q.data_ptr(), out.data_ptr(), heads=4), ws, status_ptr=status.data_ptr())
        torch.cuda.synchronize()
        return out, status.tolist()

    base, status = attend(lengths)
    assert status == [0, 0, 0, 0]
    out, status = attend([40, -1, 49, 2 ** 31 - 1])
    assert status == [0, rt.CAPACITY, rt.CAPACITY, rt.CAPACITY]
    assert torch.equal(out[0], base[0]) and (out[1:] == 0).all()
    # a page outside the pool is not seen, written or read
    table = c.table.clone()
    c.table[1, 1], c.table[2, 0] = c.pool, -5
    out, status = attend(lengths)
    assert status == [0, rt.INVALID, rt.INVALID, 0]
    assert torch.equal(out[0], base[0]) and torch.equal(out[3], base[3]) and torch.isfinite(out).all()
    status = torch.zeros(4, dtype=torch.int32, device="cuda")
    got = c.read(lengths, status=status.data_ptr())
    assert status.tolist() == [0, rt.INVALID, rt.INVALID, 0]
    assert (got[0][1][16:32] == 0).all() and (got[1][2][:16] == 0).all()
    np.testing.assert_array_equal(got[0][1][:16], good[0][1][:16])
    status.zero_()
    c.append(lengths, *new, status=status.data_ptr())
    c.table.copy_(table)
    assert status.tolist() == [0, rt.INVALID, rt.INVALID, 0]
    for a, b in zip(c.read(lengths), good):
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y)
    # rows outside the call's: nothing of that sequence is touched
    begin, length = i32([0, 1, 2, 5, 4]), i32(lengths)
    out = torch.full_like(q, 9.0)
    status.zero_()
    c.kv.attention(rt.kv8_batch(4, length.data_ptr(), c.table.data_ptr(), c.stride, max_length=48, rows=4,
                                row_begin_ptr=begin.data_ptr(), max_rows=2),
                   rt.kv8_query(q.data_ptr(), out.data_ptr(), heads=4), ws, status_ptr=status.data_ptr())
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0, rt.INVALID, rt.INVALID]
    assert torch.equal(out[:2], base[:2]) and (out[2:] == 9).all()
    # a query with a NaN is flagged and NaN; its neighbours are not
    q2 = q.clone()
    q2[1, 2, 7], q2[3, 0, 0] = float("nan"), float("inf")
    out, status = attend(lengths, q=q2)
    assert status == [0, rt.NON_FINITE, 0, rt.NON_FINITE]
    assert torch.isnan(out[1, 2]).all() and torch.isnan(out[3, 0]).all()
    keep = torch.ones(4, 4, dtype=torch.bool)
    keep[1, 2] = keep[3, 0] = False
    assert torch.equal(out[keep.cuda()], base[keep.cuda()])


def test_host_refusals(cuda_ok):
    c = Cache(2, 64, [16])
    ws = rt.Kv8Workspace(c.kv)
    x = torch.zeros(16, 2, 64, device="cuda")
    length = i32([16])

    def batch(**kw):
        a = dict(sequences=1, lengths_ptr=length.data_ptr(), pages_ptr=c.table.data_ptr(), page_stride=1,
                 max_length=16) | kw
        return rt.kv8_batch(**a)

    def query(**kw):
        return rt.kv8_query(**(dict(q_ptr=x.data_ptr(), out_ptr=x.data_ptr(), heads=2) | kw))

    rows_ok = rt.kv8_rows(x.data_ptr(), x.data_ptr())
    bad_batches = [dict(sequences=0), dict(lengths_ptr=None), dict(pages_ptr=None), dict(page_stride=0),
                   dict(max_length=17), dict(max_rows=0), dict(rows=2)]
    for kw in bad_batches:
        for call in (lambda: c.kv.append(batch(**kw), rows_ok), lambda: c.kv.read(batch(**kw), rows_ok),
                     lambda: c.kv.attention(batch(**kw), query(), ws)):
            with pytest.raises(rt.CudaError) as e:
                call()
            assert e.value.status == rt.INVALID, kw
    for r in (rt.kv8_rows(None, x.data_ptr()), rt.kv8_rows(x.data_ptr() + 4, x.data_ptr()),
              rt.kv8_rows(x.data_ptr(), x.data_ptr(), stride=120), rt.kv8_rows(x.data_ptr(), x.data_ptr(), stride=132),
              rt.kv8_rows(x.data_ptr(), x.data_ptr(), 2)):
        with pytest.raises(rt.CudaError):
            c.kv.append(batch(), r)
    for kw in (dict(heads=3), dict(heads=0), dict(q_ptr=None), dict(out_ptr=x.data_ptr() + 8), dict(q_stride=100),
               dict(scale=float("nan")), dict(scale=-1.0), dict(type=5)):
        with pytest.raises(rt.CudaError):
            c.kv.attention(batch(), query(**kw), ws)
    with pytest.raises(rt.CudaError):
        c.kv.append(batch(), rows_ok, layer=1)
    begin = i32([0, 0])
    empty = batch(rows=0, row_begin_ptr=begin.data_ptr())
    c.kv.append(empty, rows_ok)  # no row: nothing to do
    c.kv.attention(empty, query(), ws)
    torch.cuda.synchronize()


# ------------------------------------------------------- streams and capture
def test_captured_calls_replay_with_new_lengths(cuda_ok):
    """A decode step (append, attend) captured once and replayed while the device-side lengths advance, on a stream
    of its own, beside another captured step with its own workspace and cache."""
    rng = np.random.default_rng(13)
    steps, n, start = 20, 3, [0, 13, 30]
    sets = []
    for k in range(2):
        c = Cache(2, 64, [s + steps for s in start], seed=k)
        first = [[rows(rng, s, 2, 64) for s in start] for _ in range(2)]
        c.append(start, *first)
        s = dict(c=c, ws=rt.Kv8Workspace(c.kv), length=i32(start), q=torch.empty(n, 4, 64, device="cuda"),
                 k=torch.empty(n, 2, 64, device="cuda"), v=torch.empty(n, 2, 64, device="cuda"),
                 out=torch.empty(n, 4, 64, device="cuda"), stream=torch.cuda.Stream(),
                 held=[[model.Held(2, 64) for _ in start] for _ in range(2)])
        for w in range(2):
            for h, r in zip(s["held"][w], first[w]):
                if len(r):
                    h.append(f64(r))
        s["batch"] = rt.kv8_batch(n, s["length"].data_ptr(), c.table.data_ptr(), c.stride, max_length=c.stride * 16)
        s["rows"] = rt.kv8_rows(s["k"].data_ptr(), s["v"].data_ptr())
        s["query"] = rt.kv8_query(s["q"].data_ptr(), s["out"].data_ptr(), heads=4)
        s["graph"] = torch.cuda.CUDAGraph()
        sets.append(s)
    torch.cuda.synchronize()
    for s in sets:
        with torch.cuda.graph(s["graph"], stream=s["stream"]):
            s["length"] += 1
            st = torch.cuda.current_stream().cuda_stream
            s["c"].kv.append(s["batch"], s["rows"], stream_ptr=st)
            s["c"].kv.attention(s["batch"], s["query"], s["ws"], stream_ptr=st)
    inputs = [[[rows(rng, n, h, 64) for h in (4, 2, 2)] for _ in range(steps)] for _ in sets]
    outs = [[], []]
    torch.cuda.synchronize()
    for t in range(steps):
        for s, x in zip(sets, inputs):
            with torch.cuda.stream(s["stream"]):
                for name, value in zip(("q", "k", "v"), x[t]):
                    s[name].copy_(value)
                s["graph"].replay()
        for s, o in zip(sets, outs):
            with torch.cuda.stream(s["stream"]):
                o.append(s["out"].clone())
    torch.cuda.synchronize()
    for s, x, o in zip(sets, inputs, outs):
        for t in range(steps):
            q, k, v = (f64(a) for a in x[t])
            got = f64(o[t])
            for i in range(n):
                s["held"][0][i].append(k[i:i + 1])
                s["held"][1][i].append(v[i:i + 1])
                kk, vv = s["held"][0][i].values(), s["held"][1][i].values()
                want, size = model.attention(q[i:i + 1], kk, vv)
                bound = model.attention_bound(size, np.abs(vv).max(), want, 64, len(kk), False)
                assert (np.abs(got[i:i + 1] - want) <= bound).all(), (t, i)
    for s in sets:
        s["graph"].reset()


def test_repeated_calls_are_bit_identical(cuda_ok):
    """Splits merge in order, whichever arrives last."""
    rng = np.random.default_rng(14)
    lengths = [3000, 17, 900]
    c = Cache(2, 64, lengths)
    c.append(lengths, *[[rows(rng, n, 2, 64) for n in lengths] for _ in range(2)])
    q = rows(rng, 3, 2, 64)
    ws = rt.Kv8Workspace(c.kv)
    outs = []
    for _ in range(20):
        out = torch.empty_like(q)
        c.kv.attention(c.batch(lengths, [1, 1, 1]), rt.kv8_query(q.data_ptr(), out.data_ptr(), heads=2), ws)
        outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_one_row_appends_refuse_and_keep(cuda_ok):
    """The form for one row a sequence: bad pages, bad lengths, non-finite and extreme values, and what it must leave."""
    rng = np.random.default_rng(15)
    lengths = [17, 18, 33, 5, 1, 40]
    c = Cache(3, 64, lengths)
    first = [n - 1 for n in lengths]
    old = [[rows(rng, n, 3, 64) for n in first] for _ in range(2)]
    c.append(first, *old)
    held = [[model.Held(3, 64) for _ in lengths] for _ in range(2)]
    for w in range(2):
        for h, r in zip(held[w], old[w]):
            h.append(f64(r))
    new = [[rows(rng, 1, 3, 64) * 50 for _ in lengths] for _ in range(2)]  # raises every scale
    new[0][1][0, 0, 3], new[1][1][0, 2, 7] = float("nan"), float("-inf")
    new[0][2][0, 1, :2] = torch.tensor([3e38, -3e38])
    table = c.table.clone()
    c.table[3, 0] = c.pool + 7
    status = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
    told = list(lengths)
    told[5] = -3  # refused: nothing of sequence 5 changes
    k, v = torch.cat(new[0]), torch.cat(new[1])
    length = i32(told)
    batch = rt.kv8_batch(len(lengths), length.data_ptr(), c.table.data_ptr(), c.stride, max_length=48)
    c.kv.append(batch, rt.kv8_rows(k.data_ptr(), v.data_ptr()), status_ptr=status.data_ptr())
    torch.cuda.synchronize()
    assert status.tolist() == [0, rt.NON_FINITE, 0, rt.INVALID, 0, rt.CAPACITY]
    c.table.copy_(table)
    for w in range(2):
        for i, h in enumerate(held[w]):
            if i not in (3, 5):
                h.append(f64(new[w][i]))
    now = [n if i not in (3, 5) else n - 1 for i, n in enumerate(lengths)]
    for got, want in zip(c.read(now), held):
        for g, h in zip(got, want):
            np.testing.assert_array_equal(g, h.values().astype(np.float32))


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_single_rows_equal_one_append(cuda_ok, dim):
    """40 one-row appends, a scale rising inside the block or not, against the definition and the many-row form."""
    rng = np.random.default_rng(dim)
    n = 40
    x = rng.standard_normal((n, 2, dim)) * 4.0 ** rng.integers(-3, 4, (n, 2, 1))
    x[16:32] = x[16:17] / (1 + np.arange(16)[:, None, None])  # never rises
    k = dev(x, torch.float32)
    one, many = Cache(2, dim, [n]), Cache(2, dim, [n])
    h = model.Held(2, dim)
    for t in range(n):
        one.append([t + 1], [k[t:t + 1]], [-k[t:t + 1]])
        h.append(x[t:t + 1].astype(np.float32))
    for t in range(0, n, 2):
        many.append([t + 2], [k[t:t + 2]], [-k[t:t + 2]])
    got = one.read([n])
    np.testing.assert_array_equal(got[0][0], h.values().astype(np.float32))
    np.testing.assert_array_equal(got[1][0], -h.values().astype(np.float32))
    pairs = model.Held(2, dim)
    for t in range(0, n, 2):
        pairs.append(x[t:t + 2].astype(np.float32))
    np.testing.assert_array_equal(many.read([n])[0][0], pairs.values().astype(np.float32))


def test_more_rows_than_positions(cuda_ok):
    """Rows that would lie before position 0 are not written and read as 0."""
    rng = np.random.default_rng(16)
    c = Cache(1, 32, [3, 20])
    k = [rows(rng, 8, 1, 32), rows(rng, 8, 1, 32)]
    v = [rows(rng, 8, 1, 32), rows(rng, 8, 1, 32)]
    c.append([3, 8], k, v)
    for got, new in zip(c.read([3, 8], [5, 8]), (k, v)):
        for g, r, n in zip(got, new, (3, 8)):
            h = model.Held(1, 32)
            h.append(f64(r[8 - n:]))
            assert (g[:len(g) - n] == 0).all()
            np.testing.assert_array_equal(g[len(g) - n:], h.values().astype(np.float32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group,count", [(1, 1), (1, 20)])
def test_all_keys_alike_and_one_key_far_ahead(cuda_ok, group, count, dtype):
    """Flat softmax over many keys, and one that a single key takes: the weights at both ends of their range."""
    n = 2000
    rng = np.random.default_rng(17)
    k = np.ones((n, 1, 64), np.float32)
    far = k.copy()
    far[::2] *= -1
    far[777] = 100.0
    c = Cache(1, 64, [n, n])
    v = rows(rng, n, 1, 64, dtype)
    c.append([n, n], [dev(k).to(dtype), dev(far).to(dtype)], [v, v])
    q = torch.full((2 * count, group, 64), 1.5, device="cuda").to(dtype)
    out = torch.empty_like(q)
    kind = rt.ROWS_BF16 if dtype == torch.bfloat16 else rt.ROWS_F32
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(c.batch([n, n], [count, count]), rt.kv8_query(q.data_ptr(), out.data_ptr(), kind, heads=group), ws)
    torch.cuda.synchronize()
    for i, keys in enumerate((k, far)):
        hk, hv = model.Held(1, 64), model.Held(1, 64)
        hk.append(keys)
        hv.append(f64(v))
        part = f64(q[i * count:(i + 1) * count])
        want, size = model.attention(part, hk.values(), hv.values())
        bound = model.attention_bound(size, np.abs(hv.values()).max(), want, 64, n, dtype == torch.bfloat16)
        assert (np.abs(f64(out[i * count:(i + 1) * count]) - want) <= bound).all()


# ------------------------------------------- many rows (the 128-row kernel)
# Calls with work enough for it: all rows * query heads * pages of the longest
# 454656 or more (148 SMs), 64 rows of a K/V head or more. Row tiles of one row, of 128 and of
# 129 to 256 (two streams); splits; every tile edge among the lengths.
MANY = [
    # kv_heads, group, dim, lengths, rows, window
    (2, 1, 64, [4100, 1, 0, 16, 17, 127, 128, 129, 300, 2048, 5, 5, 5, 31, 33], 128, 0),
    (1, 8, 128, [2000, 20, 1, 513] * 6, 40, 0),
    (3, 1, 32, [1500, 129, 300, 0] * 8, 129, 0),
    (2, 3, 64, [1000, 90, 33] * 20, 43, 0),
    (8, 2, 64, [600, 30, 599] * 14, 100, 77),
    (1, 5, 32, [8000], 400, 0),
    (4, 1, 128, [8190], 450, 0),
    (8, 1, 64, [300, 17, 2] * 36, 64, 1),
    (2, 4, 128, [260, 1100] * 16, 100, 500),
    (4, 64, 64, [1333, 5] * 22, 1, 0),
    (8, 1, 128, [640, 641, 255] * 16, 256, 0),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv_heads,group,dim,lengths,count,window", MANY)
def test_many_rows_against_the_definition(cuda_ok, kv_heads, group, dim, lengths, count, window, dtype):
    test_attention_against_the_definition(cuda_ok, kv_heads, group, dim, lengths, count, window, dtype)


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_many_rows_of_bad_q_and_bad_pages(cuda_ok, dim):
    """A row of q that is not finite is NaN and flagged, alone; a page id outside the pool hides its positions."""
    rng = np.random.default_rng(18)
    lengths, count = [300, 420] + [1000] * 60, 130
    c = Cache(2, dim, lengths)
    new = [[rows(rng, n, 2, dim) for n in lengths] for _ in range(2)]
    c.append(lengths, *new)
    held = [[model.Held(2, dim) for _ in range(2)] for _ in range(2)]
    for w in range(2):
        for h, r in zip(held[w], new[w]):
            h.append(f64(r))
    q = rows(rng, len(lengths) * count, 2, dim)
    q[5, 0, 3] = float("inf")
    q[129, 1, dim - 1] = float("nan")
    c.table[1, 2] = c.pool  # positions 32..47 of the second sequence
    out = torch.empty_like(q)
    status = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(c.batch(lengths, [count] * len(lengths)), rt.kv8_query(q.data_ptr(), out.data_ptr(), heads=2), ws,
                   status_ptr=status.data_ptr())
    torch.cuda.synchronize()
    assert status.tolist() == [rt.NON_FINITE, rt.INVALID] + [0] * 60
    got = f64(out)
    bad = np.zeros((len(got), 2), bool)
    bad[5, 0] = bad[129, 1] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    good = np.where(bad[:, :, None], 0.0, f64(q))
    for i, n in enumerate(lengths[:2]):
        k, v = held[0][i].values(), held[1][i].values()
        part = good[i * count:(i + 1) * count]
        want, size = model.attention(part, k, v)
        if i == 1:  # every row sees position 47: without them the sequence is 16 positions shorter
            keep = np.r_[0:32, 48:n]
            want, _ = model.attention(part, k[keep], v[keep])
        bound = model.attention_bound(size, np.abs(v).max(), want, dim, n, False)
        ok = ~bad[i * count:(i + 1) * count]
        assert (np.abs(got[i * count:(i + 1) * count] - want) <= bound)[ok].all()


def test_many_rows_scaled_strided_and_very_different_blocks(cuda_ok):
    """A scale, rows inside wider ones, and values and scores over a wide range."""
    rng = np.random.default_rng(20)
    lengths, count = [200, 77] + [1000] * 28, 256
    c = Cache(2, 64, lengths)
    keys = [rows(rng, n, 2, 64) for n in lengths]
    values = [rows(rng, n, 2, 64) * torch.exp2(torch.randint(-30, 31, (n, 1, 1), device="cuda")).float() for n in lengths]
    c.append(lengths, keys, values)
    q = rows(rng, len(lengths) * count, 6, 64)  # 2 heads of queries, 2 of outputs, 2 untouched
    before = q.clone()
    ws = rt.Kv8Workspace(c.kv)
    c.kv.attention(c.batch(lengths, [count] * len(lengths)),
                   rt.kv8_query(q.data_ptr(), q.data_ptr() + 2 * 64 * 4, heads=2, scale=0.7, q_stride=384, out_stride=384), ws)
    torch.cuda.synchronize()
    assert torch.equal(q[:, :2], before[:, :2]) and torch.equal(q[:, 4:], before[:, 4:])
    for i, n in enumerate(lengths[:3]):
        hk, hv = model.Held(2, 64), model.Held(2, 64)
        hk.append(f64(keys[i]))
        hv.append(f64(values[i]))
        want, size = model.attention(f64(before[i * count:(i + 1) * count, :2]), hk.values(), hv.values(), scale=0.7)
        biggest = np.maximum.accumulate(np.abs(hv.values()).max((1, 2)))  # among what a row sees
        seen = np.arange(n - count, n)
        most = np.where(seen >= 0, biggest[np.maximum(seen, 0)], 0.0)[:, None, None]
        bound = model.attention_bound(size, 1.0, 0 * want, 64, n, False) * most + 2.0 ** -23 * np.abs(want)
        assert (np.abs(f64(q[i * count:(i + 1) * count, 2:4]) - want) <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows_repeat_bit_for_bit_and_in_graphs(cuda_ok, dtype):
    """Split and unsplit calls: the same bits from every call and replay, whichever split arrives last."""
    rng = np.random.default_rng(19)
    kind = rt.ROWS_BF16 if dtype == torch.bfloat16 else rt.ROWS_F32
    for kv_heads, lengths, count in ((4, [8000], 480), (8, [700, 20, 350, 900] * 8, 70)):
        c = Cache(kv_heads, 64, lengths)
        c.append(lengths, *[[rows(rng, n, kv_heads, 64, dtype) for n in lengths] for _ in range(2)])
        q = rows(rng, count * len(lengths), kv_heads, 64, dtype)
        ws = rt.Kv8Workspace(c.kv)
        outs = [torch.empty_like(q) for _ in range(3)]
        batch = c.batch(lengths, [count] * len(lengths))

        def call(out, stream=0):
            c.kv.attention(batch, rt.kv8_query(q.data_ptr(), out.data_ptr(), kind, heads=kv_heads), ws, stream_ptr=stream)

        call(outs[0])
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(outs[1], torch.cuda.current_stream().cuda_stream)
            call(outs[2], torch.cuda.current_stream().cuda_stream)
        for _ in range(5):
            outs[1].zero_()
            outs[2].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_scales_past_the_bound_are_refused(cuda_ok):
    c = Cache(1, 64, [4])
    q = torch.zeros(1, 1, 64, device="cuda")
    ws = rt.Kv8Workspace(c.kv)
    for scale, fine in ((1e30, True), (2e30, False), (float("inf"), False)):
        query = rt.kv8_query(q.data_ptr(), q.data_ptr(), heads=1, scale=scale)
        if fine:
            c.kv.attention(c.batch([4], [1]), query, ws)
        else:
            with pytest.raises(rt.CudaError):
                c.kv.attention(c.batch([4], [1]), query, ws)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows_padded_and_on_two_streams_at_once(cuda_ok, dtype):
    """Row and length bounds far above the batch's own, a sequence without rows, rows behind the last one left as they
    were; and calls of two streams at once, a workspace each, give the bits of a call alone."""
    rng = np.random.default_rng(23)
    kind = rt.ROWS_BF16 if dtype == torch.bfloat16 else rt.ROWS_F32
    lengths, counts = [1500, 40, 900, 1500, 700, 1200] * 4, [200, 0, 129, 128, 256, 70] * 4
    c = Cache(4, 64, lengths)
    c.append(lengths, *[[rows(rng, n, 4, 64, dtype) for n in lengths] for _ in range(2)])
    q = rows(rng, sum(counts) + 5, 8, 64, dtype)
    ws = [rt.Kv8Workspace(c.kv) for _ in range(2)]
    tight, loose = c.batch(lengths, counts), c.batch(lengths, counts, max_rows=1000)
    outs = [torch.full_like(q, 3.0) for _ in range(6)]

    def call(batch, out, w, stream=0):
        c.kv.attention(batch, rt.kv8_query(q.data_ptr(), out.data_ptr(), kind, heads=8), ws[w], stream_ptr=stream)

    call(tight, outs[0], 0)
    call(loose, outs[1], 0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for k in range(2):
        for w in range(2):
            call(tight, outs[2 + 2 * k + w], w, streams[w].cuda_stream)
    torch.cuda.synchronize()
    for out in outs:
        assert torch.isfinite(out.float()).all() and (out[sum(counts):] == 3).all()
    for out in outs[2:]:
        assert torch.equal(outs[0], out)
    # Other bounds may split the positions elsewhere: the same up to both calls' roundings. bf16: the outputs' own, 2^-8
    # each. fp32: 24 turns of 64 positions, a sum of 16 truncated steps a turn, 2^-23 each: 2 * 40 * 2^-23.
    close = 2.0 ** -7 if dtype == torch.bfloat16 else 1e-5
    assert (outs[0] - outs[1]).float().norm() <= close * outs[0].float().norm()


def test_attention_in_place_with_another_stride_is_refused(cuda_ok):
    c = Cache(1, 64, [4, 4])
    q = torch.zeros(4, 1, 64, device="cuda")
    ws = rt.Kv8Workspace(c.kv)
    with pytest.raises(rt.CudaError) as e:
        c.kv.attention(c.batch([4, 4], [1, 1]), rt.kv8_query(q.data_ptr(), q.data_ptr(), heads=1, q_stride=128), ws)
    assert e.value.status == rt.INVALID
    c.kv.attention(c.batch([4, 4], [1, 1]), rt.kv8_query(q.data_ptr(), q.data_ptr(), heads=1, q_stride=128, out_stride=128), ws)
    torch.cuda.synchronize()
