"""Rows in 8 bits and their product with 8-bit weights against the formulas in
64 bits."""
import numpy as np
import pytest

from phonon_b200 import runtime as rt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def quantized(x):
    """(integers, scales) of rows x in 64 bits; the scales are numbers of 32 bits."""
    top = np.abs(x).max(1)
    scales = np.maximum((top / 127).astype(np.float32), np.float32(2.0 ** -126)).astype(np.float64)
    return np.rint(x / scales[:, None]), scales


def run_quantize(x, bf16, x_stride=0, q_stride=0, status=None, stream=0):
    rows, cols = x.shape
    q = torch.full((rows + 1, q_stride or cols), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((rows + 1,), -3.0, device="cuda")
    rt.QuantizeRows(x.data_ptr(), q.data_ptr(), scales.data_ptr(), rows, cols, rt.ROWS_BF16 if bf16 else rt.ROWS_F32,
                    x_stride, q_stride)(None if status is None else status.data_ptr(), stream)
    torch.cuda.synchronize()
    assert (q[rows:] == 77).all() and (q[:, cols:] == 77).all() and (scales[rows:] == -3).all()
    return q[:rows, :cols].cpu().numpy().astype(np.float64), scales[:rows].double().cpu().numpy()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 16), (64, 512), (3, 256), (9, 272), (7, 1024), (5, 1040), (300, 4096), (2, 4112),
                                       (3, 8192), (33, 8208), (1, 40016), (70000, 16)])
def test_rows_become_the_nearest_integers(cuda_ok, rows, cols, bf16):
    rng = np.random.default_rng(rows + cols)
    x = rng.standard_normal((rows, cols)) * np.exp(3 * rng.standard_normal((rows, 1)))
    x = torch.tensor(x, dtype=torch.float32).to(torch.bfloat16 if bf16 else torch.float32).cuda()
    status = torch.zeros(rows, dtype=torch.int32, device="cuda")
    q, scales = run_quantize(x, bf16, status=status)
    want_q, want_s = quantized(x.double().cpu().numpy())
    assert not status.any()
    assert np.array_equal(scales, want_s) and np.array_equal(q, want_q)


def test_ties_borders_and_the_ends_of_the_range(cuda_ok):
    """Quotients of exactly and of nearly k + 1/2, rows of zeros, of the smallest numbers, of the largest."""
    rng = np.random.default_rng(1)
    rows = []
    for scale in (1.0, 2.0 ** -100, 0.37, 3.1e30, 1.7e-38):
        s = np.float32(max(np.float32(127 * scale) / np.float32(127), 2.0 ** -126))
        k = rng.integers(-127, 127, 512)
        near = ((k + 0.5) * float(s)).astype(np.float32)
        row = np.where(rng.random(512) < 0.4, near, np.nextafter(near, np.where(rng.random(512) < 0.5, 1, -1) * np.float32(np.inf), dtype=np.float32))
        row[0] = np.float32(127 * scale)
        rows.append(np.clip(row, -row[0], row[0]))
    rows.append(np.zeros(512, np.float32))
    rows.append((rng.integers(-5, 6, 512) * np.float64(2.0 ** -149)).astype(np.float32))
    rows.append((rng.standard_normal(512) * 1e38).clip(-3.4028234e38, 3.4028234e38).astype(np.float32))
    x = np.stack(rows)
    x[-1, 7] = np.finfo(np.float32).max
    q, scales = run_quantize(torch.tensor(x).cuda(), False)
    want_q, want_s = quantized(x.astype(np.float64))
    assert np.array_equal(scales, want_s) and np.array_equal(q, want_q)


def test_strided_rows_on_a_stream_and_non_finite_ones(cuda_ok):
    rng = np.random.default_rng(2)
    wide = torch.tensor(rng.standard_normal((20, 3 * 528)), dtype=torch.float32).cuda()
    x = wide[:, 528:1056]
    x[3, 100], x[4, 0], x[19, 527] = float("inf"), float("-inf"), float("nan")
    status = torch.zeros(20, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    q, scales = run_quantize(x, False, x_stride=wide.stride(0), q_stride=544, status=status, stream=stream.cuda_stream)
    bad = np.isin(np.arange(20), (3, 4, 19))
    assert status.tolist() == [rt.NON_FINITE if b else 0 for b in bad]
    want_q, want_s = quantized(np.where(bad[:, None], 0, x.double().cpu().numpy()))
    assert np.isnan(scales[bad]).all() and (q[bad] == 0).all()
    assert np.array_equal(scales[~bad], want_s[~bad]) and np.array_equal(q[~bad], want_q[~bad])


def product_case(rng, rows, channels, depth, full=False):
    low = -128 if full else -127
    x = torch.tensor(rng.integers(low, 128, (rows, depth)), dtype=torch.int8, device="cuda")
    w = torch.tensor(rng.integers(low, 128, (channels, depth)), dtype=torch.int8, device="cuda")
    xs = torch.tensor(np.exp(rng.standard_normal(rows)), dtype=torch.float32, device="cuda")
    ws = torch.tensor(np.exp(rng.standard_normal(channels)) / depth, dtype=torch.float32, device="cuda")
    return x, w, xs, ws


def product_want(x, w, xs, ws, bias):
    """(result, its part before the bias) in 64 bits; the sums are exact in any."""
    y = (x.double() @ w.double().t() * xs.double()[:, None] * ws.double()).cpu().numpy()
    return (y if bias is None else y + bias.double().cpu().numpy()), y


def check_product(got, want, part, bf16):
    """The sum to 32 bits, times x_scale, times w_scale (plus the bias): three roundings of 2^-24 relative to a value of
    the part's size or (the last) the result's; bf16 rounds what comes of it by 2^-8."""
    u = 2.0 ** -24
    lim = (3 * np.abs(part) + np.abs(want)) * u * 1.001
    if bf16:
        lim = lim * 1.01 + 2.0 ** -8 * (np.abs(want) + lim)
    assert (np.abs(got.double().cpu().numpy() - want) <= lim).all()


SHAPES = [(1, 1, 16), (1, 1536, 512), (8, 16, 64), (9, 17, 80), (16, 4096, 4096), (17, 100, 144), (32, 33, 1008),
          (33, 64, 128), (64, 500, 528), (127, 129, 2048), (128, 256, 16), (300, 1001, 272), (513, 512, 2048),
          (1000, 2500, 400), (2049, 4100, 640), (40, 9000, 1040), (5000, 7, 96)]


@pytest.mark.parametrize("bf16,with_bias", [(False, True), (True, False)])
@pytest.mark.parametrize("rows,channels,depth", SHAPES)
def test_product_against_the_formula(cuda_ok, rows, channels, depth, bf16, with_bias):
    rng = np.random.default_rng(rows + channels + depth)
    x, w, xs, ws = product_case(rng, rows, channels, depth)
    bias = torch.tensor(rng.standard_normal(channels), dtype=torch.float32, device="cuda") if with_bias else None
    y = torch.full((rows + 2, channels), 7.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    status = torch.zeros(rows, dtype=torch.int32, device="cuda")
    rt.I8Product(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, channels, depth,
                 rt.ROWS_BF16 if bf16 else rt.ROWS_F32, None if bias is None else bias.data_ptr())(status.data_ptr())
    torch.cuda.synchronize()
    assert not status.any() and (y[rows:] == 7).all()
    check_product(y[:rows], *product_want(x, w, xs, ws, bias), bf16)


@pytest.mark.parametrize("rows,channels", [(3, 40), (20, 40), (200, 300)])
def test_the_largest_sums_are_exact(cuda_ok, rows, channels):
    """All of -128 at the greatest depth: 2^14 (2^17 - 16) is under 2^31; every second row the other way."""
    depth = (1 << 17) - 16
    x = torch.full((rows, depth), -128, dtype=torch.int8, device="cuda")
    w = torch.full((channels, depth), -128, dtype=torch.int8, device="cuda")
    x[1::2] = 127
    one_r, one_c = torch.ones(rows, device="cuda"), torch.ones(channels, device="cuda")
    y = torch.empty(rows, channels, device="cuda")
    rt.I8Product(x.data_ptr(), one_r.data_ptr(), w.data_ptr(), one_c.data_ptr(), y.data_ptr(), rows, channels, depth)()
    torch.cuda.synchronize()
    assert (y[0::2] == float(np.float32(depth * 16384))).all() and (y[1::2] == float(np.float32(-depth * 16256))).all()


@pytest.mark.parametrize("rows,channels", [(5, 70), (24, 70), (150, 330)])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_strided_operands_and_what_lies_between(cuda_ok, rows, channels, pad):
    """Rows of larger arrays; what lies beside the result stays, and what lies beside the operands does not count."""
    rng = np.random.default_rng(pad)
    depth = 208
    x, w, xs, ws = product_case(rng, rows, channels, 3 * depth, full=True)
    y = torch.full((rows, channels + 3 + pad), 7.0, dtype=torch.bfloat16, device="cuda")
    rt.I8Product(x[:, depth:].data_ptr(), xs.data_ptr(), w[:, depth:].data_ptr(), ws.data_ptr(), y.data_ptr(), rows, channels,
                 depth, rt.ROWS_BF16, x_stride=3 * depth, w_stride=3 * depth, y_stride=channels + 3 + pad)()
    torch.cuda.synchronize()
    assert (y[:, channels:] == 7).all()
    want, part = product_want(x[:, depth:2 * depth], w[:, depth:2 * depth], xs, ws, None)
    check_product(y[:, :channels], want, part, True)


@pytest.mark.parametrize("rows", [4, 30, 140])
def test_rows_that_are_not_finite_are_named(cuda_ok, rows):
    rng = np.random.default_rng(rows)
    x, w, xs, ws = product_case(rng, rows, 80, 64)
    xs[2] = float("nan")
    xs[rows - 1] = 3e38  # over fp32's range for some channel
    status = torch.zeros(rows, dtype=torch.int32, device="cuda")
    y = torch.empty(rows, 80, device="cuda")
    rt.I8Product(x.data_ptr(), xs.data_ptr(), w.data_ptr(), (ws * 1e3).data_ptr(), y.data_ptr(), rows, 80, 64)(status.data_ptr())
    torch.cuda.synchronize()
    assert status.tolist() == [rt.NON_FINITE if r in (2, rows - 1) else 0 for r in range(rows)]
    assert y[2].isnan().all() and y[:2].isfinite().all()


def test_captured_and_replayed_with_other_data(cuda_ok):
    """A quantise pass and the product that reads it, captured once, replayed over other rows."""
    rng = np.random.default_rng(4)
    rows, channels, depth = 70, 96, 256
    x = torch.empty(rows, depth, device="cuda")
    _, w, _, ws = product_case(rng, 1, channels, depth)
    q = torch.empty(rows, depth, dtype=torch.int8, device="cuda")
    s = torch.empty(rows, device="cuda")
    y = torch.empty(rows, channels, device="cuda")
    first = rt.QuantizeRows(x.data_ptr(), q.data_ptr(), s.data_ptr(), rows, depth)
    second = rt.I8Product(q.data_ptr(), s.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, channels, depth)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        first(stream_ptr=stream)
        second(stream_ptr=stream)
    for seed in range(3):
        x.copy_(torch.tensor(np.random.default_rng(seed).standard_normal((rows, depth)), dtype=torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        want_q, want_s = quantized(x.double().cpu().numpy())
        assert np.array_equal(q.double().cpu().numpy(), want_q)
        check_product(y, *product_want(q, w, s, ws, None), False)


def test_refusals(cuda_ok):
    a = torch.zeros(4096, device="cuda")
    p = a.data_ptr()

    def status(f, *args, **kw):
        try:
            f(*args, **kw)()
        except rt.CudaError as e:
            return e.status
        return rt.OK

    def quantize(x=p, q=p + 4096, s=p + 8192, rows=2, cols=32, type=rt.ROWS_F32, **kw):
        return status(rt.QuantizeRows, x, q, s, rows, cols, type, **kw)

    assert quantize() == rt.OK and quantize(rows=0) == rt.OK
    for kw in (dict(x=None), dict(q=None), dict(s=None), dict(cols=0), dict(cols=24), dict(type=2), dict(x=p + 8), dict(q=p + 4104),
               dict(x_stride=16), dict(x_stride=36), dict(q_stride=40), dict(q_stride=16), dict(rows=(1 << 30) + 1)):
        assert quantize(**kw) == rt.INVALID, kw

    def product(x=p, xs=p + 4096, w=p + 8192, ws=p + 4096, y=p + 12288, rows=2, channels=16, depth=32, type=rt.ROWS_F32, **kw):
        return status(rt.I8Product, x, xs, w, ws, y, rows, channels, depth, type, **kw)

    assert product() == rt.OK and product(rows=0) == rt.OK
    for kw in (dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(y=None), dict(channels=0), dict(depth=0),
               dict(depth=24), dict(depth=1 << 17), dict(type=3), dict(x=p + 4), dict(w=p + 8200), dict(y=p + 12290),
               dict(x_stride=16), dict(x_stride=40), dict(w_stride=24), dict(y_stride=15), dict(rows=(1 << 30) + 1)):
        assert product(**kw) == rt.INVALID, kw
    torch.cuda.synchronize()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("rows,depth,channels", [(33, 80, (1, 2, 3, 31, 33, 63, 64, 65, 95, 97, 127, 130, 257)),
                                                 (270, 80, (32, 96, 129, 159, 161, 193, 255, 385, 511, 513)),
                                                 (1100, 528, (3001, 4099, 4351, 4353)), (1001, 2064, (4865, 5001, 5121))])
def test_rows_of_every_alignment_and_width(cuda_ok, rows, depth, channels, bf16):
    """Results whose rows start between two words or two sectors, and end in the middle of one, of a tile's half or behind it:
    every element, and none beside them."""
    for n in channels:
        for pad in (0, 1, 2, 6):
            rng = np.random.default_rng(n + pad)
            x, w, xs, ws = product_case(rng, rows, n, depth)
            bias = torch.tensor(rng.standard_normal(n), dtype=torch.float32, device="cuda")
            y = torch.full((rows + 1, n + pad), 7.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
            rt.I8Product(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, n, depth,
                         rt.ROWS_BF16 if bf16 else rt.ROWS_F32, bias_ptr=bias.data_ptr(), y_stride=n + pad)()
            torch.cuda.synchronize()
            check_product(y[:rows, :n], *product_want(x, w, xs, ws, bias), bf16)
            assert (y[rows:] == 7).all() and (y[:, n:] == 7).all()


@pytest.mark.parametrize("rows", [1, 12, 40])
def test_weights_that_the_pass_ahead_has_written(cuda_ok, rows):
    """Weights quantised on the device, the product right behind, again and again over other weights: eager and replayed."""
    rng = np.random.default_rng(rows)
    channels, depth = 2000, 1040
    x, _, xs, _ = product_case(rng, rows, 1, depth)
    raw = torch.empty(channels, depth, device="cuda")
    w, ws = torch.zeros(channels, depth, dtype=torch.int8, device="cuda"), torch.zeros(channels, device="cuda")
    y = torch.empty(rows, channels, device="cuda")
    first = rt.QuantizeRows(raw.data_ptr(), w.data_ptr(), ws.data_ptr(), channels, depth)
    second = rt.I8Product(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, channels, depth)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in (first, second):
            c(stream_ptr=torch.cuda.current_stream().cuda_stream)
    for turn in range(6):
        raw.copy_(torch.tensor(rng.standard_normal((channels, depth)), dtype=torch.float32))
        if turn % 2:
            graph.replay()
        else:
            first(stream_ptr=torch.cuda.current_stream().cuda_stream)
            second(stream_ptr=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        want_q, want_s = quantized(raw.double().cpu().numpy())
        assert np.array_equal(w.double().cpu().numpy(), want_q)
        check_product(y, *product_want(x, torch.tensor(want_q, device="cuda"), xs, torch.tensor(want_s, device="cuda"), None), False)


@pytest.mark.parametrize("exponent", [0, 100, -110, -119, -126, -133])
def test_every_pair_of_bf16_mantissas(cuda_ok, exponent):
    """A row for each mantissa of the largest element, every mantissa at twelve powers of two below: quotients of k + 1/2 but for
    the scale's rounding among them, and (the last exponents) scales at the smallest."""
    m = np.arange(128, 256, dtype=np.float64)
    x = np.concatenate([m * 2.0 ** -j for j in range(12)])
    x = np.where(x[None] <= m[:, None], x[None], m[:, None]) * np.where(np.arange(len(x)) % 2, -1.0, 1.0) * 2.0 ** exponent
    x[:, 0] = m * 2.0 ** exponent
    held = torch.tensor(x).to(torch.bfloat16).cuda()  # (below 2^-133 of the last ones: rounded)
    q, scales = run_quantize(held, True)
    want_q, want_s = quantized(held.double().cpu().numpy())
    assert np.array_equal(scales, want_s) and np.array_equal(q, want_q)


def test_calls_at_the_same_time(cuda_ok):
    """Every kernel of the product on three streams at once, again and again: what each gives alone, bit for bit."""
    rng = np.random.default_rng(12)
    streams = [torch.cuda.Stream() for _ in range(3)]
    jobs = []
    for rows, channels, depth in ((9, 1536, 512), (40, 512, 2048), (512, 1000, 1024), (520, 4096, 4096), (1030, 5003, 2064)):
        x, w, xs, ws = product_case(rng, rows, channels, depth)
        outs = [torch.empty(rows, channels, dtype=torch.bfloat16, device="cuda") for _ in range(len(streams) + 1)]
        calls = [rt.I8Product(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, channels, depth, rt.ROWS_BF16)
                 for y in outs]
        jobs.append((x, w, xs, ws, outs, calls))
    for *_, calls in jobs:
        calls[-1]()
    torch.cuda.synchronize()
    for x, w, xs, ws, outs, _ in jobs:
        check_product(outs[-1], *product_want(x, w, xs, ws, None), True)
    for turn in range(5):
        for i, s in enumerate(streams):
            for j in range(len(jobs)):
                jobs[(j + i + turn) % len(jobs)][-1][i](stream_ptr=s.cuda_stream)
    torch.cuda.synchronize()
    for *_, outs, _ in jobs:
        for y in outs[:-1]:
            assert torch.equal(y, outs[-1])
