"""Per-head norm and rotation on device rows against the formula in 64 bits."""
import math

import numpy as np
import pytest

from phonon_b200 import runtime as rt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def formula(x, weight, positions, rotary, halves, eps, theta):
    """[rows][heads][dim] in 64 bits."""
    y = x.copy()
    if weight is not None:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps) * weight
    angle = positions[:, None, None] * theta ** (-np.arange(0, rotary, 2) / rotary)
    c, s = np.cos(angle), np.sin(angle)
    if halves:
        a, b = y[..., :rotary // 2].copy(), y[..., rotary // 2:rotary].copy()
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = a * c - b * s, a * s + b * c
    else:
        a, b = y[..., 0:rotary:2].copy(), y[..., 1:rotary:2].copy()
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * c - b * s, a * s + b * c
    return y


def bound(x, weight, rotary, eps, out, bf16):
    """Per element. u = 2^-23. The norm: dim/4 + 8 additions and products of positive terms and a division, a root
    and two products, under (dim/8 + 12) u relative. The rotation: an angle within 2^-25 turns (2 pi 2^-25 < 2u) and
    sine and cosine within 2u each, of both values of a pair, and two rounded operations. bf16 rounds the result once, by 2^-8 of it."""
    u = 2.0 ** -23
    y = np.abs(formula(x, weight, np.zeros(len(x)), rotary, False, eps, 1e4))
    most = y.max(-1, keepdims=True)  # of a pair, generously of the head
    return 2 * most * ((x.shape[-1] / 8 + 12) + 8) * u + (2.0 ** -8 if bf16 else 0) * np.abs(out) + 1e-37


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,rotary,halves,norms", [
    (1, 8, 8, 64, 64, False, "qk"), (64, 8, 8, 64, 64, False, ""), (7, 5, 1, 128, 96, True, "qk"),
    (33, 3, 2, 32, 24, True, "k"), (5, 1, 0, 32, 2, False, "q"), (9, 0, 3, 64, 6, False, "k"),
    (300, 32, 8, 128, 128, True, "qk"), (2, 7, 7, 32, 8, True, "qk"), (1000, 2, 1, 128, 30, False, "q"),
])
def test_against_the_formula(cuda_ok, rows, heads, kv_heads, dim, rotary, halves, norms, bf16):
    rng = np.random.default_rng(rows + dim)
    dtype = torch.bfloat16 if bf16 else torch.float32
    packed = torch.tensor(rng.standard_normal((rows, heads + 2 * kv_heads, dim)) * 3, dtype=torch.float32).to(dtype).cuda()
    q, k = packed[:, :heads], packed[:, heads:heads + kv_heads]
    positions = rng.integers(0, 2_000_000, rows)
    positions[0] = 0
    weights = {c: torch.tensor(1 + 0.3 * rng.standard_normal(dim), dtype=torch.float32, device="cuda") for c in norms}
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    q_out = torch.full((rows + 1, heads, dim), 7.0, dtype=dtype, device="cuda")
    k_out = torch.full((rows + 1, kv_heads + 1, dim), 7.0, dtype=dtype, device="cuda")
    status = torch.zeros(rows, dtype=torch.int32, device="cuda")
    call = rt.QkNormRope(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), rows, heads, kv_heads, dim,
                         pos.data_ptr(), rt.ROWS_BF16 if bf16 else rt.ROWS_F32, q_stride=packed.stride(0),
                         k_stride=packed.stride(0), k_out_stride=(kv_heads + 1) * dim,
                         q_weight_ptr=weights["q"].data_ptr() if "q" in weights else None,
                         k_weight_ptr=weights["k"].data_ptr() if "k" in weights else None, epsilon=1e-5,
                         theta=500000.0, rotary_dim=rotary, halves=halves)
    call(status.data_ptr())
    torch.cuda.synchronize()
    assert not status.any() and (q_out[rows:] == 7).all() and (k_out[rows:] == 7).all() and (k_out[:, kv_heads:] == 7).all()
    for got, x, side in ((q_out[:rows], q, "q"), (k_out[:rows, :kv_heads], k, "k")):
        if not x.numel():
            continue
        x = x.double().cpu().numpy()
        w = weights[side].double().cpu().numpy() if side in weights else None
        want = formula(x, w, positions, rotary, halves, 1e-5, 500000.0)
        err = np.abs(got.double().cpu().numpy() - want)
        assert (err <= bound(x, w, rotary, 1e-5, want, bf16)).all()


@pytest.mark.parametrize("theta", [1.0, 0.01, 1e6])
def test_frequencies_of_any_base(cuda_ok, theta):
    """Bases below 1 turn more than once a position; far and negative positions."""
    rng = np.random.default_rng(7)
    x = torch.tensor(rng.standard_normal((6, 1, 64)), dtype=torch.float32, device="cuda")
    positions = np.array([0, 1, -1, 4_000_000, -77_777, 12])
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    rt.QkNormRope(x.data_ptr(), None, out.data_ptr(), None, 6, 1, 0, 64, pos.data_ptr(), theta=theta)()
    torch.cuda.synchronize()
    theta = float(np.float32(theta))  # the argument is a float: 0.01 is not one
    want = formula(x.double().cpu().numpy(), None, positions, 64, False, 1e-6, theta)
    # a frequency f is within 2^-53 of itself (the library's exp2): |position| f 2^-52 of an angle, in either form
    freq = theta ** (-np.arange(0, 64, 2) / 64)
    slack = np.repeat(np.abs(positions)[:, None] * freq * 2.0 ** -51, 2, -1)[:, None] * np.abs(x.cpu().numpy()).max()
    lim = bound(x.double().cpu().numpy(), None, 64, 1e-6, want, False) + slack
    assert (np.abs(out.double().cpu().numpy() - want) <= lim).all()


def test_in_place_on_a_stream_and_non_finite_rows(cuda_ok):
    rng = np.random.default_rng(5)
    x = torch.tensor(rng.standard_normal((40, 6, 64)), dtype=torch.float32, device="cuda")
    x[3, 1, 2], x[17, 5, 0] = float("inf"), float("nan")
    start = x.double().cpu().numpy()
    pos = torch.arange(40, dtype=torch.int32, device="cuda")
    w = torch.ones(64, device="cuda")
    status = torch.zeros(40, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    call = rt.QkNormRope(x.data_ptr(), x[:, 4:].data_ptr(), x.data_ptr(), x[:, 4:].data_ptr(), 40, 4, 2, 64,
                         pos.data_ptr(), q_stride=384, k_stride=384, q_out_stride=384, k_out_stride=384,
                         q_weight_ptr=w.data_ptr(), k_weight_ptr=w.data_ptr())
    call(status.data_ptr(), stream.cuda_stream)
    stream.synchronize()
    assert [i for i, s in enumerate(status.tolist()) if s] == [3, 17]
    assert set(status.tolist()) == {0, rt.NON_FINITE}
    fine = np.ones((40, 6), bool)
    fine[3, 1] = fine[17, 5] = False
    want = formula(np.where(fine[..., None], start, 0.0), np.ones(64), np.arange(40), 64, False, 1e-6, 10000.0)
    err = np.abs(x.double().cpu().numpy() - want)[fine]
    assert (err <= bound(np.where(fine[..., None], start, 0.0), np.ones(64), 64, 1e-6, want, False)[fine]).all()


def test_refusals(cuda_ok):
    x = torch.zeros(4, 2, 64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    good = dict(q_ptr=x.data_ptr(), k_ptr=x.data_ptr(), q_out_ptr=x.data_ptr(), k_out_ptr=x.data_ptr(), rows=4, heads=2,
                kv_heads=2, head_dim=64, positions_ptr=pos.data_ptr())
    for kw in (dict(heads=0, kv_heads=0), dict(head_dim=48), dict(rotary_dim=0), dict(rotary_dim=66), dict(rotary_dim=3),
               dict(rotary_dim=12, halves=True), dict(positions_ptr=None), dict(theta=0.0), dict(theta=math.inf),
               dict(epsilon=-1.0), dict(q_ptr=None), dict(k_out_ptr=x.data_ptr() + 4), dict(q_stride=64),
               dict(q_weight_ptr=x.data_ptr() + 8), dict(type=2)):
        with pytest.raises(rt.CudaError) as e:
            rt.QkNormRope(**(good | kw))()
        assert e.value.status == rt.INVALID, kw
    rt.QkNormRope(**(good | dict(rows=0)))()


def test_a_layer_of_device_calls(cuda_ok):
    """The calls as a layer uses them: queries and keys normed and rotated out of the packed projection, keys and
    values appended to the 8-bit cache, attention, for a prompt and then row by row, against the same steps in 64 bits."""
    import kv8_model as model
    rng = np.random.default_rng(21)
    heads, kv_heads, dim, prompt, steps = 4, 2, 64, 37, 12
    total = prompt + steps
    packed = torch.tensor(rng.standard_normal((total, heads + 2 * kv_heads, dim)), dtype=torch.float32, device="cuda")
    w = [torch.tensor(1 + 0.2 * rng.standard_normal(dim), dtype=torch.float32, device="cuda") for _ in range(2)]
    pos = torch.arange(total, dtype=torch.int32, device="cuda")
    q, k = torch.empty(total, heads, dim, device="cuda"), torch.empty(total, kv_heads, dim, device="cuda")
    out = torch.empty_like(q)
    kv = rt.Kv8Cache(kv_heads, dim, 8)
    ws = rt.Kv8Workspace(kv)
    table = torch.tensor([5, 2, 7, 0], dtype=torch.int32, device="cuda")
    keep = []

    def layer(a, b):
        rt.QkNormRope(packed[a:].data_ptr(), packed[a:, heads:].data_ptr(), q[a:].data_ptr(), k[a:].data_ptr(), b - a,
                      heads, kv_heads, dim, pos[a:].data_ptr(), q_stride=packed.stride(0), k_stride=packed.stride(0),
                      q_weight_ptr=w[0].data_ptr(), k_weight_ptr=w[1].data_ptr())()
        begin = torch.tensor([0, b - a], dtype=torch.int32, device="cuda")
        length = torch.tensor([b], dtype=torch.int32, device="cuda")
        v = packed[a:b, heads + kv_heads:].contiguous()
        keep.extend([begin, length, v])
        batch = rt.kv8_batch(1, length.data_ptr(), table.data_ptr(), 4, max_length=64, rows=b - a,
                             row_begin_ptr=begin.data_ptr(), max_rows=b - a)
        kv.append(batch, rt.kv8_rows(k[a:].data_ptr(), v.data_ptr()))
        kv.attention(batch, rt.kv8_query(q[a:].data_ptr(), out[a:].data_ptr(), heads=heads), ws)

    layer(0, prompt)
    for t in range(prompt, total):
        layer(t, t + 1)
    torch.cuda.synchronize()
    x = packed.double().cpu().numpy()
    # the cache is fed the kernel's own keys: their rounding to 8 bits is not the formula's to predict
    held = [model.Held(kv_heads, dim) for _ in range(2)]
    for a, b in [(0, prompt)] + [(t, t + 1) for t in range(prompt, total)]:
        held[0].append(k[a:b].double().cpu().numpy())
        held[1].append(x[a:b, heads + kv_heads:])
        qa = q[a:b].double().cpu().numpy()
        want_q = formula(x[a:b, :heads], w[0].double().cpu().numpy(), np.arange(a, b), dim, False, 1e-6, 10000.0)
        assert (np.abs(qa - want_q) <= bound(x[a:b, :heads], w[0].double().cpu().numpy(), dim, 1e-6, want_q, False)).all()
        vals = held[1].values()
        want, size = model.attention(qa, held[0].values(), vals)
        lim = model.attention_bound(size, np.abs(vals).max(), want, dim, b, False)
        assert (np.abs(out[a:b].double().cpu().numpy() - want) <= lim).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,heads,kv_heads,dim", [(3, 8, 8, 64), (1, 5, 0, 64), (40, 3, 1, 128), (7, 1, 9, 32), (2000, 5, 2, 32)])
def test_no_epsilon_flags_no_fine_row(cuda_ok, rows, heads, kv_heads, dim, bf16):
    """epsilon 0 and head counts that leave passes partly empty: outputs are finite, and so says the status."""
    rng = np.random.default_rng(heads)
    dtype = torch.bfloat16 if bf16 else torch.float32
    x = torch.tensor(rng.standard_normal((rows, heads + kv_heads, dim)), dtype=torch.float32).to(dtype).cuda()
    positions = np.arange(rows)
    pos = torch.tensor(positions, dtype=torch.int32, device="cuda")
    w = torch.tensor(1 + 0.3 * rng.standard_normal(dim), dtype=torch.float32, device="cuda")
    out = torch.empty_like(x)
    status = torch.zeros(rows, dtype=torch.int32, device="cuda")
    wide = (heads + kv_heads) * dim
    rt.QkNormRope(x.data_ptr(), x[:, heads:].data_ptr(), out.data_ptr(), out[:, heads:].data_ptr(), rows, heads, kv_heads, dim,
                  pos.data_ptr(), rt.ROWS_BF16 if bf16 else rt.ROWS_F32, q_stride=wide, k_stride=wide, q_out_stride=wide,
                  k_out_stride=wide, q_weight_ptr=w.data_ptr(), k_weight_ptr=w.data_ptr(), epsilon=0.0)(status.data_ptr())
    torch.cuda.synchronize()
    assert not status.any()
    want = formula(x.double().cpu().numpy(), w.double().cpu().numpy(), positions, dim, False, 0.0, 10000.0)
    lim = bound(x.double().cpu().numpy(), w.double().cpu().numpy(), dim, 0.0, want, bf16)
    assert (np.abs(out.double().cpu().numpy() - want) <= lim).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size,eps", [(1e30, 1e-6), (1e19, 1e-6), (3e37, 0.0), (1e-20, 0.0), (1e-30, 0.0), (1e-36, 1e-72), (1e-12, 1e-26)])
def test_squares_outside_the_range_of_floats(cuda_ok, size, eps, bf16):
    """Rows whose squares overflow or vanish in 32 bits, beside an ordinary head, have the formula's norm."""
    rng = np.random.default_rng(int(abs(math.log10(size))))
    dtype = torch.bfloat16 if bf16 else torch.float32
    x = torch.tensor(rng.standard_normal((9, 5, 64)) * np.array([size, 1.0, size, 1.0, size])[None, :, None], dtype=torch.float32).to(dtype).cuda()
    pos = torch.arange(9, dtype=torch.int32, device="cuda")
    w = torch.tensor(1 + 0.3 * rng.standard_normal(64), dtype=torch.float32, device="cuda")
    out = torch.empty_like(x)
    status = torch.zeros(9, dtype=torch.int32, device="cuda")
    rt.QkNormRope(x.data_ptr(), None, out.data_ptr(), None, 9, 5, 0, 64, pos.data_ptr(), rt.ROWS_BF16 if bf16 else rt.ROWS_F32,
                  q_weight_ptr=w.data_ptr(), epsilon=eps)(status.data_ptr())
    torch.cuda.synchronize()
    assert not status.any()
    eps = float(np.float32(eps))
    want = formula(x.double().cpu().numpy(), w.double().cpu().numpy(), np.arange(9), 64, False, eps, 10000.0)
    lim = bound(x.double().cpu().numpy(), w.double().cpu().numpy(), 64, eps, want, bf16)
    assert (np.abs(out.double().cpu().numpy() - want) <= lim).all()


def test_outputs_that_overflow_bf16_are_flagged(cuda_ok):
    """Finite in 32 bits, infinite once rounded: values from 3.3953e38 on."""
    x = torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    for weight, flagged in ((3.4e38, True), (3.38e38, False)):
        w = torch.full((64,), weight, device="cuda")
        status = torch.zeros(3, dtype=torch.int32, device="cuda")
        rt.QkNormRope(x.data_ptr(), None, out.data_ptr(), None, 3, 1, 0, 64, pos.data_ptr(), rt.ROWS_BF16, q_weight_ptr=w.data_ptr(),
                      epsilon=0.0)(status.data_ptr())
        torch.cuda.synchronize()
        assert torch.isinf(out).all().item() == flagged and status.tolist() == [rt.NON_FINITE if flagged else 0] * 3


def test_a_larger_code_stays(cuda_ok):
    """Status words that hold a larger code already (an expired wait, a bad length) keep it."""
    x = torch.full((4, 1, 64), float("nan"), device="cuda")
    x[3] = 1.0
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    status = torch.tensor([rt.DEVICE_ERROR, 0, rt.CAPACITY, rt.INVALID], dtype=torch.int32, device="cuda")
    rt.QkNormRope(x.data_ptr(), None, x.data_ptr(), None, 4, 1, 0, 64, pos.data_ptr())(status.data_ptr())
    torch.cuda.synchronize()
    assert status.tolist() == [rt.DEVICE_ERROR, rt.NON_FINITE, rt.CAPACITY, rt.INVALID]


def test_in_place_with_another_stride_is_refused(cuda_ok):
    x = torch.zeros(4, 2, 64, device="cuda")
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    for rows, refused in ((4, True), (1, False)):
        call = rt.QkNormRope(x.data_ptr(), None, x.data_ptr(), None, rows, 1, 0, 64, pos.data_ptr(), q_stride=128)
        if refused:
            with pytest.raises(rt.CudaError) as e:
                call()
            assert e.value.status == rt.INVALID
        else:
            call()
    torch.cuda.synchronize()
