"""Attention over packed prompts where values come near the end of the type's range: softmax(...) v is a mean of the values
that a row sees, so finite values give a finite output, however many there are."""
import numpy as np
import pytest

from phonon_b200 import runtime as rt
from test_gpu_prompt import begins, call, formula, rows_of

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def most(bf16):
    return torch.finfo(torch.bfloat16 if bf16 else torch.float32).max


def attend(q, k, v, begin, bf16, **kw):
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    status = torch.zeros(len(begin) - 1, dtype=torch.int32, device="cuda")
    call(q, k, v, out, begin, bf16=bf16, **kw)(status.data_ptr())
    torch.cuda.synchronize()
    return out, status.tolist()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("size", [1e34, 1e37, 3e38])
@pytest.mark.parametrize("window", [0, 100])
def test_large_values(cuda_ok, dim, size, window, bf16):
    """All values of a size, of one sign (head 0) and of both (head 1); scores that rise along the rows, so that the
    maximum that weights are relative to lags behind."""
    rng = np.random.default_rng(dim)
    begin = begins([700, 5, 300])
    packed, q, k, v = rows_of(rng, begin[-1], 4, 2, dim, bf16)
    q[..., 0] = 1.0
    k[..., 0] = torch.linspace(0, 4 * dim ** 0.5, begin[-1], device="cuda").to(q.dtype)[:, None]
    wide = torch.tensor(rng.uniform(-size, size, v.shape), device="cuda")
    wide[:, 0] = wide[:, 0].abs()
    v.copy_(wide.to(v.dtype))
    out, status = attend(q, k, v, begin, bf16, window=window)
    assert status == [0, 0, 0] and out.isfinite().all()
    want, lim = formula(q, k, v, begin, window, tol=bf16)
    assert ((out.double() - want).abs() <= lim).all()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_the_largest_values(cuda_ok, dim, bf16):
    """The mean of equal values is the value: no rounding on the way may carry it over the end."""
    rng = np.random.default_rng(dim + 1)
    begin = begins([1, 2, 9, 400])
    packed, q, k, v = rows_of(rng, begin[-1], 4, 2, dim, bf16)
    v[:, 0], v[:, 1] = most(bf16), -most(bf16)
    out, status = attend(q, k, v, begin, bf16)
    assert status == [0] * 4 and out.isfinite().all()
    want, lim = formula(q, k, v, begin, tol=bf16)
    assert ((out.double() - want).abs() <= lim).all()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("window", [0, 120])
@pytest.mark.parametrize("in_place", [False, True])
def test_rows_beside_them(cuda_ok, in_place, dim, window, bf16):
    """Large values and ones that are not finite in the same prompt: rows that see neither are bit for bit what they are
    without them, rows that see the large ones alone are within their bound, rows that see the others are named."""
    rng = np.random.default_rng(dim + 2)
    begin = begins([420, 300])
    packed, q, k, v = rows_of(rng, begin[-1], 4, 2, dim, bf16)
    clean, status = attend(q, k, v, begin, bf16, window=window)
    assert status == [0, 0]
    v[100:110, 0] = 3e38
    v[100:110, 0, 1] = -3e38
    v[300, 0, dim - 1] = float("nan")
    v[500:503, 1, 3] = most(bf16)
    want, lim = formula(q, k, torch.where(v.isnan(), torch.zeros_like(v), v), begin, window, tol=bf16)
    if in_place:
        out, codes = q, torch.zeros(2, dtype=torch.int32, device="cuda")
        call(q, k, v, q, begin, bf16=bf16, window=window)(codes.data_ptr())
        torch.cuda.synchronize()
        status = codes.tolist()
    else:
        out, status = attend(q, k, v, begin, bf16, window=window)
    assert status == [rt.NON_FINITE, 0]
    at = torch.arange(720, device="cuda")

    def sees(a, b, end):  # one of the positions [a, b)
        return (at >= a) & (at < end) & ((at < b - 1 + window) if window else True)
    broken, large = sees(300, 301, 420), sees(100, 110, 420)
    other = sees(500, 503, 720)
    assert out[broken][:, :2].isnan().any(-1).all() and out[~broken].isfinite().all() and out[:, 2:].isfinite().all()
    assert torch.equal(out[~broken & ~large][:, :2], clean[~broken & ~large][:, :2])
    assert torch.equal(out[~other][:, 2:], clean[~other][:, 2:])
    off = (out.double() - want).abs() <= lim
    assert off[~broken][:, :2].all() and off[:, 2:].all()


@pytest.mark.parametrize("bf16,dim,heads,kvh", [(True, 128, 32, 8), (True, 64, 8, 8), (False, 64, 8, 8)])
def test_large_values_of_many_long_prompts(cuda_ok, dim, heads, kvh, bf16):
    """Enough of them that a CTA has two row tiles; one head's values are large."""
    rng = np.random.default_rng(7)
    begin = begins([900, 1001, 700, 1300, 810, 64, 1100, 1000, 1500, 1200])
    packed, q, k, v = rows_of(rng, begin[-1], heads, kvh, dim, bf16)
    v[:, 1] = (v[:, 1].double() / v[:, 1].double().abs().max() * 3e38).to(v.dtype)
    out, status = attend(q, k, v, begin, bf16)
    assert status == [0] * 10
    want, lim = formula(q, k, v, begin, tol=bf16)
    assert ((out.double() - want).abs() <= lim).all()


@pytest.mark.parametrize("dim", [32, 64, 128])
def test_keys_beyond_the_largest_bf16(cuda_ok, dim):
    """fp32 keys beyond the largest bf16, beside queries so small that every score is a number: weights as of any others, values
    large and small."""
    rng = np.random.default_rng(dim + 3)
    begin = begins([150, 70])
    packed, q, k, v = rows_of(rng, begin[-1], 4, 2, dim, False)
    q[..., 0] = torch.tensor(rng.uniform(-1e-37, 1e-37, q.shape[:2]), dtype=torch.float32, device="cuda")
    k[20, 0, 0], k[90, 1, 0], k[160, 0, 0] = 3.4e38, -3.395e38, most(False)
    v[30, 1] = 3.2e38
    out, status = attend(q, k, v, begin, False)
    assert status == [0, 0]
    want, lim = formula(q, k, v, begin, tol=False)
    # 3.395e38 is nearer to the largest bf16 than to the next power of two, so that it is one of three slices like any other key.
    # Of a query, parts below 2^-133 count as 0: up to 2^-133 * 3.395e38 = 0.0312 of the scores beside that key, and
    # expm1(2 * 0.0312) of a row's weights relative to one another.
    lim[90:150, 2:] += np.expm1(2 * 2.0 ** -133 * 3.395e38) * formula(q, k, v.abs(), begin)[90:150, 2:]
    assert ((out.double() - want).abs() <= lim).all()
