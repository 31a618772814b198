"""Attention over packed prompts with every kind of group: query heads that fill a tile's rows with a K/V head's, leave some of
them empty, or are too many to share them."""
import numpy as np
import pytest

from test_gpu_prompt import begins, call, formula, rows_of

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("group", [5, 9, 12, 17, 24, 31, 32, 33, 40])
def test_groups(cuda_ok, group, dim, bf16):
    rng = np.random.default_rng(group + dim)
    for kvh, lengths, window in ((1, [70, 1, 0, 131], 0), (3, [5, 200, 33], 40)):
        begin = [7 + b for b in begins(lengths)]
        packed, q, k, v = rows_of(rng, begin[-1] + 3, group * kvh, kvh, dim, bf16)
        out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
        status = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
        call(q, k, v, out, begin, bf16=bf16, window=window)(status.data_ptr())
        torch.cuda.synchronize()
        want, lim = formula(q, k, v, begin, window, tol=bf16)
        assert not status.any() and (out[:7] == 7).all() and (out[begin[-1]:] == 7).all()
        assert ((out.double() - want).abs() <= lim)[7:begin[-1]].all()


@pytest.mark.parametrize("bf16", [True, False])
def test_weights_too_small_for_fp32(cuda_ok, bf16):
    """A value of 1e38 behind a weight below 2^-126 of the row's largest: it counts as 0."""
    q, k = torch.zeros(2, 1, 32), torch.zeros(2, 1, 32)
    v = torch.ones(2, 1, 32)
    q[1, 0, 0], k[1, 0, 0], v[0, 0] = 1.0, 95 * 32 ** 0.5, 1e38  # scores of 0 and 95: a weight of 2^-137
    kind = torch.bfloat16 if bf16 else torch.float32
    q, k, v = (x.to(kind).cuda() for x in (q, k, v))
    out = torch.zeros_like(q)
    call(q, k, v, out, [0, 2], bf16=bf16)()
    torch.cuda.synchronize()
    assert (out[0] == v[0]).all() and ((out[1] - 1).abs() <= 2.0 ** -20).all()
