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
