"""The 64-bit definition of the 8-bit cache on its own, and the refusals of
the C entry points that need no device. CPU only."""
import ctypes as C

import numpy as np
import pytest

import kv8_model as model
from phonon_b200 import runtime as rt


@pytest.mark.parametrize("amax,e", [(0.0, -48), (127.0, 0), (np.nextafter(127.0, 128.0), 1), (63.5, -1), (1.0, -6),
                                    (1e-30, -48), (3e38, 64), (127.0 * 2.0 ** 64, 64)])
def test_exponent(amax, e):
    assert model.exponent(amax) == e


def test_error_of_a_block_that_fills_position_by_position():
    """Roundings at each rise of the scale sum to less than one unit of the last."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((16, 4, 32)) * 2.0 ** np.arange(16)[:, None, None]
    h = model.Held(4, 32)
    for row in x:
        h.append(row[None])
    unit = 2.0 ** h.exps[0][None, :, None]
    assert (np.abs(h.values() - x) < unit).all()
    assert (np.abs(h.codes) <= 127).all()


def test_attention_of_equal_keys_is_the_mean():
    v = np.arange(12.0).reshape(6, 1, 2)
    out, _ = model.attention(np.ones((2, 2, 2)), np.ones((6, 1, 2)), v, window=3)
    np.testing.assert_allclose(out[:, 0], [v[2:5, 0].mean(0), v[3:6, 0].mean(0)])
    out, _ = model.attention(np.ones((3, 1, 2)), np.ones((2, 1, 2)), v[:2])
    assert (out[0] == 0).all()


def test_null_handles_are_refused():
    L = rt.lib()
    h = C.c_void_p()
    b, r, q = rt.Kv8Batch(), rt.Kv8Rows(), rt.Kv8Query()
    assert L.phonon_cuda_kv8_create(None, C.byref(h)) == rt.INVALID
    assert L.phonon_cuda_kv8_append_device(None, 0, b, r, None, None) == rt.INVALID
    assert L.phonon_cuda_kv8_read_device(None, 0, b, r, None, None) == rt.INVALID
    assert L.phonon_cuda_kv8_attention_device(None, 0, b, q, None, None, None) == rt.INVALID
    assert L.phonon_cuda_kv8_workspace_create(None, C.byref(h)) == rt.INVALID
    assert L.phonon_cuda_kv8_bytes(None) == 0
    L.phonon_cuda_kv8_destroy(None)
    L.phonon_cuda_kv8_workspace_destroy(None)


@pytest.mark.parametrize("kw", [dict(kv_heads=0), dict(head_dim=48), dict(head_dim=256), dict(pool_pages=0),
                                dict(layers=0), dict(kv_heads=2000)])
def test_cache_shapes_are_refused(kw):
    with pytest.raises(rt.CudaError) as e:
        rt.Kv8Cache(**(dict(kv_heads=8, head_dim=64, pool_pages=4) | kw))
    assert e.value.status == rt.INVALID
