"""What the quantising pass, the 8-bit product and the attention over packed prompts refuse: arguments are checked before
anything is asked of a device, so this runs without one."""
import pytest

from phonon_b200 import runtime as rt

P = 1 << 20  # an address that nothing reads: every call here is refused, or has no rows


def status(f, *args, at=None, **kw):
    try:
        f(*args, **kw)(at)
    except rt.CudaError as e:
        return e.status
    return rt.OK


def quantize(x=P, q=P + 4096, s=P + 8192, rows=2, cols=32, type=rt.ROWS_F32, **kw):
    return status(rt.QuantizeRows, x, q, s, rows, cols, type, **kw)


def product(x=P, xs=P + 4096, w=P + 8192, ws=P + 4096, y=P + 12288, rows=2, channels=16, depth=32, type=rt.ROWS_F32, **kw):
    return status(rt.I8Product, x, xs, w, ws, y, rows, channels, depth, type, **kw)


def attention(q=P, k=P + 4096, v=P + 8192, out=P + 12288, begin=P, prompts=1, rows=4, max_rows=4, heads=2, kv_heads=1, head_dim=32, **kw):
    return status(rt.PromptAttention, q, k, v, out, begin, prompts, rows, max_rows, heads, kv_heads, head_dim, **kw)


@pytest.mark.parametrize("kw", [dict(x=None), dict(q=None), dict(s=None), dict(cols=0), dict(cols=24), dict(cols=(1 << 24) + 16),
                                dict(type=2), dict(x=P + 8), dict(q=P + 4104), dict(s=P + 8193), dict(at=P + 2), dict(q=P),
                                dict(x_stride=16), dict(x_stride=36), dict(q_stride=40), dict(q_stride=16), dict(rows=(1 << 30) + 1)])
def test_quantize(kw):
    assert quantize(**kw) == rt.INVALID and quantize(rows=0) == rt.OK


@pytest.mark.parametrize("kw", [dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(y=None), dict(channels=0),
                                dict(channels=(1 << 30) + 1), dict(depth=0), dict(depth=24), dict(depth=1 << 17), dict(type=3),
                                dict(x=P + 4), dict(w=P + 8200), dict(y=P + 12290), dict(xs=P + 4097), dict(ws=P + 4098),
                                dict(bias_ptr=P + 3), dict(at=P + 1), dict(y=P), dict(y=P + 8192), dict(x_stride=16), dict(x_stride=40),
                                dict(w_stride=24), dict(y_stride=15), dict(y_stride=(1 << 40) + 1), dict(rows=(1 << 30) + 1)])
def test_product(kw):
    assert product(**kw) == rt.INVALID and product(rows=0) == rt.OK


@pytest.mark.parametrize("kw", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(begin=None), dict(prompts=0),
                                dict(prompts=(1 << 24) + 1), dict(max_rows=0), dict(max_rows=(1 << 30) + 1), dict(heads=0),
                                dict(kv_heads=0), dict(heads=3, kv_heads=2), dict(heads=1 << 17), dict(head_dim=48),
                                dict(head_dim=256), dict(type=2), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=2e30),
                                dict(q=P + 8), dict(k=P + 4), dict(v=P + 2), dict(out=P + 12290), dict(begin=P + 2), dict(at=P + 1),
                                dict(q_stride=63), dict(q_stride=68), dict(k_stride=24), dict(v_stride=8), dict(out_stride=66),
                                dict(out=P, out_stride=128), dict(out=P + 4096), dict(out=P + 8192), dict(window=(1 << 30) + 1),
                                dict(rows=(1 << 30) + 1)])
def test_attention(kw):
    assert attention(**kw) == rt.INVALID and attention(rows=0) == rt.OK and attention(rows=0, out=P) == rt.OK


def test_more_prompts_than_a_call_takes():
    assert attention(prompts=(1 << 18) + 1) == rt.CAPACITY and attention(prompts=1 << 24) == rt.CAPACITY
