"""Operands of one row, whose stride says nothing and may be any that the calls allow."""
import numpy as np
import pytest

from phonon_b200 import runtime as rt
from test_gpu_i8 import check_product, product_case, product_want

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

FAR = 1 << 40


@pytest.mark.parametrize("rows", [1, 12, 40, 300])
def test_one_channel(cuda_ok, rows):
    rng = np.random.default_rng(rows)
    x, w, xs, ws = product_case(rng, rows, 1, 528)
    y = torch.empty(rows, 1, device="cuda")
    rt.I8Product(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, 1, 528, x_stride=FAR if rows == 1 else 0,
                 w_stride=FAR)()
    torch.cuda.synchronize()
    check_product(y, *product_want(x, w, xs, ws, None), False)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_a_prompt_of_one_row(cuda_ok, dim, bf16):
    """It sees itself alone: out is v."""
    kind = torch.bfloat16 if bf16 else torch.float32
    rng = np.random.default_rng(dim)
    q, k, v = (torch.tensor(rng.standard_normal((1, h, dim)), dtype=torch.float32).to(kind).cuda() for h in (4, 2, 2))
    out = torch.zeros_like(q)
    begin = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    rt.PromptAttention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), begin.data_ptr(), 1, 1, 1, 4, 2, dim,
                       rt.ROWS_BF16 if bf16 else rt.ROWS_F32, q_stride=FAR, k_stride=FAR, v_stride=FAR, out_stride=FAR)()
    torch.cuda.synchronize()
    want = v.double().repeat_interleave(2, 1)
    # one weight of 1: a product and a quotient, each exact but for fp32's rounding of three slices (2^-22 in all)
    assert ((out.double() - want).abs() <= want.abs() * 2.0 ** -22).all()


def test_one_row_of_codes(cuda_ok):
    x = torch.randn(1, 272, device="cuda")
    q, s = torch.zeros(1, 272, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda")
    rt.QuantizeRows(x.data_ptr(), q.data_ptr(), s.data_ptr(), 1, 272, x_stride=FAR, q_stride=FAR)()
    torch.cuda.synchronize()
    assert q.abs().max().item() == 127 and s.item() > 0
