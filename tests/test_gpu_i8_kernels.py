"""Every kernel that the 8-bit product chooses among, at sizes that choose it, against the formula in 64 bits and beside one
another."""
import numpy as np
import pytest

from launches import launches
from phonon_b200 import runtime as rt
from test_gpu_i8 import check_product, product_case, product_want

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROWS, WIDE, SPLIT = "i8_rows_kernelILi%dE", "i8_product_kernelILi%dE", "i8_split_kernelILi%dE"
SIZES = [  # the kernel, and rows x channels x depth with parts of tiles, odd rows and depths among them
    (ROWS % 1, (7, 5003, 528)), (ROWS % 2, (1, 1003, 528)), (ROWS % 2, (13, 515, 1040)), (ROWS % 4, (31, 130, 400)),
    (WIDE % 64, (333, 1001, 272)), (WIDE % 128, (2049, 4100, 640)), ("i8_pair_kernel", (1030, 5003, 2064)),
    (SPLIT % 64, (127, 129, 2048)), (SPLIT % 64, (40, 513, 2064)),
    (SPLIT % 128, (32, 4096, 4096)), (SPLIT % 128, (100, 2501, 3088)), (SPLIT % 128, (40, 4099, 4112)), (SPLIT % 128, (200, 2047, 4080)),
]


@pytest.mark.parametrize("bf16,with_bias", [(False, True), (True, False)])
@pytest.mark.parametrize("pad", [0, 1, 4])
@pytest.mark.parametrize("kernel,size", SIZES)
def test_each_kernel_against_the_formula(cuda_ok, kernel, size, pad, bf16, with_bias):
    rows, channels, depth = size
    rng = np.random.default_rng(rows + channels + depth)
    x, w, xs, ws = product_case(rng, rows, channels, depth, full=True)
    bias = torch.tensor(rng.standard_normal(channels), dtype=torch.float32, device="cuda") if with_bias else None
    y = torch.full((rows + 2, channels + pad), 7.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    status = torch.zeros(rows, dtype=torch.int32, device="cuda")
    call = rt.I8Product(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, channels, depth,
                        rt.ROWS_BF16 if bf16 else rt.ROWS_F32, None if bias is None else bias.data_ptr(), y_stride=channels + pad)
    names = launches(lambda stream: call(status.data_ptr(), stream))
    assert len(names) == 1 and kernel in names[0][0], names
    assert not status.any() and (y[rows:] == 7).all() and (y[:, channels:] == 7).all()
    check_product(y[:rows, :channels], *product_want(x, w, xs, ws, bias), bf16)


def test_all_of_them_at_the_same_time(cuda_ok):
    """Each kernel on three streams at once, in other orders, again and again: what each gives alone, bit for bit."""
    rng = np.random.default_rng(13)
    streams = [torch.cuda.Stream() for _ in range(3)]
    jobs, seen = [], set()
    for kernel, (rows, channels, depth) in SIZES:
        x, w, xs, ws = product_case(rng, rows, channels, depth)
        outs = [torch.empty(rows, channels, dtype=torch.bfloat16, device="cuda") for _ in range(len(streams) + 1)]
        calls = [rt.I8Product(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data_ptr(), rows, channels, depth, rt.ROWS_BF16)
                 for y in outs]
        seen.update(name for name, _ in launches(lambda stream, c=calls[-1]: c(stream_ptr=stream)))
        jobs.append((x, w, xs, ws, outs, calls))
    assert len(seen) == 8
    for x, w, xs, ws, outs, _ in jobs:
        check_product(outs[-1], *product_want(x, w, xs, ws, None), True)
    torch.cuda.synchronize()
    for turn in range(6):
        for i, s in enumerate(streams):
            for j in range(len(jobs)):
                jobs[(j * (1, 5, 7)[i] + turn) % len(jobs)][-1][i](stream_ptr=s.cuda_stream)
    torch.cuda.synchronize()
    for *_, outs, _ in jobs:
        for y in outs[:-1]:
            assert torch.equal(y, outs[-1])
