"""What the sources of the 8-bit product and of the attention over packed prompts must keep that no run would show."""
import re

import pytest

from phonon_b200._libs import CSRC


@pytest.mark.parametrize("name", ["phonon_i8.cuh", "phonon_prompt.cuh"])
def test_rows_scales_and_tables_are_not_read_as_constants(name):
    """Every kernel here is launched before the one ahead of it has ended, and reads what that may still write."""
    code = re.sub(r"//.*", "", (CSRC / name).read_text())
    kernels = re.split(r"__global__", code)[1:]
    assert kernels and all("pdl_wait();" in k for k in kernels)
    assert "__ldg" not in code and "ld.global.nc" not in code and "__restrict__" not in code
    # and nothing is read ahead of the wait: no operand but the kernel's own parameters' addresses is named before it
    for k in kernels:
        ahead = k[k.index(") {") + 3:k.index("pdl_wait();")]
        ahead = ahead.replace("cp.async.bulk.prefetch.L2.global", "")  # a hint: what is written after it is found all the same
        assert "tma_load" not in ahead and "cp.async" not in ahead and not re.search(r"\bp\.(x|w|k|v|q|begin|x_scales|w_scales|bias)\[", ahead)


def test_no_load_goes_to_several_ctas():
    for name in ("phonon_i8.cuh", "phonon_prompt.cuh"):
        code = re.sub(r"//.*", "", (CSRC / name).read_text())
        for text in re.findall(r'"(cp\.async\.bulk[^"]*)"', code):
            assert "multicast" not in text


@pytest.mark.parametrize("name", ["phonon_i8.cuh", "phonon_prompt.cuh"])
def test_the_next_launch_starts_when_tensor_memory_is_held(name):
    """A launch that starts early waits for the end of the one ahead, with tensor memory of its own in hand: a CTA of the one
    ahead that still had to get its own could wait for it in turn, for good."""
    code = re.sub(r"//.*", "", (CSRC / name).read_text())
    for k in re.split(r"__global__", code)[1:]:
        if "tcgen05.alloc" in k:
            assert k.count("pdl_trigger();") == 1
            between = k[k.index("tcgen05.alloc"):k.index("pdl_trigger();")]
            assert "\n    }" not in between or "__syncthreads();" in between  # the same warp's, or behind a barrier
