"""The host's rules on status words (csrc/phonon_status.h), compiled as C. CPU only."""
import ctypes as C
import subprocess

import numpy as np
import pytest

from phonon_b200 import runtime as rt
from phonon_b200._libs import CSRC, INCLUDE


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    at = tmp_path_factory.mktemp("status")
    (at / "rule.c").write_text('#include "phonon_status.h"\n'
                               "int rule(const int32_t *status, int rows) { return phonon_rows_status(status, rows); }\n")
    subprocess.run(["gcc", "-std=c17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", f"-I{INCLUDE}",
                    "-o", str(at / "rule.so"), str(at / "rule.c")], check=True)
    fn = C.CDLL(str(at / "rule.so")).rule

    def call(status):
        words = np.array(status, np.int32)
        return fn(words.ctypes.data_as(C.c_void_p), len(words))

    return call


@pytest.mark.parametrize("status,result", [
    ([], rt.OK), ([0, 0, 0], rt.OK), ([0, rt.NON_FINITE, 0], rt.NON_FINITE), ([rt.DEVICE_ERROR], rt.DEVICE_ERROR),
    ([0, rt.NON_FINITE, rt.DEVICE_ERROR, rt.NON_FINITE], rt.DEVICE_ERROR), ([rt.DEVICE_ERROR, 0], rt.DEVICE_ERROR),
])
def test_an_expired_wait_is_not_a_non_finite_row(rule, status, result):
    """A prefill whose attention gave up a wait reports that, whatever its rows then hold."""
    assert rule(status) == result
