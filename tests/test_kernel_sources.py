"""What the kernels' sources must keep that no run would show. CPU only."""
import re

import pytest

from phonon_b200._libs import CSRC


@pytest.mark.parametrize("name", ["phonon_kv8.cuh", "phonon_kv8_prompt.cuh", "phonon_qk.cuh"])
def test_rows_tables_and_pages_are_not_read_as_constants(name):
    """Kernels of these files are launched before the one ahead of them has ended, and read what it may still write: rows,
    lengths, page ids, scales, pages. Read-only loads take such data for constant from the grid's start on."""
    code = re.sub(r"//.*", "", (CSRC / name).read_text())
    assert "launch" not in code or "pdl_wait" in code
    assert "__ldg" not in code and "ld.global.nc" not in code and "__restrict__" not in code
