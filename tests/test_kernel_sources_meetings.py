"""Where warps of the 8-bit product's kernels have to be whole again. CPU only: what follows from a warp that is not would be
undefined, so no run is asked."""
import re

from phonon_b200._libs import CSRC

WHOLE = ("__syncwarp();", "__syncthreads();")


def test_warps_are_whole_where_a_cluster_meets():
    """barrier.cluster's aligned forms want all of a warp's threads at once, which a loop with a `continue` or a branch ahead
    of them does not leave so by itself."""
    code = re.sub(r"//.*", "", (CSRC / "phonon_i8.cuh").read_text())
    lines = [x.strip() for x in code.splitlines() if x.strip()]
    meets = [i for i, x in enumerate(lines) if x == "cluster_meet();"]
    assert len(meets) >= 4
    assert all(lines[i - 1] in WHOLE for i in meets), [lines[i - 1] for i in meets]
