"""Where a kernel's warps have to be whole again, and from where on the next launch may start. CPU only: what follows where
that is not kept is undefined or a wait for good, so no run is asked."""
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


def test_no_kernel_lets_the_next_launch_start_before_it_holds_its_tensor_memory():
    """The next launch waits for this one's end, and may hold tensor memory by then: CTAs of this one that still had to get
    theirs would wait for it in turn, for good. A kernel that does it all the same states, where it is compiled, that its CTAs
    have all registers of an SM (which the host checks before the launch), so that no other CTA is beside one."""
    found = 0
    for path in sorted(CSRC.glob("*.cuh")):
        code = re.sub(r"//.*", "", path.read_text())
        for kernel in re.split(r"__global__", code)[1:]:
            if "tcgen05.alloc" not in kernel or "pdl_trigger();" not in kernel:
                continue
            found += 1
            ahead = kernel[:kernel.index("pdl_trigger();")]
            assert "tcgen05.alloc" in ahead or re.search(r"static_assert\(k\w+Registers == 64 \* 1024,", ahead), path.name
    assert found >= 8


def test_a_bounded_wait_for_the_last_commits_begins_when_the_work_is_over():
    """The second CTA of a pair waits for the commits of the first before it gives its memory back. That wait is bounded by two
    seconds, which a large product may take itself: it begins behind the barrier that all warps come to with their work done."""
    code = re.sub(r"//.*", "", (CSRC / "phonon_i8.cuh").read_text())
    kernel = code[code.index("i8_pair_kernel("):]
    over = kernel.rindex("__syncthreads();")
    settle = [m.start() for m in re.finditer(r"mbar_settle\(idle, 0\);", kernel)]
    assert len(settle) == 2
    ahead, behind = kernel[:settle[0]], kernel[over:settle[1]]
    assert ahead.rstrip().endswith("commit(idle);") and settle[1] > over and "rank != 0" in behind
