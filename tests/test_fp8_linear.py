"""The e4m3 product: what its kernels wait on."""
import os
import re

from conftest import PKG


# ---------------------------------------------------------------------------------------------------- waits have an end
def gemm_source():
    with open(os.path.join(PKG, "csrc", "edb200_fp8_gemm.cu")) as fh:
        return re.sub(r"//[^\n]*", "", fh.read())


def test_no_barrier_among_some_of_the_warps():
    """A warp whose wait has given up goes to the end of the kernel.  Others may have seen the same phase complete: a barrier
    among them without a limit would wait for that warp for good.  So between set-up and teardown, where every
    thread arrives, there is none; mbarrier waits have a limit."""
    assert not re.search(r"named_bar_sync|bar\.sync|barrier\.sync|barrier\.cta", gemm_source())
