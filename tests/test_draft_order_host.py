"""Rules of the drafted step's kernels that no run can show to hold, read off their sources."""
import re

from tests.test_kernel_order_host import SOURCES, closing, code, kernels


def source(name):
    return code(next(p for p in SOURCES if p.endswith("/" + name)))


def test_the_verification_stores_into_blocks_that_have_started():
    """The blocks of a cluster are placed together but do not start together: a store into another one's shared memory needs a barrier
    of the cluster first, and every block has to come to it, those without nodes too."""
    s = source("draft_verify.cu")
    remote = []
    for m in re.finditer(r"__device__ __forceinline__ [\w ]+?(\w+)\(", s):
        if "shared::cluster." in s[m.start():closing(s, s.index("{", closing(s, m.end() - 1)))]:
            remote.append(m.group(1))
    assert remote == ["put_remote"]
    (k,) = kernels(s)
    wait = k.find("cluster_wait();")
    assert 0 <= k.find("cluster_arrive();") < k.index("rv_grid_dep_wait()") < wait
    assert "return" not in k[:wait] and wait < k.index("put_remote") and wait < k.index("cluster_sync();")


def test_the_verifications_warps_come_to_a_barrier_whole():
    """An aligned barrier is undefined for a warp whose lanes come to it apart, and the compiler need not bring them together behind a
    branch: here the lanes that store a sum, and the one that writes the next token."""
    s = source("draft_verify.cu")
    assert len(re.findall(r"barrier\.cluster\.(?:arrive|wait)", s)) == 2
    for m in re.finditer(r"barrier\.cluster\.[\w.]*\.aligned", s):
        assert re.search(r"__syncwarp\(\);\s*asm volatile\(\"$", s[:m.start()])
