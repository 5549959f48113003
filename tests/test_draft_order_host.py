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
