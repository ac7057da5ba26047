"""Two rules of synchronisation that no run can be relied on to show broken, read from the 8-bit cache's kernel sources."""
import os
import re

import strix_halo_maxx_b200 as pkg


def _kernel(name, file):
    """The source of one kernel, comments taken out."""
    src = open(os.path.join(os.path.dirname(pkg.__file__), "csrc", file)).read()
    src = re.sub(r"//[^\n]*", "", src)
    body = src[src.index(f" {name}("):]
    return body[:body.index("\n}\n")]


def test_no_store_into_another_cta_before_its_cluster_has_started():
    """Another CTA's shared memory may be written only after a cluster barrier has shown that the CTA runs; and the barrier is
    one for whole warps, so that a branch of single threads before it has to be joined."""
    k = _kernel("__launch_bounds__(THREADS) kv8_select_kernel", "kv8.cu")
    assert 0 <= k.find("cluster_sync();") < k.index("mapa_shared(")
    for m in re.finditer(r"st\.shared::cluster", k):
        rest = k[m.end():]
        assert "__syncwarp();" in rest[:rest.index("cluster_sync();")]


def test_a_warp_group_changes_its_registers_at_one_instruction():
    """setmaxnreg is one instruction for all four warps of a group, so no branch that leads to one may part a group."""
    k = _kernel("attn_kv8_tc_kernel", "kv8_tc.cu")
    uses = [m.start() for m in re.finditer(r"set_regs_(up|down)<", k)]
    assert len(uses) == 3
    for at in uses:
        assert int(re.findall(r"if \(warp >= (\d+)\)", k[:at])[-1]) % 4 == 0
