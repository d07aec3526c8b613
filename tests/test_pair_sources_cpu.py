"""CPU: the kernels on pairs of SMs.  The leader's commits arrive in the shared memory of both CTAs; a CTA that left before the last of
them would hand its memory on with arrivals under way, which no run would show but once in a great while.  So the sources are held
to it: what a commit signals is waited for by an epilogue, or drained by the role that fills the slots."""
import os
import re

import pytest

from moe_gen_b200 import build as b

# complete accumulators: every one is waited for by the epilogue that reads it
WAITED_FOR = {"dfull", "tfull"}


def _kernels():
    out = {}
    for f in b.SOURCES:
        text = re.sub(r"//[^\n]*", "", open(os.path.join(b.CSRC, f)).read())
        for part in re.split(r"(?=__global__)", text)[1:]:
            name = re.search(r"(\w+_kernel)\s*\(", part)
            if name and "tc_commit_pair(" in part:
                out[name.group(1)] = part
    return out


KERNELS = _kernels()


def test_there_are_such_kernels():
    assert set(KERNELS) == {"grouped_gemm_wl_kernel", "grouped_gemm2_kernel"}


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_every_release_by_a_pairs_commit_is_drained(name):
    body = KERNELS[name]
    signalled = set(re.findall(r"tc_commit_pair\(smem_u32\(&(\w+)\[", body))
    drained = set(re.findall(r"drain_slots\((\w+)", body))
    assert len(signalled) >= 3 and signalled - WAITED_FOR == drained
    for bar in signalled & WAITED_FOR:
        assert re.search(rf"wait\w*\(smem_u32\(&{bar}\[", body)
    # behind the drains, the CTAs meet before either leaves
    assert body.rindex("drain_slots(") < body.rindex("cluster_sync_all()") < body.rindex("tcgen05.dealloc")
