"""CPU: the adapters' kernels.  Their roles are played by whole warps, which go on to instructions that want all lanes together (tensor
memory's loads, barriers of the block and of the cluster), and lanes that wait each for itself may leave the wait at different times.  No run
would show that but once in a great while, so the sources are held to it: every wait is the warp's vote."""
import os
import re

import pytest

from moe_gen_b200 import build as b

TEXT = re.sub(r"//[^\n]*", "", open(os.path.join(b.CSRC, "adapter.cu")).read())
KERNELS = {re.search(r"(\w+_kernel)\s*\(", part).group(1): part for part in re.split(r"(?=__global__)", TEXT)[1:]}


def test_which_kernels_wait():
    assert {k for k, body in KERNELS.items() if "mbar_init(" in body} == {"adapter_tile_kernel", "adapter_grad_kernel"}


@pytest.mark.parametrize("name", ("adapter_tile_kernel", "adapter_grad_kernel"))
def test_warps_wait_by_one_vote(name):
    body = KERNELS[name]
    assert "wait_warp(" in body and not re.search(r"\bmbar_(try_)?wait\(", body)


def test_few_rows_are_always_a_clusters():
    """The launch gives a row two to eight blocks, and the kernel has no other form."""
    launch = re.search(r"int launch_direct_as\(.*?\n}", TEXT, re.S).group(0)
    assert re.search(r"int cs = 8;\s*while \(cs > 2 &&", launch) and "cs > 1" not in KERNELS["adapter_direct_kernel"]
