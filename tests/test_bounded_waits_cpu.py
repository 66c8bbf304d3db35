"""Kernels with bounded waits: what happens after one has run out, read from their sources."""

import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tt-mlir_b200", "csrc")


def kernels():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(path) as f:
            for part in f.read().split("__global__")[1:]:
                if "mbarWait(" in part and "tcgen05.dealloc" in part:
                    yield os.path.basename(path), re.search(r"(\w+Kernel)\(", part).group(1), part


@pytest.mark.parametrize("name,part", [pytest.param(k, p, id=f"{f}:{k}") for f, k, p in kernels()])
def test_an_aborted_kernel_lets_its_copies_land_before_it_gives_its_memory_back(name, part):
    """A wait that runs out leaves bulk copies and products in flight; shared and tensor memory must outlive them."""
    release = part.index("tcgen05.dealloc")
    tail = part[part.rindex("mbarWait(", 0, release):release]
    barrier = tail.rindex("__syncthreads()")
    assert "drainAborted(" in tail[:barrier] or "if (*abortFlag)" in tail[:barrier], name


def test_all_tensor_core_kernels_are_looked_at():
    assert {k for _, k, _ in kernels()} >= {"sdpaTcgen05Kernel", "sdpaTcgen05PairKernel", "sdpaWindowTcgen05Kernel", "sdpaCachedTcgen05Kernel"}
