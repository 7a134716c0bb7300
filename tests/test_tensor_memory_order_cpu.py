"""Order of tensor memory and early launches in the sources of the kernels that use both."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "ssd_b200" / "csrc"


def _kernels():
    for path in sorted(CSRC.glob("*.cuh")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        starts = [m.start() for m in re.finditer(r"__global__", text)] + [len(text)]
        for a, b in zip(starts, starts[1:]):
            body = text[a:b]
            if re.search(r"tmem_alloc(_pair)?\(", body) and "pdl_launch_dependents()" in body:
                yield pytest.param(body, id=re.search(r"\b(\w+_kernel)\(", body).group(1))


@pytest.mark.parametrize("body", list(_kernels()))
def test_tensor_memory_is_held_before_the_next_kernel_may_start(body):
    """A grid's successor may be scheduled as soon as every block has had a thread ask for it.  Its blocks take tensor memory and wait for this grid, so every block
    of this one has its own by then: between the allocation and the request lies a barrier of the block."""
    alloc, ask = re.search(r"tmem_alloc(_pair)?\(", body).start(), body.index("pdl_launch_dependents()")
    barrier = re.search(r"__syncthreads\(\)|cluster_sync_all\(\)", body[alloc:])
    assert barrier and alloc + barrier.start() < ask


def test_kernels_are_found():
    assert len(list(_kernels())) >= 4
