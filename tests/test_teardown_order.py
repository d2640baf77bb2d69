"""The end of the tensor-core kernels, read from their sources: after a wait that ran out, MMAs and copies that are still in flight
are given time to land before the tensor memory that they write is freed (another CTA of the SM may get it at once)."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "deplodock_b200" / "csrc"


def _kernels():
    for path in sorted(CSRC.glob("*.cu")):
        parts = re.split(r"^(?=__global__|extern \"C\")", path.read_text(), flags=re.M)
        for part in parts:
            if part.startswith("__global__") and re.search(r"\btmem_dealloc(_pair)?\(", part):
                yield pytest.param(part, id=re.search(r"(\w+_kernel)\(", part).group(1))


@pytest.mark.parametrize("kernel", list(_kernels()))
def test_tensor_memory_is_freed_after_the_drain(kernel):
    free = re.search(r"\btmem_dealloc(_pair)?\(", kernel).start()
    drain = kernel.find("abort_drain()")
    assert 0 <= drain < free
