"""The order that csrc/launch.h asks of kernels that take tensor memory: dependents are released only behind a block barrier
that follows the allocation. Unmet, it shows as a hang of two kernels on one SM, so it is read off the sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jepa.cpp_b200", "csrc")


def kernels():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = f.read()
        starts = [m.start() for m in re.finditer("__global__", text)] + [len(text)]
        for a, b in zip(starts, starts[1:]):
            body = text[a:b]
            if "tcgen05.alloc" in body and "griddepcontrol.launch_dependents" in body:
                yield os.path.basename(path), re.search(r"\b(k_\w+)\s*\(", body).group(1), body


def test_the_kernels_are_found():
    assert {name for _, name, _ in kernels()} >= {"k_kv4_tiles", "k_attention_tc"} and len(list(kernels())) >= 5


@pytest.mark.parametrize("file,name,body", list(kernels()), ids=lambda x: x if len(x) < 40 else "")
def test_dependents_are_released_behind_the_allocation(file, name, body):
    alloc = body.index("tcgen05.alloc")
    for m in re.finditer("griddepcontrol.launch_dependents", body):
        assert alloc < m.start() and re.search(r"\b(__syncthreads|cta_sync)\(\);", body[alloc:m.start()]), f"{file}: {name}"
