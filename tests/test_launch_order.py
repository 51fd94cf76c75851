"""Kernels that may start before the stream's kernel before them has ended (CPU: their source).

Such a kernel is shown what that one wrote, and what that one had waited for, only by its own
griddepcontrol.wait: every thread has to make it before it reads anything.
"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dsa_triton_ascend_b200", "csrc")


def kernels(name):
    """(name, body) of each __global__ function of a file."""
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    for m in re.finditer(r"__global__ void(?: __\w+__\([^)]*\))*\s+(\w+)\(", text):
        at, depth = text.index(") {", m.end()) + 2, 0
        for end in range(at, len(text)):
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            if depth == 0:
                break
        yield m.group(1), text[at + 1:end]


@pytest.mark.parametrize("name,count", [("attn_paged_heads.cuh", 1), ("attn_paged_pair.cuh", 1), ("attn_paged_wide.cuh", 1),
                                        ("attn_paged_join.cuh", 1), ("attn_shared.cu", 2), ("batch_plan.cu", 4)])
def test_nothing_is_read_before_the_wait(name, count):
    found = list(kernels(name))
    assert len(found) == count
    for kernel, body in found:
        waits = list(re.finditer(r"^  griddep_wait\(\);", body, re.M))   # on no condition
        assert len(waits) == 1, kernel
        before = re.sub(r"//[^\n]*", "", body[:waits[0].start()])
        # neither a call of what reads the inputs nor an argument with an index
        assert not re.search(r"\b(share_of|plan_\w+|request_of|\w+_seen|token_keys|row_keys)\b", before), kernel
        assert not re.search(r"\b[ap]\.\w+(\.\w+)?\[", before), kernel
        # a kernel that ends early waits as well, as its end stands for that of the one before it
        for part in re.findall(r"\{([^{}]*)\breturn;", before):
            assert "griddep_wait();" in part, kernel


@pytest.mark.parametrize("name", ["attn_paged_heads.cuh", "attn_paged_pair.cuh", "attn_paged_wide.cuh"])
def test_the_next_kernel_starts_behind_the_tensor_memory(name):
    """A kernel that waits for this one with tensor memory of its own must not have taken it first.  (With
    Args the next one is a join, which takes none.)"""
    (_, body), = kernels(name)
    alloc, barrier = body.index("tmem_alloc<"), body.index("__syncthreads();")
    assert alloc < barrier < body.index("release_next<true>(a);") and "griddep_launch_dependents" not in body
    with open(os.path.join(CSRC, "attn_paged.cuh")) as f:
        text = f.read()
    items = re.search(r"release_next\(const ItemArgs&\) \{([^}]*)\}", text).group(1)
    assert items.strip() == "if (kBehind) griddep_launch_dependents();"
