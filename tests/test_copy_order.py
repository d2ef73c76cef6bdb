"""Kernels whose first barrier waits for the copies of one stage and leaves later ones in flight count copies in the order of their
issue.  Nothing but issue_order_fence() keeps the compiler from issuing a later stage's copy first, and then the barrier lets a
stage be read before it is there; whether it does is a matter of scheduling, so the sources are held to the fence itself."""

import glob
import os
import re

import pytest

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-vulkan_amd", "csrc", "kernels")


def source(path):
    return re.sub(r"//[^\n]*", "", open(path).read())


def counting():
    """(file, body) of every kernel that uses a barrier which leaves accesses in flight (63: the field's limit, waits for none)."""
    for path in sorted(glob.glob(os.path.join(KERNELS, "*"))):
        if os.path.basename(path) == "lds_stage.h":  # the barriers themselves
            continue
        for body in source(path).split("__global__")[1:]:
            if re.search(r"barrier_keep_vm(_lds)?<(?!0>|63>)", body):
                yield os.path.basename(path), body


@pytest.mark.parametrize("name,body", [pytest.param(n, b, id=f"{n}-{i}") for i, (n, b) in enumerate(counting())])
def test_kernels_that_count_copies_fence_their_issue(name, body):
    assert "issue_order_fence();" in body, name


@pytest.mark.parametrize("name,first,later", [
    ("mx4_back.hip", "copy(std::integral_constant<int, 0>(), 0);", "copy(std::integral_constant<int, 1>(), 1);"),
    ("mx4_gemm.hip", "copy_x(0, xbuf(std::integral_constant<int, 0>()));", "copy_x(1, xbuf(std::integral_constant<int, 1>()));")])
def test_the_first_stage_is_issued_first(name, first, later):
    text = source(os.path.join(KERNELS, name))
    between = text[text.index(first):text.index(later)]
    assert text.count(first) == text.count(later) == 1 and "issue_order_fence();" in between
