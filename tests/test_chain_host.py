"""Kernels that may start before the one in front of them has finished (chain_begin) read what it wrote only with
ordinary loads.  A load through the read-only path (__ldg, or a parameter that is const and __restrict__) says that
the memory does not change while the kernel runs, which is false before the wait: compiler and hardware may then
take it from before the wait.  Checked in the source text."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "knet.jl_b200", "csrc")


def text(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def kernels(src):
    """(head, body) of every __global__ function"""
    for m in re.finditer(r"__global__", src):
        at = src.index("{", m.end())
        depth, k = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(src[k], 0)
            k += 1
        yield src[m.start():at], src[at:k]


def chained():
    found = []
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh")):
            for head, body in kernels(text(name)):
                if "chain_begin()" in body:
                    found.append((name, re.findall(r"(\w+)\s*\(", head)[-1], head, body))
    return found


def test_there_are_chained_kernels():
    assert len(chained()) >= 15


@pytest.mark.parametrize("kernel", chained(), ids=lambda k: k[1])
def test_chained_kernels_declare_no_read_only_memory(kernel):
    name, fn, head, body = kernel
    assert "__restrict__" not in head and "__ldg" not in body


@pytest.mark.parametrize("name", ["linear_nll.cu", "linear_nll.cuh", "linear_nll_mma.cuh", "linear_nll_small.cuh"])
def test_functions_of_chained_kernels(name):
    """All kernels of these files are chained, so the functions they share keep to the same loads."""
    assert "__ldg" not in text(name) and "__restrict__" not in text(name)


def test_the_updates_device_scalars():
    src = text("optim.cu")
    at = src.index("AdamF<T> resolve(const AdamDevF<T>& d)")
    assert "__ldg" not in src[at:src.index("}", at)]


def test_launches_that_may_start_early_are_of_chained_kernels():
    """launch_chained only with kernels that wait."""
    ok = {k[1] for k in chained()}
    for name in sorted(os.listdir(CSRC)):
        if name.endswith(".cu"):
            for m in re.finditer(r"launch_chained(?:_cluster\(\w+,|\()\s*(\w+)", text(name)):
                assert m.group(1) in ok, (name, m.group(1))
