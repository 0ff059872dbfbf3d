"""Kernels that start beside the one before them (csrc/ptx.cuh, grid_wait_dependencies) read memory
that the earlier kernel is still writing when they begin, or that they write themselves (a result in
place of the residual).  ``__restrict__`` and ``__ldg`` promise that nobody writes it while the kernel
runs: the compiler may then move such a load above the wait.  So neither is used on it there."""
from __future__ import annotations

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ltx-2_b200", "csrc")


def _kernels():
    """(file, signature, body) of every __global__ function."""
    for f in sorted(os.listdir(CSRC)):
        if not f.endswith((".cu", ".cuh")):
            continue
        src = open(os.path.join(CSRC, f)).read()
        for m in re.finditer(r"__global__ void\b", src):
            brace = src.index(") {", m.start()) + 2
            depth, i = 0, brace
            while True:
                depth += {"{": 1, "}": -1}.get(src[i], 0)
                i += 1
                if depth == 0:
                    break
            yield f, src[m.start():brace], src[brace:i]


def test_dependent_kernels_promise_nothing_about_their_inputs():
    found = {}
    for f, signature, body in _kernels():
        if "grid_wait_dependencies()" not in body:
            continue
        found[re.search(r"(\w+)\(const", signature).group(1)] = True
        assert "__restrict__" not in signature, f"{f}: {signature}"
        # the bias is an input of the whole operator, complete before its first kernel
        for load in re.findall(r"__ldg\([^;]*;", body):
            assert "p.bias" in load, f"{f}: {load}"
    assert set(found) == {"col_sum_kernel", "splitk_reduce_kernel", "wgrad_reduce_kernel"}
