"""Kernels that run under the launch before them (``grid_dependency_wait``) may not promise the compiler that what they read
stays the same for the whole kernel: loads of a ``const __restrict__`` parameter need not stay behind the wait.  A source check;
it holds for every kernel of the package, whichever of its pointers the earlier launch writes."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "optimus_lm_b200", "csrc")


def closing(text, at, pair):
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == pair[0]) - (text[i] == pair[1])
        if depth == 0:
            return i
    raise ValueError("no closing " + pair[1])


def kernels(text):
    """(name, parameters, body) of every ``__global__`` function with a body."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__\s+void", text):
        at = m.end()
        while True:   # attributes with arguments of their own stand before the name
            head = re.compile(r"\s*(\w+)\s*\(").match(text, at)
            end = closing(text, head.end() - 1, "()")
            if not head.group(1).startswith("__"):
                break
            at = end + 1
        brace = re.compile(r"\s*\{").match(text, end + 1)
        if brace:
            yield head.group(1), text[head.end():end], text[brace.end() - 1:closing(text, brace.end() - 1, "{}") + 1]


def promises(text):
    return [(name, p.strip()) for name, params, body in kernels(text) if "grid_dependency_wait" in body
            for p in params.split(",") if "__restrict__" in p and "const " in p]


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.cu"))), ids=os.path.basename)
def test_no_promise_behind_a_wait(path):
    assert promises(open(path).read()) == []


def test_the_check_finds_what_it_looks_for():
    text = """template <int N> __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(f(1, N), 1)
    k(const T<N> t, const double* __restrict__ p, int* __restrict__ out) { if (N) { grid_dependency_wait(); } }
    __global__ void q(const double* __restrict__ p) { }"""
    assert promises(text) == [("k", "const double* __restrict__ p")]
    seen = {name for path in glob.glob(os.path.join(CSRC, "*.cu")) for name, _, body in kernels(open(path).read()) if "grid_dependency_wait" in body}
    assert {"gemm_bf16_kernel", "gemm_bf16_pair_kernel", "tail_sum_kernel", "lce_finish_kernel", "grad_scale_kernel"} <= seen
