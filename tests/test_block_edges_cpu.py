"""Refusals of the block's operators that need no GPU, and that no test hides another."""
import ast
import collections
import glob
import os

import pytest

from test_block_cpu import attention, refused


@pytest.mark.parametrize("scale", [2.4e38, -3e38])
def test_scales_that_overflow_in_base_two(native_lib, scale):
    """scale x log2(e) is what the kernels multiply by."""
    refused(attention(native_lib, scale=scale), "scale is too large")


# test_gpu_block.py defines this name twice; what its first one tests is
# test_append_of_many_requests of test_gpu_block_edges.py.
HIDDEN = {"test_gpu_block.py": {"test_append_many_rows"}}


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(os.path.dirname(__file__), "test_*.py"))), ids=os.path.basename)
def test_no_name_is_defined_twice(path):
    """Python keeps the last definition of a name: an earlier test of it would never run."""
    with open(path) as f:
        body = ast.parse(f.read()).body
    for scope in [body] + [n.body for n in body if isinstance(n, ast.ClassDef)]:
        names = collections.Counter(n.name for n in scope if isinstance(n, (ast.FunctionDef, ast.ClassDef)))
        assert {n for n, times in names.items() if times > 1} <= HIDDEN.get(os.path.basename(path), set())
