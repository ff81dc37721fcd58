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
