"""A property of the kernels' sources that no run can show reliably."""

import os
import re

import pytest

import flaggems_vllm_b200


@pytest.mark.parametrize("name", ["rms_norm.cu", "balance.cu"])
def test_inputs_of_kernels_that_start_early_are_not_read_only(name):
    """A kernel launched before its predecessor has ended may not declare what that one writes constant for its own life
    (const __restrict__): such loads need not stay behind the wait."""
    with open(os.path.join(os.path.dirname(flaggems_vllm_b200.__file__), "csrc", name)) as fh:
        source = fh.read()
    assert "pdl_wait" in source and not re.search(r"const\s+\w+\s*\*\s*__restrict__|__ldg\(|ld\.global\.nc", source)
