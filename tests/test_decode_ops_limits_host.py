"""Refusals of the decode-step operators that need no GPU."""
import pytest

from electrock_infer_b200 import _lib


@pytest.mark.parametrize("splits", [-1, 0, 65, 1000, 2 ** 31 - 1])
def test_no_scratch_for_numbers_of_splits_that_are_refused(splits):
    lib = _lib.load()
    assert lib.b200moe_paged_attn_fp8_workspace_bytes(200, 32, 8, splits) == 0
    assert lib.b200moe_paged_attn_fp8_workspace_bytes(200, 32, 8, 64) > 0
