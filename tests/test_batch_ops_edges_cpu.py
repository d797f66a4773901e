"""Edges of the batched-decoding operators' arguments, without a GPU."""
import pytest

from managedllama2_b200 import _lib
from test_batch_ops_cpu import ATTN, call, calls, refused  # noqa: F401  (calls is a fixture)


@pytest.mark.parametrize("scale", [3e38, -2.4e38])
def test_prefix_attention_refuses_a_scale_that_overflows_in_powers_of_two(calls, scale):  # noqa: F811
    lib, ctx, _ = calls
    refused(lib, call(lib.ml2_prefix_attention, _lib.PREFIX_ATTENTION, dict(ATTN, ctx=ctx, scale=scale)), "scale")
