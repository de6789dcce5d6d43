"""Refusals of the serving rows at the C boundary that test_serving_cpu does not
reach: extents past 32 bits and outputs over their inputs."""

import pytest

from test_serving_cpu import ROPE, call, rope


@pytest.mark.parametrize("geom", [rope(block_size=2**31), rope(block_size=2**32), rope(num_blocks=2**31), rope(num_blocks=-1)])
def test_rope_append_refuses_cache_extents_past_32_bits(geom):
    """A slot is divided by the block size in 32 bits: 2**32 places would have been none."""
    got, msg = call("nb2_rope_append", geom, *ROPE)
    assert got == -1 and "cache" in msg
