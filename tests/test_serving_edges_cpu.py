"""Refusals of the serving rows at the C boundary that test_serving_cpu does not
reach: extents past 32 bits and outputs over their inputs; and what the kernels'
source must hold to where no run can show it."""

import glob
import os
import re

import pytest

from conftest import ROOT
from test_serving_cpu import ROPE, call, rope


@pytest.mark.parametrize("geom", [rope(block_size=2**31), rope(block_size=2**32), rope(num_blocks=2**31), rope(num_blocks=-1)])
def test_rope_append_refuses_cache_extents_past_32_bits(geom):
    """A slot is divided by the block size in 32 bits: 2**32 places would have been none."""
    got, msg = call("nb2_rope_append", geom, *ROPE)
    assert got == -1 and "cache" in msg


def test_tensor_memory_loads_wait_in_their_own_statement():
    """Registers of a tcgen05.ld may be used only after its wait; between two statements the compiler may use them."""
    seen = 0
    for path in glob.glob(os.path.join(ROOT, "nert_b200", "csrc", "**", "*.cu*"), recursive=True):
        with open(path) as f:
            for statement in re.findall(r"\basm\b.*?;\s*\n", f.read().replace(';\\n', ' '), re.S):
                if "tcgen05.ld." in statement:
                    seen += 1
                    assert "tcgen05.wait::ld" in statement, f"{os.path.basename(path)}: {statement}"
    assert seen >= 4
