"""Refusals of the serving rows at the C boundary that test_serving_cpu does not
reach: extents past 32 bits and outputs over their inputs; and what the kernels'
source must hold to where no run can show it."""

import glob
import os
import re

import pytest

from conftest import ROOT
from test_serving_cpu import ATTN, ROPE, attn, call, rope


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


def test_the_python_module_guards_the_current_gpu():
    """Each function that Python calls restores the current GPU (with one GPU no run can show it)."""
    with open(os.path.join(ROOT, "nert_b200", "csrc", "torch", "serving_torch.cpp")) as f:
        source = f.read()
    functions = re.findall(r'm\.def\("\w+", &(\w+)\)', source)
    assert len(functions) == 6
    for name in functions:
        body = re.search(r"^[\w:<>, \n]*\b%s\([^{;]*\{\n(.*?)^\}" % name, source, re.S | re.M).group(1)
        assert "OnGpu guard(" in body and ("context(" not in body or body.index("OnGpu guard(") < body.index("context(")), name


ONES = [dict(tokens=1, q_stride=257, o_stride=3), dict(q_heads=1, kv_heads=1, q_head_stride=1, o_head_stride=7),
        dict(kv_heads=1, kc_head_stride=1, vc_head_stride=0), dict(num_blocks=1, kc_block_stride=5, vc_block_stride=1),
        dict(block_size=1, kc_place_stride=3, vc_place_stride=1)]


@pytest.mark.parametrize("one", ONES)
def test_tree_attention_takes_any_stride_of_a_dimension_of_one(one):
    """Past its checks the call asks for its device."""
    assert call("nb2_tree_attention", attn(**one), *ATTN) == (-1, "null device")
    two = {n: 2 for n in ("tokens", "q_heads", "kv_heads", "num_blocks", "block_size") if n in one}
    got, msg = call("nb2_tree_attention", attn(**(one | two)), *ATTN)
    assert got == -1 and "16 bytes" in msg


@pytest.mark.parametrize("q_out,k_out,geom,refused", [
    (1, 9, dict(qo_stride=128, qo_head_stride=64), True), (1, 9, dict(qo_stride=256, qo_head_stride=32), True),
    (9, 2, dict(ko_stride=64, ko_head_stride=64), True), (1, 2, dict(ko_head_stride=128), True), (1, 2, dict(), False),
    (9, 8, dict(qo_stride=128, ko_stride=64), False), (1, 2, dict(tokens=1, qo_stride=128, ko_stride=3), False)])
def test_rope_append_in_place_needs_equal_strides(q_out, k_out, geom, refused):
    """A thread reads both elements of a pair before it writes them, where they come from and go to the same places."""
    strides = dict(q_stride=256, q_head_stride=64, qo_stride=256, qo_head_stride=64, k_stride=128, k_head_stride=64,
                   ko_stride=128, ko_head_stride=64)
    at = 4096
    got, msg = call("nb2_rope_append", rope(**(strides | geom)), at, 2 * at, 3 * at, 4 * at, 5 * at, 6 * at, q_out * at, k_out * at,
                    11 * at, 12 * at)
    assert got == -1 and msg == ("RopeAppend: in place needs equal strides" if refused else "null device")


@pytest.mark.parametrize("geom,refused", [(dict(o_stride=512), True), (dict(o_head_stride=128), True), (dict(), False),
                                          (dict(tokens=1, o_stride=512), False)])
def test_tree_attention_in_place_needs_equal_strides(geom, refused):
    """A row is written when all that read its query have; with other strides it would lie over other rows' queries."""
    got, msg = call("nb2_tree_attention", attn(**geom), *ATTN)  # out is q there
    assert got == -1 and msg == ("TreeAttention: in place needs equal strides" if refused else "null device")
