"""The serving rows' refusals at the C boundary: what the host can see is checked
before anything touches a GPU, so these calls return a status and a message
without one."""

import ctypes

import pytest

from nert_b200 import _lib

FAKE = 0x1000  # an address that no call here gets to use


def call(fn, geom, *args):
    status = getattr(_lib.lib(), fn)(None, ctypes.byref(geom), *args)
    return status, _lib.lib().nb2_last_error().decode()


def plan(**kw):
    g = dict(batch=2, tokens=4, block_size=16, table_blocks=8, table_stride=8, free_blocks=4, mask_words=0) | kw
    return _lib.PagePlanGeom(**g)


PLAN = [FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, None, 5 * FAKE, 6 * FAKE, 7 * FAKE, 8 * FAKE, 9 * FAKE, 10 * FAKE, None]


@pytest.mark.parametrize("geom,word,status", [
    (plan(block_size=0), "block size", -1), (plan(tokens=-1), "extents", -1), (plan(table_stride=7), "overlap", -1),
    (plan(batch=8193), "8192", -4), (plan(mask_words=33), "1024", -4), (plan(mask_words=1), "parents", -1),
    (plan(free_blocks=2**31), "extents", -1)])
def test_page_plan_refusals(geom, word, status):
    got, msg = call("nb2_page_plan", geom, *PLAN)
    assert got == status and word in msg


def test_page_plan_refuses_aliases_and_null():
    args = list(PLAN)
    args[6] = args[0]  # new_total over seq_lens
    assert call("nb2_page_plan", plan(), *args) == (-1, "PagePlan: new_total may not be seq_lens")
    args = list(PLAN)
    args[8] = args[3]
    assert call("nb2_page_plan", plan(), *args) == (-1, "PagePlan: free_head_out may not be free_head")
    args = list(PLAN)
    args[9] = None
    assert call("nb2_page_plan", plan(), *args) == (-1, "PagePlan: null buffer")
    assert call("nb2_page_plan", plan(), *PLAN) == (-1, "null device")


def rope(**kw):
    g = dict(tokens=2, q_heads=4, kv_heads=2, head_dim=64, rot_dim=64, table_len=10, axes=1, dtype=_lib.BF16,
             block_size=16, num_blocks=4) | kw
    return _lib.RopeGeom(**g)


ROPE = [FAKE] * 10


@pytest.mark.parametrize("geom,word,status", [
    (rope(dtype=_lib.I64), "type", -1), (rope(head_dim=63), "even", -1), (rope(rot_dim=66), "within", -1),
    (rope(head_dim=514), "512", -4), (rope(axes=0), "axes", -1), (rope(table_len=0), "table", -1), (rope(q_heads=0), "heads", -1),
    (rope(axes=1, axis_of=(ctypes.c_uint8 * 256)(1)), "axis", -1), (rope(block_size=0), "cache", -1)])
def test_rope_append_refusals(geom, word, status):
    got, msg = call("nb2_rope_append", geom, *ROPE)
    assert got == status and word in msg


def test_rope_append_refuses_half_a_cache():
    args = list(ROPE)
    args[2] = None  # no v
    assert call("nb2_rope_append", rope(), *args)[1].endswith("come together")
    args = [FAKE, FAKE, None, FAKE, FAKE, None, FAKE, None, None, None]
    assert call("nb2_rope_append", rope(), *args)[1].endswith("nowhere to go")
    assert call("nb2_rope_append", rope(tokens=0), *args)[0] == 0  # nothing to do


def attn(**kw):
    g = dict(batch=1, tokens=2, q_heads=4, kv_heads=2, head_dim=64, max_new=2, q_stride=256, q_head_stride=64, o_stride=256,
             o_head_stride=64, block_size=16, num_blocks=4, table_blocks=4, table_stride=4, kc_block_stride=2048,
             kc_place_stride=128, kc_head_stride=64, vc_block_stride=2048, vc_place_stride=128, vc_head_stride=64,
             mask_words=1, scale=0.125, dtype=_lib.F16) | kw
    return _lib.TreeAttnGeom(**g)


ATTN = [FAKE] * 9


@pytest.mark.parametrize("geom,word,status", [
    (attn(q_heads=3), "multiple", -1), (attn(head_dim=60), "multiple of 8", -1), (attn(head_dim=264), "256", -4),
    (attn(batch=8193), "8192", -4), (attn(scale=float("nan")), "finite", -1), (attn(scale=float("inf")), "finite", -1),
    (attn(mask_words=0), "width", -1), (attn(q_stride=257), "16 bytes", -1), (attn(vc_place_stride=4), "16 bytes", -1),
    (attn(table_stride=3), "table", -1), (attn(max_new=-1), "bound", -1), (attn(block_size=0), "cache", -1),
    (attn(dtype=9), "type", -1)])
def test_tree_attention_refusals(geom, word, status):
    got, msg = call("nb2_tree_attention", geom, *ATTN)
    assert got == status and word in msg


def test_tree_attention_refuses_unaligned_buffers():
    args = list(ATTN)
    args[0] = FAKE + 2
    assert call("nb2_tree_attention", attn(), *args) == (-1, "TreeAttention: buffers must be 16-byte aligned")
    assert call("nb2_tree_attention", attn(tokens=0), *args)[0] == 0


def logits(**kw):
    g = dict(rows=2, vocab=100, requests=2, in_stride=100, out_stride=100, grammar_count=2, grammar_stride=4, prompt_count=3,
             output_count=3, bias_count=1, in_dtype=_lib.F32, out_dtype=_lib.F32) | kw
    return _lib.LogitsGeom(**g)


LOGITS = [FAKE, 2 * FAKE] + [FAKE] * 13


@pytest.mark.parametrize("geom,word,status", [
    (logits(in_dtype=_lib.BOOL), "types", -1), (logits(rows=-1), "extents", -1), (logits(grammar_stride=3), "too short", -1),
    (logits(out_stride=99), "overlap", -1), (logits(output_count=2**30), "2^30", -1)])
def test_logits_process_refusals(geom, word, status):
    got, msg = call("nb2_logits_process", geom, *LOGITS)
    assert got == status and word in msg


def test_logits_process_refuses_half_lists_and_mixed_places():
    args = list(LOGITS)
    args[4] = None  # prompt without offsets
    assert "offsets" in call("nb2_logits_process", logits(), *args)[1]
    args = list(LOGITS)
    args[11] = None  # bias without values
    assert "bias" in call("nb2_logits_process", logits(), *args)[1]
    args = list(LOGITS)
    args[1] = args[0]
    assert "in place" in call("nb2_logits_process", logits(out_dtype=_lib.F16), *args)[1]
    assert call("nb2_logits_process", logits(vocab=0, grammar_stride=0), *LOGITS)[0] == 0


def test_contexts_are_refused_where_they_cannot_be():
    L = _lib.lib()
    h = ctypes.c_void_p()
    assert L.nb2_device_on_stream(-1, None, ctypes.byref(h)) == -1 and "ordinal" in L.nb2_last_error().decode()
    assert L.nb2_device_on_stream(0, None, None) == -1
    assert L.nb2_device_release(None) == 0


def test_python_module_checks_before_the_library():
    import torch

    from nert_b200 import serving

    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        serving.page_plan(ints, ints, torch.zeros(2, 2, dtype=torch.int32), ints, 16, 1)
    with pytest.raises(ValueError, match="GPU"):
        serving.logits_process(torch.zeros(2, 5))
    assert serving.contiguous_axes((2, 0, 3)) == (0, 0, 2, 2, 2)
