"""Serving rows over torch CUDA tensors: one step of a server over a paged cache.

``page_plan`` once a step, then ``rope_append`` and ``tree_attention`` for each
layer, and ``logits_process`` before picking tokens. torch provides memory and
the stream; every computation is a kernel of libnert_b200.so.

Unlike the wrappers of ``nert_b200.ops``, these launch on torch's current
stream (through one context a stream, made on first use) and return without
synchronising, so a step can be queued, overlapped or captured in a CUDA graph
(after one uncaptured call, which sizes the workspace). Arguments that the host
can see are checked before the launch (``ValueError``, or ``NB2Error`` from the
library); values on the device (lengths, blocks, slots, token ids) are checked
by the kernels, and ``synchronize()`` raises what they recorded.

Metadata tensors are contiguous int32; masks are int32 words of 32 bits.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check, lib

MAX_FREQ = 256

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_contexts: dict[tuple[int, int], int] = {}


def context(device: torch.device | None = None) -> int:
    """The library's context for torch's current stream on the device."""
    stream = torch.cuda.current_stream(device)
    key = (stream.device_index, stream.cuda_stream)
    dev = _contexts.get(key)
    if dev is None:
        h = _lib.vp()
        check(lib().nb2_device_on_stream(key[0], key[1] or None, ctypes.byref(h)))
        dev = _contexts[key] = h.value
    return dev


def synchronize(device: torch.device | None = None) -> None:
    """Waits for torch's current stream; raises what the kernels of this module
    recorded on it (NB2Error with status ERR_DEVICE)."""
    check(lib().nb2_device_synchronize(context(device)))


def _need(ok, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _ints(t, name: str, dim: int = 1) -> int:
    """Address of a contiguous int32 CUDA tensor (None passes)."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.dim() != dim or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous {dim}-d int32 CUDA tensor")
    return t.data_ptr()


def _floats(t, name: str, n: int) -> int:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.shape != (n,) or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name}: expected {n} contiguous float32 values on the GPU")
    return t.data_ptr()


def _heads(t, name: str, tokens: int, dtype, dim: int):
    if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != dim or t.dtype != dtype or not t.is_cuda:
        raise ValueError(f"{name}: expected [{tokens}, heads, {dim}] {dtype} on the GPU")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: a head's elements must be contiguous")
    return t


def _caches(k_cache, v_cache, dtype, kv_heads: int, dim: int):
    for c, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if c.dim() != 4 or c.shape[2] != kv_heads or c.shape[3] != dim or c.dtype != dtype or not c.is_cuda:
            raise ValueError(f"{name}: expected [blocks, block_size, {kv_heads}, {dim}] {dtype} on the GPU")
        if c.stride(3) != 1:
            raise ValueError(f"{name}: a head's elements must be contiguous")
    _need(k_cache.shape == v_cache.shape, "k_cache and v_cache differ in shape")


class PagePlan(NamedTuple):
    """What a step's rows read. ``tree_mask`` is None for chains."""

    seq_lens: torch.Tensor  # [batch] places of each request, the new ones included
    token_offsets: torch.Tensor  # [batch + 1] first new token of each request
    slots: torch.Tensor  # [tokens] cache slot of each new token, -1 where it has none
    positions: torch.Tensor  # [tokens] cached tokens + depth among the new ones
    tree_mask: torch.Tensor | None  # [tokens, words] the new tokens that each sees
    free_head: torch.Tensor  # [1] first free block not taken


def page_plan(seq_lens, new_lens, block_table, free_blocks, block_size: int, tokens: int, parents=None,
              mask_words: int = 0, free_head=None) -> PagePlan:
    """Block tables, slots, positions and tree masks from the request lengths.

    Request r has ``seq_lens[r]`` cached tokens and adds ``new_lens[r]``; the
    blocks it needs are taken in request order from ``free_blocks`` from
    ``free_head`` (default 0) on and written to ``block_table`` [batch, blocks],
    in place. ``tokens`` is the size of the per-token outputs: at least the sum
    of new_lens, and the tail is padding (slot -1). ``parents`` [tokens] gives a
    drafted token's parent among its request's new tokens (-1: child of the
    cached text); then ``mask_words`` is ceil(most new tokens of a request / 32).
    """
    batch = seq_lens.shape[0]
    dev = context(seq_lens.device)
    _need(block_table.dim() == 2 and block_table.shape[0] == batch and block_table.dtype == torch.int32
          and block_table.is_cuda and (block_table.stride(1) == 1 or block_table.shape[1] <= 1),
          "block_table: expected [batch, blocks] int32 on the GPU")
    _need(new_lens.shape == seq_lens.shape, "new_lens and seq_lens differ in length")
    _need(parents is None or parents.shape[0] >= tokens, "parents: fewer than tokens")
    opt = dict(device=seq_lens.device, dtype=torch.int32)
    total, offsets = torch.empty(batch, **opt), torch.empty(batch + 1, **opt)
    slots, positions, head = torch.empty(tokens, **opt), torch.empty(tokens, **opt), torch.empty(1, **opt)
    # a tree's mask keeps an address of its own even when no token is new
    mask = torch.empty((max(tokens, 1), mask_words), **opt)[:tokens] if parents is not None else None
    g = _lib.PagePlanGeom(batch, tokens, block_size, block_table.shape[1],
                          max(block_table.stride(0), block_table.shape[1]), free_blocks.shape[0], mask_words)
    keep = parents
    if parents is not None and parents.shape[0] == 0:
        keep = torch.empty(1, **opt)
    check(lib().nb2_page_plan(dev, ctypes.byref(g), _ints(seq_lens, "seq_lens"), _ints(new_lens, "new_lens"),
                              _ints(free_blocks, "free_blocks"), _ints(free_head, "free_head"),
                              _ints(keep, "parents"), block_table.data_ptr(), total.data_ptr(), offsets.data_ptr(),
                              head.data_ptr(), slots.data_ptr(), positions.data_ptr(),
                              None if mask is None else mask.data_ptr()))
    return PagePlan(total, offsets, slots, positions, mask, head)


def contiguous_axes(sections) -> tuple[int, ...]:
    """``axis_of`` for axes that own consecutive frequencies: (16, 24, 24) gives
    the first 16 frequencies axis 0, the next 24 axis 1, the last 24 axis 2."""
    return tuple(a for a, n in enumerate(sections) for _ in range(n))


_axis_cache: dict[tuple, tuple[int, ctypes.Array]] = {}


def _axes(axis_of, half: int):
    axis_of = (0,) * half if axis_of is None else tuple(axis_of)
    found = _axis_cache.get(axis_of)
    if found is None:
        _need(len(axis_of) <= MAX_FREQ, "axis_of: too many frequencies")
        found = _axis_cache[axis_of] = (max(axis_of, default=0) + 1,
                                               (ctypes.c_uint8 * MAX_FREQ)(*axis_of))
    _need(len(axis_of) == half, f"axis_of: expected {half} frequencies")
    return found


def rope_append(q, k, v, table, positions, axis_of=None, interleaved: bool = False, slots=None, k_cache=None,
                v_cache=None, q_out=None, k_out=None):
    """Rotary positions with several axes, and the write of k and v to the cache.

    q [tokens, q_heads, head_dim], k and v [tokens, kv_heads, head_dim] (any token
    and head strides: views of a fused projection are fine). ``table`` [length,
    rot_dim] float32 holds the cosines, then the sines, of each position;
    ``positions`` is [tokens], or [axes, tokens] with ``axis_of`` (a tuple of
    rot_dim/2) naming the axis of each frequency. Pairs are (f, f + rot_dim/2), or
    (2f, 2f + 1) when interleaved. With k_cache and v_cache [blocks, block_size,
    kv_heads, head_dim] (any strides), k and v go to ``slots``. Returns (q_out,
    k_out); both are made when not given, k_out only where there is no cache.
    """
    tokens, q_heads, dim = q.shape
    dev = context(q.device)
    dtype = q.dtype
    code = _DTYPES.get(dtype)
    _need(code is not None, "q: the type must be float32, float16 or bfloat16")
    _heads(q, "q", tokens, dtype, dim)
    _heads(k, "k", tokens, dtype, dim)
    kv = k.shape[1]
    _need(table.dim() == 2 and table.dtype == torch.float32 and table.is_contiguous() and table.is_cuda,
          "table: expected contiguous [length, rot_dim] float32 on the GPU")
    length, rot = table.shape
    axes, owner = _axes(axis_of, rot // 2)
    if positions.dim() == 1:
        _need(axes == 1 and positions.shape[0] >= tokens, "positions: one row for each axis")
        axis_stride = 0
        _ints(positions, "positions")
    else:
        _need(positions.dim() == 2 and positions.shape[0] >= axes and positions.shape[1] >= tokens
              and positions.dtype == torch.int32 and positions.is_cuda
              and (positions.stride(1) == 1 or positions.shape[1] == 1), "positions: expected [axes, tokens] int32")
        axis_stride = positions.stride(0)
    if q_out is None:
        q_out = torch.empty((tokens, q_heads, dim), device=q.device, dtype=dtype)
    else:
        _need(_heads(q_out, "q_out", tokens, dtype, dim).shape[1] == q_heads, "q_out: heads differ from q's")
    if k_cache is not None:
        _need(v is not None and v_cache is not None and slots is not None, "a cache needs v, v_cache and slots")
        _need(_heads(v, "v", tokens, dtype, dim).shape[1] == kv, "v: heads differ from k's")
        _caches(k_cache, v_cache, dtype, kv, dim)
        _need(slots.shape[0] >= tokens, "slots: fewer than tokens")
        ks, vs, vt = k_cache.stride(), v_cache.stride(), v.stride()
        cache = (k_cache.shape[1], k_cache.shape[0], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])
    else:
        _need(v is None and v_cache is None and slots is None, "v and slots belong to a cache")
        if k_out is None:
            k_out = torch.empty((tokens, kv, dim), device=q.device, dtype=dtype)
        cache, vt = (0,) * 8, (0, 0)
    if k_out is not None:
        _need(_heads(k_out, "k_out", tokens, dtype, dim).shape[1] == kv, "k_out: heads differ from k's")
        ko = k_out.stride()
    else:
        ko = (0, 0)
    if tokens == 0:
        return q_out, k_out
    qs, kst, qo = q.stride(), k.stride(), q_out.stride()
    g = _lib.RopeGeom(tokens, q_heads, kv, dim, rot, qs[0], qs[1], kst[0], kst[1], vt[0], vt[1], qo[0], qo[1], ko[0],
                      ko[1], length, axis_stride, *cache, axes, interleaved, code, 0, owner)
    check(lib().nb2_rope_append(dev, ctypes.byref(g), q.data_ptr(), k.data_ptr(),
                                None if v is None else v.data_ptr(), table.data_ptr(), positions.data_ptr(),
                                _ints(slots, "slots"), q_out.data_ptr(), None if k_out is None else k_out.data_ptr(),
                                None if k_cache is None else k_cache.data_ptr(),
                                None if v_cache is None else v_cache.data_ptr()))
    return q_out, k_out


def tree_attention(q, k_cache, v_cache, block_table, seq_lens, token_offsets, tree_mask=None, max_new: int | None = None,
                   scale: float | None = None, return_lse: bool = False, out=None):
    """Attention of each request's new tokens over its cache and its own tree.

    q [tokens, q_heads, head_dim]; the caches [blocks, block_size, kv_heads,
    head_dim] already hold the new tokens' keys and values; ``block_table``
    [batch, blocks], ``seq_lens`` [batch] (new tokens included), ``token_offsets``
    [batch + 1] and ``tree_mask`` [tokens, words] as ``page_plan`` gives them. A
    new token sees every older place of its request and the new ones in its mask
    row; without a mask, the new ones up to itself. ``max_new`` bounds the new
    tokens of a request (default: all of them). ``scale`` defaults to
    head_dim ** -0.5. Returns out, or (out, lse) with lse [tokens, q_heads] float32.
    A token that sees nothing has out 0 and lse -inf.
    """
    tokens, q_heads, dim = q.shape
    dev = context(q.device)
    dtype = q.dtype
    code = _DTYPES.get(dtype)
    _need(code is not None, "q: the type must be float32, float16 or bfloat16")
    _heads(q, "q", tokens, dtype, dim)
    kv = k_cache.shape[2] if k_cache.dim() == 4 else -1
    _caches(k_cache, v_cache, dtype, kv, dim)
    batch = seq_lens.shape[0]
    _need(block_table.dim() == 2 and block_table.shape[0] == batch and block_table.dtype == torch.int32
          and block_table.is_cuda and (block_table.stride(1) == 1 or block_table.shape[1] <= 1),
          "block_table: expected [batch, blocks] int32 on the GPU")
    _need(token_offsets.shape[0] == batch + 1, "token_offsets: expected batch + 1 values")
    words = 0
    if tree_mask is not None:
        _need(tree_mask.dim() == 2 and tree_mask.shape[0] >= tokens and tree_mask.shape[1] > 0,
              "tree_mask: expected [tokens, words]")
        words = tree_mask.shape[1]
    if out is None:
        out = torch.empty((tokens, q_heads, dim), device=q.device, dtype=dtype)
    else:
        _need(_heads(out, "out", tokens, dtype, dim).shape[1] == q_heads, "out: heads differ from q's")
    lse = torch.empty((tokens, q_heads), device=q.device, dtype=torch.float32) if return_lse else None
    if tokens == 0:
        return (out, lse) if return_lse else out
    qs, os_, ks, vs = q.stride(), out.stride(), k_cache.stride(), v_cache.stride()
    g = _lib.TreeAttnGeom(batch, tokens, q_heads, kv, dim, tokens if max_new is None else max_new, qs[0], qs[1], os_[0],
                          os_[1], k_cache.shape[1], k_cache.shape[0], block_table.shape[1],
                          max(block_table.stride(0), block_table.shape[1]), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                          words, dim ** -0.5 if scale is None else scale, code)
    check(lib().nb2_tree_attention(dev, ctypes.byref(g), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                   block_table.data_ptr(), _ints(seq_lens, "seq_lens"),
                                   _ints(token_offsets, "token_offsets"), _ints(tree_mask, "tree_mask", 2),
                                   out.data_ptr(), None if lse is None else lse.data_ptr()))
    return (out, lse) if return_lse else out


def _list(pair, requests: int, name: str):
    if pair is None:
        return None, None, 0
    ids, offsets = pair
    _need(offsets.shape[0] == requests + 1, f"{name}: expected requests + 1 offsets")
    return _ints(ids, name), _ints(offsets, name + " offsets"), ids.shape[0]


def logits_process(logits, prompt=None, output=None, row_request=None, repetition=None, presence=None, frequency=None,
                   bias=None, grammar=None, out_dtype=None, out=None, requests: int | None = None):
    """Repeated-token penalties, biases and grammar masks on logits [rows, vocab].

    ``prompt`` and ``output`` are (ids, offsets): the request's tokens so far, ids
    [offsets[r], offsets[r+1]). ``row_request`` [rows] names each row's request
    (default: row i is request i). A token in either list has a positive logit
    divided, another one multiplied, by ``repetition[r]``; one in the output list
    loses ``frequency[r]`` a time and ``presence[r]`` once. ``bias`` is (ids, values,
    offsets): added; an id's last value counts. ``grammar`` is (masks [n, words],
    rows or None): where bit v of masks[rows[i]] is clear, logit v of row i becomes
    -inf; a negative row has no rule. The result is float32 arithmetic, rounded
    once to ``out_dtype`` (default: the logits' type); ``out`` may be the logits.
    """
    _need(logits.dim() == 2 and logits.is_cuda and (logits.stride(1) == 1 or logits.shape[1] <= 1),
          "logits: expected [rows, vocab] on the GPU")
    rows, vocab = logits.shape
    dev = context(logits.device)
    code = _DTYPES.get(logits.dtype)
    _need(code is not None, "logits: the type must be float32, float16 or bfloat16")
    if out is None:
        out = torch.empty((rows, vocab), device=logits.device, dtype=out_dtype or logits.dtype)
    else:
        _need(out.shape == logits.shape and out.is_cuda and (out.stride(1) == 1 or vocab <= 1)
              and (out_dtype is None or out.dtype == out_dtype), "out: expected the logits' shape")
    out_code = _DTYPES.get(out.dtype)
    _need(out_code is not None, "out: the type must be float32, float16 or bfloat16")
    if requests is None:
        first = next((x for x in (repetition, presence, frequency) if x is not None), None)
        lists = next((x[-1] for x in (prompt, output, bias) if x is not None), None)
        requests = first.shape[0] if first is not None else lists.shape[0] - 1 if lists is not None else rows
    _need(row_request is not None or requests >= rows or rows == 0, "row_request: rows and requests differ")
    _need(row_request is None or row_request.shape == (rows,), "row_request: expected one request a row")
    p_ids, p_off, p_n = _list(prompt, requests, "prompt")
    o_ids, o_off, o_n = _list(output, requests, "output")
    b_ids = b_val = b_off = None
    b_n = 0
    if bias is not None:
        b_ids, b_off, b_n = _list((bias[0], bias[2]), requests, "bias")
        b_val = _floats(bias[1], "bias values", b_n)
    m = m_rows = None
    m_n = m_stride = 0
    if grammar is not None:
        mask, at = grammar
        _need(mask.dim() == 2 and mask.dtype == torch.int32 and mask.is_cuda
              and (mask.stride(1) == 1 or mask.shape[1] <= 1) and mask.shape[1] * 32 >= vocab,
              "grammar: expected [n, ceil(vocab / 32)] int32 words on the GPU")
        _need(at is None or at.shape == (rows,), "grammar rows: expected one a row")
        m, m_rows, m_n, m_stride = mask.data_ptr(), _ints(at, "grammar rows"), mask.shape[0], mask.stride(0)
        if m_n <= 1:
            m_stride = max(m_stride, mask.shape[1])
    in_stride, out_stride = logits.stride(0), out.stride(0)
    g = _lib.LogitsGeom(rows, vocab, requests, in_stride, out_stride, m_n, m_stride, p_n, o_n, b_n, code, out_code)
    check(lib().nb2_logits_process(dev, ctypes.byref(g), logits.data_ptr(), out.data_ptr(),
                                   _ints(row_request, "row_request"), p_ids, p_off, o_ids, o_off,
                                   _floats(repetition, "repetition", requests),
                                   _floats(presence, "presence", requests),
                                   _floats(frequency, "frequency", requests), b_ids, b_val, b_off, m, m_rows))
    return out
