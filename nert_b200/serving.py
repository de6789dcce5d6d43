"""Serving rows over torch CUDA tensors: one step of a server over a paged cache.

``page_plan`` once a step, then ``rope_append`` and ``tree_attention`` for each
layer, and ``logits_process`` before picking tokens. torch provides memory and
the stream; every computation is a kernel of libnert_b200.so.

Unlike the wrappers of ``nert_b200.ops``, these launch on torch's current
stream (through one context a stream, made on first use) and return without
synchronising, so a step can be queued, overlapped or captured in a CUDA graph
(after one uncaptured call, or ``context()``, on the capturing stream). A captured
graph has a workspace of its own, so it may be replayed on any stream, beside
other graphs and calls; one replay at a time of each, as CUDA has it.
Arguments that the host can see are checked before the launch (``ValueError``,
or ``NB2Error`` from the library); values on the device (lengths, blocks, slots,
token ids) are checked by the kernels, and ``synchronize()`` raises what they
recorded. The checks and the call run in nert_b200_torch.so
(``csrc/torch/serving_torch.cpp``); there is no fallback without it.

Inference only: outputs carry no gradient, whatever the inputs ask for. The
context of a stream is kept for the life of the process, with its workspace (up
to 40 MB, outside torch's allocator); torch's streams come from fixed pools.

Metadata tensors are contiguous int32; masks are int32 words of 32 bits.
"""

from __future__ import annotations

import importlib.util
import os
from typing import NamedTuple

import torch

from . import _lib

_lib.lib()  # the native library, or a clear error


def _load():
    path = os.path.join(_lib.HERE, "lib", "nert_b200_torch.so")
    if not os.path.exists(path):
        raise RuntimeError(f"native module missing: {path}; run python nert_b200/build.py")
    spec = importlib.util.spec_from_file_location("nert_b200_torch", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


_native = _load()


def synchronize(device: torch.device | str = "cuda") -> None:
    """Waits for torch's current stream; raises what the kernels of this module
    recorded on it, and what the GPU's replayed graphs did, on whatever stream
    (NB2Error with status ERR_DEVICE)."""
    _native.synchronize(torch.device(device))


def context(device: torch.device | str = "cuda") -> int:
    """The library's context (an ``nb2_device*``) for torch's current stream."""
    return _native.context(torch.device(device))


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
    return PagePlan(*_native.page_plan(seq_lens, new_lens, block_table, free_blocks, block_size, tokens, parents,
                                       mask_words, free_head))


def contiguous_axes(sections) -> tuple[int, ...]:
    """``axis_of`` for axes that own consecutive frequencies: (16, 24, 24) gives
    the first 16 frequencies axis 0, the next 24 axis 1, the last 24 axis 2."""
    return tuple(a for a, n in enumerate(sections) for _ in range(n))


_axis_cache: dict[tuple[int, ...], tuple[int, bytes]] = {}


def _axes(axis_of) -> tuple[int, bytes]:
    found = _axis_cache[axis_of] = (max(axis_of, default=0) + 1, bytes(axis_of))
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
    if axis_of is None:
        axes, owner = 1, None
    else:
        axis_of = tuple(axis_of)
        axes, owner = _axis_cache.get(axis_of) or _axes(axis_of)
    return _native.rope_append(q, k, v, table, positions, owner, axes, interleaved, slots, k_cache, v_cache, q_out,
                               k_out)


def tree_attention(q, k_cache, v_cache, block_table, seq_lens, token_offsets, tree_mask=None, max_new: int | None = None,
                   scale: float | None = None, return_lse: bool = False, out=None):
    """Attention of each request's new tokens over its cache and its own tree.

    q [tokens, q_heads, head_dim]; the caches [blocks, block_size, kv_heads,
    head_dim] already hold the new tokens' keys and values; ``block_table``
    [batch, blocks], ``seq_lens`` [batch] (new tokens included), ``token_offsets``
    [batch + 1] and ``tree_mask`` [tokens, words] as ``page_plan`` gives them. A
    new token sees every older place of its request and the new ones in its mask
    row; without a mask, the new ones up to itself. ``max_new`` bounds the new
    tokens of a request (default: all of them) and picks the kernel: give it,
    where a call has many requests of few tokens. ``scale`` defaults to
    head_dim ** -0.5. Returns out, or (out, lse) with lse [tokens, q_heads] float32.
    A token that sees nothing has out 0 and lse -inf.
    """
    result = _native.tree_attention(q, k_cache, v_cache, block_table, seq_lens, token_offsets, tree_mask, max_new, scale,
                                    return_lse, out)
    return result if return_lse else result[0]


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
    return _native.logits_process(logits, prompt, output, row_request, repetition, presence, frequency, bias, grammar,
                                  out_dtype, out, requests)
