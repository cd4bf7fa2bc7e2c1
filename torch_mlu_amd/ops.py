"""Python entry points over the registered ops.

Names and argument meaning follow the reference's op layer
(torch_mlu/csrc/aten/operators/cnnl/transformers/attention.cpp:48-203, schemas codegen/mlu_functions.yaml:1313,1315).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch
import torch.nn.functional as F

from . import backends


def scaled_dot_product_flash_attention(query, key, value, dropout_p: float = 0.0, is_causal: bool = False,
                                       return_debug_mask: bool = False, *, scale: Optional[float] = None):
    """`aten::_scaled_dot_product_flash_attention` — q [B,Hq,Sq,D], k/v [B,Hk,Sk,D] ->
    (out, logsumexp, cum_seq_q, cum_seq_k, max_q, max_k, philox_seed, philox_offset, debug_attn_mask)."""
    return torch.ops.aten._scaled_dot_product_flash_attention(query, key, value, dropout_p, is_causal,
                                                               return_debug_mask, scale=scale)


def flash_attention_forward(query, key, value, cum_seq_q, cum_seq_k, max_q: int, max_k: int,
                            dropout_p: float = 0.0, is_causal: bool = False, return_debug_mask: bool = False, *,
                            scale: Optional[float] = None):
    """`aten::_flash_attention_forward` — packed q [Tq,Hq,D], k/v [Tk,Hk,D] with int32 cu_seqlens [B+1] ->
    (out, softmax_logsumexp [Hq,Tq], philox_seed, philox_offset, debug_attn_mask)."""
    return torch.ops.aten._flash_attention_forward(query, key, value, cum_seq_q, cum_seq_k, max_q, max_k, dropout_p,
                                                   is_causal, return_debug_mask, scale=scale)


def sdpa(query, key, value, *, is_causal: bool = False, scale: Optional[float] = None, enable_gqa: bool = False):
    """`F.scaled_dot_product_attention` with the flash backend forced, i.e. what the reference's tests do with
    `sdp_kernel(enable_flash=True, enable_math=False, enable_mem_efficient=False)`
    (test/torch_ops/test_scaled_dot_product_attention.py:24-43)."""
    with backends.sdp_kernel(enable_flash=True, enable_math=False, enable_mem_efficient=False):
        return F.scaled_dot_product_attention(query, key, value, is_causal=is_causal, scale=scale,
                                              enable_gqa=enable_gqa)


def paged_attention(query, key_pages, value_pages, block_table, seqused_k, *, is_causal: bool = False,
                    scale: Optional[float] = None, key_scales=None, value_scales=None, cu_seqlens_q=None,
                    max_seqlen_q: Optional[int] = None):
    """Decode, a few speculative tokens, or a chunk of a chunked prefill against a paged KV cache, through the C ABI
    (`fa_fwd_params.block_table`; the reference's ops have no such argument).  query [B, Hq, Sq, D]; key_pages /
    value_pages [pages, page_size, Hk, D] with page_size a multiple of 32; block_table int32 [B, max_pages] and
    seqused_k int32 [B] on the device.  -> (out [B, Hq, Sq, D], logsumexp [B, Hq, Sq]).  Inference only.

    A cache in 8 bits (float8_e4m3fn or int8 pages) goes with key_scales / value_scales, fp32 [pages, blocks, Hk]: a page has
    `blocks` blocks of a multiple of 32 tokens, and a stored value stands for itself times its block's and head's scale
    (finite, not negative).  head_dim is then a multiple of 16.  Table entries outside the pool hide their keys.

    With such a cache the query may also be packed, [T, Hq, D] with cu_seqlens_q int32 [B + 1] on the device and
    max_seqlen_q, the longest sequence's rows: prompts and decodes in one call.  -> (out [T, Hq, D], logsumexp [Hq, T]);
    rows that no sequence owns are not written."""
    if key_scales is not None or value_scales is not None:
        if key_scales is None or value_scales is None:
            raise ValueError("key_scales and value_scales go together")
        return torch.ops.torch_mlu_amd.paged_attention_8bit(query, key_pages, value_pages, key_scales, value_scales, block_table,
                                                            seqused_k, cu_seqlens_q, max_seqlen_q, is_causal, scale)
    if cu_seqlens_q is not None or max_seqlen_q is not None:
        raise ValueError("packed queries need a cache in 8 bits (key_scales and value_scales)")
    if key_pages.element_size() == 1 or value_pages.element_size() == 1:
        raise ValueError("a cache in 8 bits needs key_scales and value_scales")
    from . import capi

    return capi.fa_forward_paged(query, key_pages, value_pages, block_table, seqused_k, is_causal=is_causal, scale=scale)


class PagedPlan(NamedTuple):
    """What paged_plan returns, all on the device."""

    cu_seqlens: torch.Tensor  # int32 [B + 1]: rows before each request
    seqused_k: torch.Tensor   # int32 [B]: tokens each request holds after the step (the next step's `cached`)
    positions: torch.Tensor   # int32 [max_tokens]: position of a row in its request, 0 behind the last
    slots: torch.Tensor       # int64 [max_tokens]: page * page_size + offset of a row; -1 where it has none
    admitted: torch.Tensor    # bool [B]: the request's tokens and pages fit
    free_count: torch.Tensor  # int32 [1]: entries of free_pages that are still free


def paged_plan(cached, new_tokens, block_table, free_pages, free_count, *, page_size: int, max_tokens: int) -> PagedPlan:
    """The plan of a serving step, in one launch.  Request b holds cached[b] tokens in the pages that its row of block_table
    names and gets new_tokens[b] more (int32 [B] each; below 0 counts as 0).  Pages come off the end of free_pages (int32 [F],
    of which the first free_count[0] are free) in the requests' order, and are entered into block_table (int32
    [B, max_pages]) in place; free_pages is not changed.  A request whose rows go beyond max_tokens, whose tokens beyond its
    row of the table, or for whose pages what is free is not enough after the requests before it, is not admitted: it gets
    no pages, its rows get slot -1 and its seqused_k stays at cached.  At most 8192 requests."""
    return PagedPlan(*torch.ops.torch_mlu_amd.paged_plan(cached, new_tokens, block_table, free_pages, free_count, page_size, max_tokens))


def paged_cache_write(key, value, key_pages, value_pages, key_scales, value_scales, slots) -> None:
    """Write rows into a paged cache in 8 bits, in place.  key / value [T, Hk, D] in float16 or bfloat16, pages
    [pages, page_size, Hk, D] in float8_e4m3fn or int8, scales fp32 [pages, blocks, Hk], slots int64 [T] (paged_plan's; rows
    with a slot below 0 or beyond the pool are left out).

    A block's scale for a head only grows: to the power of two (float8_e4m3fn) or the 127th part (int8) that the largest
    finite magnitude of the new rows needs, and where it grows the block's other rows are rounded again.  A row for a block's
    first token starts the block anew.  Infinities are stored as the largest magnitude, NaN as NaN (int8: 0).  The rows of a
    call that go to one block stand next to each other and no slot is given twice, as in paged_plan's slots; otherwise such a
    block's contents are undefined, and so are those of one pool given for keys and values alike.  Inference only."""
    torch.ops.torch_mlu_amd.paged_cache_write(key, value, key_pages, value_pages, key_scales, value_scales, slots)


def rotary(query, key, positions, inv_freq, axes, *, interleaved: bool = False):
    """Rotary positions with one or several axes (time, height, width).  query [B, Hq, S, D] and key [B, Hk, S, D], or packed
    [T, H, D]; key may be None.  positions int32 or int64 [axes, S], [axes, B, S] or packed [axes, T]; inv_freq float64 or
    float32 [n] and axes int32 [n]: pair i is turned by positions[axes[i]] * inv_freq[i] (rotary_frequencies makes both).
    Pair i is elements (i, i + n) of a head, or (2 i, 2 i + 1) when interleaved; elements from 2 n on are only copied.
    Angles are formed in 64 bits.  -> (query, key), differentiable in both; with key None the second result is None."""
    q, k = torch.ops.torch_mlu_amd.rotary(query, key, positions, inv_freq, axes, interleaved, False)
    return q, (k if key is not None else None)


def rotary_frequencies(pairs: Sequence[int], *, theta: float = 10000.0, per_axis: bool = False, device=None):
    """(inv_freq float64 [n], axes int32 [n]) for `rotary`: axis a turns pairs[a] pairs, one axis after the other.  The
    frequencies theta^(-i / n) run on over all pairs, or, per_axis, over each axis's own pairs."""
    n = sum(pairs)
    if n <= 0 or any(p < 0 for p in pairs):
        raise ValueError("pairs must be counts of pairs, one for each axis")
    axes = [a for a, p in enumerate(pairs) for _ in range(p)]
    steps = [i / p for p in pairs for i in range(p)] if per_axis else [i / n for i in range(n)]
    return (torch.tensor([theta ** -s for s in steps], dtype=torch.float64, device=device),
            torch.tensor(axes, dtype=torch.int32, device=device))


def launch_count() -> int:
    """How many times this build's HIP kernels were enqueued through the registered ops."""
    return torch.ops.torch_mlu_amd._launch_count()
