"""Paged-attention kernel API for MI355X -- drop-in for the reference's
``sglang_mlx.metal_kernels`` (metal_kernels.py:1-96) over PyTorch-ROCm
tensors.

Operations:
    paged_attention_v1   single-softmax paged decode attention
    paged_attention_v2   split-K paged decode with a log-sum-exp merge
    paged_attention_cascade  decode with radix-shared prefixes computed once
                         per group of sequences (a host-built plan)
    reshape_and_cache    scatter new KV tokens into the cache (in place)
    build_step_tables    block tables, slots and positions of a step, from
                         request lengths
    qk_norm_rope         per-head norm of queries and keys and their rotation
                         by position (rotary.rotary_table makes the table)
    qk_norm_rope_and_cache  the same with the append of keys and values
    paged_attention_window  decode over a sliding window and a few first tokens
    paged_attention_extend  causal attention of several new tokens per sequence
                         (prefills, chunks of them, drafted tokens)
    copy_blocks          block copies inside the caches
    swap_blocks          block copies between two buffers
    convert_fp8          element-wise conversion with a scale, FP8 E4M3 codes
                         as uint8 tensors

Tensors live on a HIP device; kernels run asynchronously on the current
stream of that device.
"""

from __future__ import annotations

import torch

from . import _ext


def paged_attention_v1(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    num_kv_heads: int,
    scale: float,
    block_size: int,
    max_seq_len: int,
    alibi_slopes: torch.Tensor | None = None,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> torch.Tensor:
    """Single-pass paged attention (metal_kernels.py:20-61).

    Args:
        query: [num_seqs, num_heads, head_size]
        key_cache: [num_blocks, num_kv_heads, head_size/x, block_size, x]
        value_cache: [num_blocks, num_kv_heads, head_size, block_size]
        block_tables: [num_seqs, max_num_blocks_per_seq] (32-bit ids)
        context_lens: [num_seqs]
        num_kv_heads: Number of KV heads
        scale: Attention scaling factor
        block_size: Number of tokens per block
        max_seq_len: Maximum sequence length
        alibi_slopes: Optional ALiBi slopes [num_heads]
        k_scale, v_scale: for uint8 (FP8 E4M3) caches, K = decode(code) *
            k_scale and V = decode(code) * v_scale; ignored otherwise

    Returns:
        Output tensor [num_seqs, num_heads, head_size], dtype of query.
    """
    return _ext.paged_attention_v1(query, key_cache, value_cache, block_tables, context_lens,
                                   num_kv_heads, scale, block_size, max_seq_len, alibi_slopes, k_scale, v_scale)


def paged_attention_v2(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    num_kv_heads: int,
    scale: float,
    block_size: int,
    max_seq_len: int,
    alibi_slopes: torch.Tensor | None = None,
    partition_size: int = 512,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> torch.Tensor:
    """Split-K paged attention for long contexts: each partition of
    ``partition_size`` tokens yields (max, sum, output); partitions are merged
    by log-sum-exp.  Same arguments and result as ``paged_attention_v1``."""
    return _ext.paged_attention_v2(query, key_cache, value_cache, block_tables, context_lens,
                                   num_kv_heads, scale, block_size, max_seq_len, alibi_slopes,
                                   partition_size, k_scale, v_scale)


def paged_attention_cascade(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    num_kv_heads: int,
    scale: float,
    block_size: int,
    max_seq_len: int,
    plan,
    alibi_slopes: torch.Tensor | None = None,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> torch.Tensor:
    """Paged attention with radix-shared prefixes computed once per group of
    sequences (``plan``: srt.mem_cache.build_cascade_plan over the same block
    tables).  Same arguments and result as ``paged_attention_v1`` (paged 5-D
    caches), to within floating-point rounding."""
    return _ext.paged_attention_cascade(query, key_cache, value_cache, block_tables, context_lens, num_kv_heads,
                                        scale, block_size, max_seq_len, plan, alibi_slopes, k_scale, v_scale)


def reshape_and_cache(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> list[torch.Tensor]:
    """Scatter-write new KV tokens into the cache (metal_kernels.py:64-74).

    key/value: [num_tokens, num_kv_heads, head_size]; slot_mapping:
    [num_tokens], -1 = padding (skipped).  The caches are updated in place
    and returned as [key_cache, value_cache].  Paged 5-D caches and 3-D
    MHATokenPool buffers [num_slots, num_kv_heads, head_size] are accepted.
    uint8 caches hold FP8 E4M3 codes (the reference's format) of
    key / k_scale and value / v_scale; the paged layout then has x = 16.
    """
    return _ext.reshape_and_cache(key, value, key_cache, value_cache, slot_mapping, k_scale, v_scale)


def build_step_tables(
    request_blocks: torch.Tensor,
    rows: torch.Tensor,
    context_lens: torch.Tensor,
    query_lens: torch.Tensor,
    new_blocks: torch.Tensor,
    block_size: int,
    num_tokens: int,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Block tables, slots and positions of one step, on the device.

    Args:
        request_blocks: [num_requests, max_blocks] int32, contiguous: each open
            request's block ids in context order.  The blocks that the step
            adds are stored into it.
        rows: [num_seqs], each sequence's row of request_blocks, all different;
            -1 (any row outside the table) is a padding sequence without tokens
        context_lens: [num_seqs], tokens of each sequence with its new ones
        query_lens: [num_seqs], its new tokens
        new_blocks: 1-D, free block ids: sequences take theirs from it in order,
            ceil(context / block_size) - ceil((context - new) / block_size) each
        block_size: Number of tokens per block
        num_tokens: length of the token outputs (padding included)

    Returns:
        block_tables [num_seqs, max_blocks] (-1 past a sequence's blocks),
        slot_mapping and positions [num_tokens] of the new tokens end to end
        (-1 and 0 past the last), query_start_loc [num_seqs + 1]; all int32.

    A sequence whose context exceeds max_blocks * block_size has no tokens; with
    too few new_blocks the blocks and slots that are missing are -1.
    """
    return _ext.build_step_tables(request_blocks, rows, context_lens, query_lens, new_blocks, block_size, num_tokens)


def qk_norm_rope(
    query: torch.Tensor,
    key: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm of each head of queries and keys, then their rotation by position.

    Args:
        query: [num_tokens, num_heads, head_size], head_size a multiple of 8 up
            to 256; rows may be views of a wider projection
        key: [num_tokens, num_kv_heads, head_size], the same type
        positions: [num_tokens] (32-bit ids); those outside the table take its
            nearest row
        cos_sin: [num_positions, rotary_dim] float32, rotary_dim / 2 cosines,
            then as many sines (rotary.rotary_table); the head's first
            rotary_dim elements turn, the others stay
        q_weight, k_weight: [head_size], of the queries' type or float32: rows
            become x / sqrt(mean(x^2) + eps) * weight first; None: no norm
        interleaved: pairs are neighbours (2 i, 2 i + 1) rather than halves
            (i, i + rotary_dim / 2)

    Returns:
        New contiguous (query, key).  Computed in float32, rounded once.
    """
    return _ext.qk_norm_rope(query, key, positions, cos_sin, q_weight, k_weight, eps, interleaved)


def qk_norm_rope_and_cache(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    positions: torch.Tensor,
    cos_sin: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> list[torch.Tensor]:
    """``qk_norm_rope`` and ``reshape_and_cache`` of its keys and of the values
    in one launch; returns [query, key_cache, value_cache].

    Caches, slot_mapping and scales as in ``reshape_and_cache`` (paged 5-D with
    blocks of 8, 16 or 32 tokens, or token rows [..., num_kv_heads, head_size]).
    Keys are rounded once, from float32 to the cache's type.
    """
    return _ext.qk_norm_rope_and_cache(query, key, value, positions, cos_sin, key_cache, value_cache, slot_mapping,
                                       q_weight, k_weight, eps, interleaved, k_scale, v_scale)


def paged_attention_window(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    num_kv_heads: int,
    scale: float,
    block_size: int,
    max_seq_len: int,
    window: int,
    num_sinks: int = 0,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> torch.Tensor:
    """Decode attention over a sliding window: each sequence's query attends to
    the last ``window`` tokens of its context (its own among them) and to the
    first ``num_sinks``.  Arguments as ``paged_attention_v1`` (paged 5-D caches;
    bfloat16 or float16 queries over caches of their type or uint8); only the
    tokens that are attended to are read.
    """
    return _ext.paged_attention_window(query, key_cache, value_cache, block_tables, context_lens, num_kv_heads, scale,
                                       block_size, max_seq_len, window, num_sinks, k_scale, v_scale)


def paged_attention_extend(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    num_kv_heads: int,
    scale: float,
    block_size: int,
    max_seq_len: int,
    max_query_len: int,
    window: int = 0,
    num_sinks: int = 0,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> torch.Tensor:
    """Causal attention of each sequence's new tokens over its cached context,
    the new tokens among it (prefills, chunks of them, drafted tokens; a batch
    may mix them with single tokens).

    Args:
        query: [num_tokens, num_heads, head_size], the sequences end to end
        context_lens: [num_seqs], tokens in the cache, the new ones included: the
            n query rows of a sequence are its context's last n tokens
        query_start_loc: [num_seqs + 1], each sequence's first query row, and
            the number of rows; output rows behind it are zero
        max_query_len: at least the most query rows of one sequence; the
            closer, the better the kernel fits (one for a few rows per sequence,
            one for many)
        window, num_sinks: with a window > 0 a query sees the ``window`` last
            tokens up to its own, and the context's first ``num_sinks``
        The others as ``paged_attention_window``.

    Returns:
        [num_tokens, num_heads, head_size]; a row that sees no token (context 0
        or beyond max_seq_len, a sequence of more than max_query_len rows, rows
        before the context's first token) is zero.
    """
    return _ext.paged_attention_extend(query, key_cache, value_cache, block_tables, context_lens, query_start_loc,
                                       num_kv_heads, scale, block_size, max_seq_len, max_query_len, window, num_sinks,
                                       k_scale, v_scale)


def copy_blocks(
    key_caches: list[torch.Tensor],
    value_caches: list[torch.Tensor],
    block_mapping: torch.Tensor,
) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
    """Copy blocks within the caches (metal_kernels.py:77-85)."""
    return _ext.copy_blocks(key_caches, value_caches, block_mapping)


def swap_blocks(src: torch.Tensor, dst: torch.Tensor, block_mapping: torch.Tensor) -> torch.Tensor:
    """Blit blocks between two buffers (metal_kernels.py:88-96)."""
    return _ext.swap_blocks(src, dst, block_mapping)


def convert_fp8(dst: torch.Tensor, src: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """Element-wise precision conversion with a scale (the reference's
    convert_fp8_kernel, convert_fp8.metal:13-80).  uint8 tensors hold FP8
    E4M3 codes in the reference's format (bias 7, exponent 15 = inf / NaN).
    fp8 -> T: decode * scale; T -> fp8: encode(x / scale); fp8 -> fp8:
    encode(decode * scale); T -> U: x * scale.  dst is written in place and
    returned."""
    return _ext.convert_fp8(dst, src, scale)

