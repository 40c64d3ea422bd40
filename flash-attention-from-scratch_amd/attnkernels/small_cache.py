"""A smaller KV cache: four bits a value, fewer tokens (none of it is in the
reference, whose cache is fp16 and only read).

The entry points check their arguments in the extension, in one pass:
ValueError for types, shapes and devices, RuntimeError for what the kernels do
not serve.
"""
from __future__ import annotations

import torch

from . import load_extension

__all__ = ["reshape_and_cache_mxfp4", "gather_cache_mxfp4", "paged_decode_mxfp4", "paged_decode_weights",
           "prompt_weights", "evict_cache"]


def reshape_and_cache_mxfp4(key, value, k_cache, k_scales, v_cache, v_scales, slot_mapping):
    """``reshape_and_cache`` into a 4-bit paged cache, in place.

    key, value:   [T, H_kv, D] fp16 or bf16 (heads contiguous, any token stride),
                  D a multiple of 32 up to 512
    k_cache:      [num_blocks, H_kv, block_size, D / 2] uint8 (v_cache the same)
    k_scales:     [num_blocks, H_kv, block_size, D / 32] uint8 (v_scales the same)
    slot_mapping: [T] int64 or int32, as in reshape_and_cache

    The format is MXFP4: 32 channels of a token and head share a scale
    2^(byte - 127), and each is a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6 in four
    bits (bit 3 the sign), the even channel in a byte's low half.  The scale's
    exponent is that of the group's largest magnitude, rounded to two significant
    bits, less 2 (at least -126); values round to the nearest, ties to the even
    code.  A group that holds an infinity or a NaN gets the scale byte 255 and
    reads NaN.  17 bytes hold 32 values, against 64 in fp16.
    """
    load_extension().reshape_and_cache_mxfp4(key, value, k_cache, k_scales, v_cache, v_scales, slot_mapping)


def gather_cache_mxfp4(k_cache, k_scales, v_cache, v_scales, slot_mapping, dtype=torch.float16):
    """The values that a 4-bit cache holds at some slots: the inverse of
    ``reshape_and_cache_mxfp4``, to move tokens to a full-precision cache or to
    look at them.

    Returns key and value, [T, H_kv, D] of dtype (fp16 or bf16).  A value that
    the type does not hold is rounded to it; slots that the writer skips
    (negative, past the pool) read zeros.
    """
    return load_extension().gather_cache_mxfp4(k_cache, k_scales, v_cache, v_scales, slot_mapping, dtype)


def paged_decode_mxfp4(q, k_cache, k_scales, v_cache, v_scales, block_tables, context_lens, max_context_len,
                       scale=None, partition_size=None, weights=None):
    """Decode attention over a 4-bit paged cache (``reshape_and_cache_mxfp4``'s).

    q:            [B, H, D] fp16 or bf16, D in {64, 128}, H / H_kv from 1 to 16; the
                  cache's values are rounded to its type
    k_cache, k_scales, v_cache, v_scales: 16-byte aligned (whole tensors and slices
                  of whole pages of 16 tokens are)
    block_tables, context_lens, max_context_len, scale: as in paged_decode; a
                  context of 0 tokens gives zeros, tokens from max_context_len on
                  are ignored
    partition_size: tokens per split (rounded up to a multiple of 256); None: the
                  kernel cuts the contexts into splits of about equal size
    weights:      None, or float32 [B, H_kv, >= max_context_len], to which each
                  token's softmax weight is added, summed over the query heads of its
                  kv head (``paged_decode_weights``)
    """
    return load_extension().paged_decode_mxfp4(q, k_cache, k_scales, v_cache, v_scales, block_tables, context_lens,
                                               max_context_len, scale, partition_size, weights)


def paged_decode_weights(q, k_cache, v_cache, block_tables, context_lens, max_context_len, weights,
                         scale=None, partition_size=None):
    """Decode attention over an fp16 or bf16 paged cache that keeps count of what
    each cached token contributes.

    Arguments and result as in ``paged_decode`` (q and the caches may be bf16 too,
    H / H_kv from 1 to 16), and

    weights:      float32 [B, H_kv, >= max_context_len], rows contiguous: to
                  weights[b, h, t] is added token t's softmax weight in sequence b,
                  summed over the query heads of kv head h.  Row b belongs to the
                  sequence, so pages that sequences share are counted apart.
                  Positions from the context length on are left as they are; keep
                  them zero (``prompt_weights`` and ``evict_cache`` do) for the
                  tokens to come.
    """
    return load_extension().paged_decode_weights(q, k_cache, v_cache, block_tables, context_lens, max_context_len,
                                                 weights, scale, partition_size)


def prompt_weights(q, k, cu_seqlens, max_seqlen, weights, last=None, scale=None):
    """What a causal prefill's attention gave each of its tokens, written to
    weights: the start of the sums that ``paged_decode_weights`` goes on with.

    q, k, cu_seqlens, max_seqlen: the packed prompts as in flash_attention_varlen
                  (fp16 or bf16; any token stride)
    weights:      float32 [B, H_kv, length], length >= max_seqlen, rows contiguous.
                  weights[b, h, j] = the sum over the query heads of kv head h and
                  over queries i >= j of softmax(scale q_i.k)_j, and 0 from the
                  sequence's length on
    last:         only the sequence's last so many queries count; None: all
    """
    load_extension().prompt_weights(q, k, cu_seqlens, max_seqlen, weights, last, scale)


def evict_cache(k_cache, v_cache, block_tables, context_lens, weights, budget, recent=0, k_scales=None, v_scales=None,
                new_block_tables=None):
    """Cut paged caches back to ``budget`` tokens a sequence: each kv head keeps
    its last ``recent`` tokens and, of the others, those of the largest weight (of
    equal ones the first; a NaN counts as the largest), in their order.

    k_cache:      [num_blocks, H_kv, block_size, D] fp16 or bf16 (v_cache the same);
                  with k_scales and v_scales a 4-bit cache
    weights:      float32 [B, H_kv, length], rows contiguous, of
                  ``paged_decode_weights`` and ``prompt_weights``
    new_block_tables: None: the kept rows move to the front of the sequence's own
                  pages, and rows past them stay as they are; a page must not be in
                  two sequences then, if one of them is cut, nor twice in that one.
                  Else [B, new_max_blocks] pages that all kept rows are written to
                  (also of sequences that keep everything), none of them in
                  block_tables or there twice

    Returns (context_lens, weights, kept): the new lengths, int32 [B]; the kept
    tokens' weights, zero past them, in new memory of the old shape; and int32
    [B, H_kv, budget], where position i's token was, -1 past the new length.
    Keys are not turned: positional encodings stay those of the old positions.
    """
    return load_extension().evict_cache(k_cache, v_cache, block_tables, context_lens, weights, budget, recent,
                                        k_scales, v_scales, new_block_tables)
