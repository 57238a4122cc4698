"""The paged int8 K/V cache for serving: append (with the position rotation on the way), attend, read back.

A cache is four tensors: codes int8 [pages, H_kv, page_size, D] and scales fp32 [pages, H_kv] for K and for
V; a page of one head stands for ``code * scale``.  ``block_table`` int32 [B, pages per sequence] names the
page of every ``page_size`` tokens of a sequence and ``context_lens`` int32 [B] counts its tokens, those of
the current step included.  The reference's paged cache keeps one scale per token (reference
superl8/ops.py:730-918); one per page costs nothing to read and can still be kept while tokens arrive one
at a time.

A step of a serving loop::

    lens += 1                                                     # on the device: no host read-back
    q = kv_append_paged(k, v, *cache, table, lens, q=q, inv_freq=inv_freq)
    out = attn_paged_cached(q, *cache, table, lens, max_context_len=longest)

Every call is asynchronous on the current stream, reads nothing back and can be captured in a CUDA graph.
None is differentiable: the results carry no gradient.
"""

from __future__ import annotations

import torch

from . import _C, _lib


def empty_paged_cache(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, device="cuda"):
    """(k_i8, k_scale, v_i8, v_scale) of an empty cache: scales of 0 mark pages that hold nothing."""
    if page_size not in (16, 32, 64, 128, 256):
        raise ValueError(f"superl8_b200 empty_paged_cache: page size must be 16/32/64/128/256, got {page_size}")
    if head_dim not in (32, 64, 128, 256):
        raise ValueError(f"superl8_b200 empty_paged_cache: head dim must be 32/64/128/256, got {head_dim}")
    codes = [torch.zeros(num_pages, num_kv_heads, page_size, head_dim, dtype=torch.int8, device=device) for _ in "kv"]
    scales = [torch.zeros(num_pages, num_kv_heads, dtype=torch.float32, device=device) for _ in "kv"]
    return codes[0], scales[0], codes[1], scales[1]


def kv_append_paged(k, v, k_i8, k_scale, v_i8, v_scale, block_table, context_lens, *, new_lens=None, q=None, positions=None,
                    inv_freq=None, freq_axis=None, interleaved: bool = False):
    """Stores the newest tokens of every sequence: k, v fp16/bf16 [B, H_kv, M, D] (strided views are taken in
    place).  Row i of sequence b is the token at place ``context_lens[b] - new_lens[b] + i``
    (``new_lens`` int32 [B], None: M for all; rows behind it are not read).

    With ``inv_freq`` K is rotated first, and ``q`` [B, H_q, M, D] with it: the call returns the rotated q
    (rows past ``new_lens`` are zeros), or None without q.  ``positions`` [B, M] or [axes, B, M] as in
    ``apply_rope``; None is the token's place.

    Per touched page and head the scale becomes max(scale of the older tokens, max|new| / 127, 2^-40), the
    new codes round(x / scale); when the scale grows, the older codes of that page are rounded again
    (each growth moves a value by at most half a step).  Whatever lies behind the last token of a page is
    left as it was.  A page that is appended to must be named once only, by one sequence; places outside the table
    and page numbers outside the cache are skipped.  A NaN or infinity makes its whole page NaN."""
    return _C.kv_append_paged(k, v, k_i8, k_scale, v_i8, v_scale, block_table, context_lens, new_lens, q, positions, inv_freq,
                              freq_axis, interleaved)


def kv_read_paged(k_i8, k_scale, v_i8, v_scale, block_table, context_lens, num_tokens: int, *, first=None,
                  dtype=torch.float16):
    """The cache's values as (k, v) fp16 / bf16 [B, H_kv, num_tokens, D]: row j is token ``first[b] + j``
    (``first`` int32 [B], None: 0), zeros where the sequence has no such token.  For handing sequences to
    the 16-bit operators, moving them elsewhere, or looking at what a cache holds."""
    return _C.kv_read_paged(k_i8, k_scale, v_i8, v_scale, block_table, context_lens, num_tokens, first, dtype)


def attn_paged_cached(q, k_i8, k_scale, v_i8, v_scale, block_table, context_lens, *, scale: float | None = None,
                      causal: bool = True, window_left: int = -1, query_lens=None, max_context_len: int | None = None,
                      backend: int = _lib.SL8_BACKEND_AUTO):
    """softmax(scale q.K^T) V over the paged cache; q fp16/bf16 [B, H_q, M, D] (rotated where the cache's
    keys are), the result like q.

    M = 1 is a decode step; with several query tokens (drafted tokens, the next piece of a prompt) row i of
    sequence b is the token at place ``context_lens[b] - query_lens[b] + i`` (``query_lens`` int32 [B],
    None: M for all; rows past it give zeros) and sees the keys up to its own place, or all of the context
    with ``causal=False``; ``window_left`` >= 0 leaves only keys in (place - window_left, ...].  A row that
    sees no key gives zeros.  ``max_context_len`` (host) is an upper bound of ``context_lens`` (keys at
    or past it are not seen); None takes what the table can hold.  With many query rows per KV head
    (M H_q / H_kv above 32, where it is estimated to be faster) the call runs on the tensor-memory path and
    widens the codes into a workspace of 4 D bytes per key and KV head, at most 2 GiB or one (sequence, head)
    at a time, sized by that bound; ``backend`` (SL8_BACKEND_MMA / SL8_BACKEND_TCGEN05) forces one of the two."""
    return _C.attn_paged(q, k_i8, k_scale, v_i8, v_scale, block_table, context_lens, scale, causal, window_left, query_lens,
                         max_context_len, backend)
