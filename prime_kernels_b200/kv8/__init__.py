"""Paged KV cache held in 8 bits, and causal attention over it (sm_100a, head dim 64).

The decode step keeps its cache in bf16; these operators store K and V rows in half the bytes, with the quantiser the
package uses elsewhere (e4m3 values, power-of-two scales rounded up so that nothing saturates), one E8M0 scale per
(page, kv head) for K and one for V, and attend to them with one query token per request (a decode step), a few
(drafts being verified) or many (prompt chunks).  The cache has the decode step's two layouts, in one byte per element:

* ``[pages, kv_heads, page_size, 128]``: K in 0..63, V in 64..127
* ``[2, pages, page_size, kv_heads, 64]``: K and V planes

``scales`` is ``[pages, kv_heads, 2]`` (K, V).  ``block_table`` int32 ``[batch, columns]`` holds each request's pages;
an entry outside the pool stands for no page (nothing is stored there, its tokens are masked).  ``seq_lens`` int32
``[batch]`` include the new tokens.  ``cu_seqlens`` int32 ``[batch + 1]``: request ``r`` owns rows
``cu[r] .. cu[r + 1] - 1`` of q / k / v, the last positions of its sequence; ``None``: row ``r`` is request ``r``.
Nothing here synchronises or keeps state between calls, so calls can be captured into CUDA graphs.
"""
from __future__ import annotations

import torch

from .._cabi import library, load_ops
from ..geometry import HEAD_DIM

load_ops()

__all__ = ["PAGE_SIZES", "empty_cache", "append", "attention", "check_status", "dequantise"]

PAGE_SIZES = (16, 32, 64, 128, 256)


@torch.library.register_fake("prime_kv8::append")
def _append_fake(k, v, cache, scales, block_table, seq_lens, cu_seqlens):
    return None


@torch.library.register_fake("prime_kv8::attention")
def _attention_fake(q, cache, scales, block_table, seq_lens, cu_seqlens, max_query_len, scale):
    return q.new_empty(q.shape)


@torch.library.register_fake("prime_kv8::attention_lse")
def _attention_lse_fake(q, cache, scales, block_table, seq_lens, cu_seqlens, max_query_len, scale):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


@torch.library.register_fake("prime_kv8::attention_out")
def _attention_out_fake(q, cache, scales, block_table, seq_lens, cu_seqlens, max_query_len, scale, out, lse):
    return None


_append = torch.ops.prime_kv8.append.default
_attention = torch.ops.prime_kv8.attention.default
_attention_lse = torch.ops.prime_kv8.attention_lse.default
_attention_out = torch.ops.prime_kv8.attention_out.default


def empty_cache(pages: int, kv_heads: int, page_size: int = 16, *, planes: bool = False, device="cuda"):
    """A cache of zeros and its scales: ``(cache e4m3, scales e8m0)``.  ``planes`` picks the K and V planes layout."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    shape = (2, pages, page_size, kv_heads, HEAD_DIM) if planes else (pages, kv_heads, page_size, 2 * HEAD_DIM)
    cache = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    return cache, torch.zeros((pages, kv_heads, 2), dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)


def append(k, v, cache, scales, block_table, seq_lens, cu_seqlens=None) -> None:
    """Store new K and V rows (bf16 ``[tokens, kv_heads, 64]``, token and head strides multiples of 8) into their pages.

    A page whose first slot is among the new tokens takes the scale of its new tokens, ``2^ceil(log2(amax / 448))``; a
    page begun by an earlier call takes the larger of that and its own, and the tokens it holds are re-rounded where
    the scale grows.  NaN and Inf do not count for the scale (Inf saturates, NaN stays).  A page that is written to
    belongs to one request; pages that several requests read may be shared."""
    _append(k, v, cache, scales, block_table, seq_lens, cu_seqlens)


def attention(q, cache, scales, block_table, seq_lens, cu_seqlens=None, *, max_query_len: int | None = None,
              scale: float | None = None, out=None, return_lse: bool = False):
    """Causal attention of ``q`` (bf16 ``[tokens, q_heads, 64]``, strides multiples of 8) over the cache.

    Token ``j`` of a request with ``n`` rows sees its first ``seq_len - n + j + 1`` positions; query head ``a`` reads kv
    head ``a // (q_heads // kv_heads)``.  A row that sees no key gets 0 (lse ``-inf``).  ``max_query_len``: the longest
    request's rows, where the caller knows it (every row is computed whatever it says); ``scale`` defaults to 1/8.
    Weights and V values meet in f16: a weight is off by ``2**-11`` of itself or ``2**-25`` of the row's largest product of
    weight and V scale, so what pages of a V scale below ``2**-13`` of another's add to dims in which that one holds nothing
    loses bits, and is lost from ``2**-25`` on.
    Returns bf16 ``out`` of q's shape, or ``(out, lse)`` with the natural-log normaliser fp32 ``[tokens, q_heads]``.
    With ``out`` given, rows that belong to no request are left as they are there; otherwise they are undefined.  ``out``
    may not share memory with ``q``.

    How keys are split over CTAs follows the width of ``block_table``, since lengths are on the device: pass
    ``block_table[:, :columns]`` where the longest sequence is known (8 requests of 5 tokens at 2047 keys: 9.6 us, 12.4 us
    with a table for 8192).  NaN among the V values of a chunk's later tokens does not reach its earlier rows, but costs:
    the kernel for prompt chunks computes the rows of such a tile once more without tensor cores, in milliseconds."""
    n, s = max_query_len or 0, HEAD_DIM ** -0.5 if scale is None else scale
    if out is None:
        return (_attention_lse if return_lse else _attention)(q, cache, scales, block_table, seq_lens, cu_seqlens, n, s)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    _attention_out(q, cache, scales, block_table, seq_lens, cu_seqlens, n, s, out, lse)
    return (out, lse) if return_lse else out


_expired: dict[int, int] = {}


def check_status(device="cuda") -> None:
    """Synchronise and raise if a bounded device-side wait of an earlier :func:`attention` call on ``device`` gave up (the
    rows that such a call could not finish are NaN, out and lse)."""
    with torch.cuda.device(device):
        at, n = torch.cuda.current_device(), library().pk_kv8_wait_timeouts()
    if n < 0:
        raise RuntimeError("kv8: the device could not be asked for expired waits")
    new, _expired[at] = n - _expired.get(at, 0), n
    if new:
        raise RuntimeError(f"kv8 attention failed on the device: {new} bounded waits gave up")


def dequantise(cache, scales):
    """The values a cache stands for, fp32 in the cache's shape (plain PyTorch; for checks)."""
    e = torch.exp2(scales.view(torch.uint8).double() - 127.0)
    x = cache.view(torch.float8_e4m3fn).double()
    if cache.dim() == 4:
        e = e[:, :, None, :, None].expand(*e.shape[:2], 1, 2, HEAD_DIM).reshape(*e.shape[:2], 1, 2 * HEAD_DIM)
    else:
        e = e.permute(2, 0, 1)[:, :, None, :, None]
    return (x * e).float()
