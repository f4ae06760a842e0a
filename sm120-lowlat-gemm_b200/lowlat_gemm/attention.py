"""The part of a decoder layer between the qkv and the o projection: a paged key/value cache and the attention over it.

    kv_append(k, v, ...)             the new tokens' keys and values into the cache, quantised on the way
    paged_attention(q, ...)          attention of the new tokens over everything cached
    kv_read(...)                     cached tokens back, for a hand-over or a check

Cache: k_cache and v_cache [pages, kv_heads, page_size, head_dim], bf16, f16 or float8_e4m3fn, with any page, head and slot
strides (a cache that is stored [pages, page_size, kv_heads, head_dim] is passed as its .transpose(1, 2)). An e4m3 cache has a
float8_e8m0fnu power of two per row beside it: k_scale and v_scale [pages, kv_heads, page_size].
Where tokens are: page_table [batch, n] int32 names each sequence's pages in order, kv_lens [batch] int32 counts its cached
tokens with the new ones, which are the last. New tokens of all sequences are stacked: q_starts [batch + 1] int32 says where
each sequence's begin; without it every sequence has tokens / batch of them. These three live on the device and are read there,
so one captured call serves every step. A length may grow beyond the n * page_size tokens that a sequence's pages hold: tokens
behind them are not stored and not seen, and positions stay those of the whole length.

A decode step with `x` [batch, hidden]:

    qkv = lowlat_gemm.gemm(x, w_qkv)
    q, k, v = (t.view(batch, -1, 128) for t in qkv.split([heads * 128, kv_heads * 128, kv_heads * 128], dim=1))
    lowlat_gemm.kv_append(k, v, k_cache, v_cache, page_table, kv_lens, k_scale=k_scale, v_scale=v_scale)
    y = lowlat_gemm.paged_attention(q, k_cache, v_cache, page_table, kv_lens, k_scale=k_scale, v_scale=v_scale)
    y = lowlat_gemm.gemm(y.view(batch, -1), w_o)

The reference has no counterpart: it leaves cache and attention to the serving framework.
"""

from __future__ import annotations

import torch

from . import _ops  # noqa: F401  (registers torch.ops.lowlat_gemm)

# resolved once: a call through the packet looks its overload up every time
_append = torch.ops.lowlat_gemm.kv_append.default
_read = torch.ops.lowlat_gemm.kv_read.default
_attention = torch.ops.lowlat_gemm.paged_attention.default


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
              kv_lens: torch.Tensor, *, q_starts: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
              v_scale: torch.Tensor | None = None) -> None:
    """Write k and v [tokens, kv_heads, head_dim] (views of the qkv projection will do) into the cache.

    A 16-bit cache takes its own type and is a copy. An e4m3 cache takes bf16, f16 or f32: per row, e is the smallest integer
    with max|x| * 2**-e <= 448, within [-100, 119]; the row is stored as e4m3(x * 2**-e), round to nearest even, saturating,
    and its scale as 2**e. A power of two costs e4m3 no accuracy and makes value * scale exact in bf16 and fp32.
    head_dim: a multiple of 16 up to 256. The slots one call writes must be distinct: sequences may share the pages of a
    common prefix, not those they append to."""
    _append(k, v, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, q_starts)


def kv_read(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor, max_len: int, *,
            k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None):
    """The first max_len tokens of every sequence: (k, v), each [batch, max_len, kv_heads, head_dim], zero behind kv_lens.
    out_dtype: a 16-bit cache's own type (the default there), or bf16 (default), f16 or f32 for an e4m3 cache; bf16 and f32
    hold value * scale exactly (of every row that kv_append wrote), f16 rounds where its range ends."""
    if max_len < 0:
        raise ValueError(f"lowlat_gemm: max_len must not be negative, got {max_len}")
    e4m3 = k_cache.dtype == torch.float8_e4m3fn
    dtype = out_dtype or (torch.bfloat16 if e4m3 else k_cache.dtype)
    k = k_cache.new_empty((kv_lens.shape[0], max_len, k_cache.shape[1], k_cache.shape[3]), dtype=dtype)
    v = torch.empty_like(k)
    _read(k, v, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens)
    return k, v


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor, *,
                    q_starts: torch.Tensor | None = None, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    scale: float | None = None, causal: bool = True, window: int = 0, out: torch.Tensor | None = None,
                    return_lse: bool = False):
    """softmax(scale * q k^T) v of every sequence's new tokens over its cached ones (append them first): [tokens, heads,
    head_dim] in q's type, or (that, lse float32 [tokens, heads]) with return_lse, lse being the natural logarithm of the
    row's sum of exponentials - what merging with another part of the keys needs.

    q [tokens, heads, head_dim], bf16 or f16; the cache in the same type or e4m3; head_dim 64 or 128; query heads h with the
    same h // (heads / kv_heads) share a kv head, up to 32 of them. scale: 1 / sqrt(head_dim) unless given. causal: query t of
    a sequence's n sees keys up to its own position kv_len - n + t. window > 0: only the last `window` keys up to there.
    A query that sees nothing (an empty sequence, fewer cached tokens than new ones) gives zeros and lse = -inf. Rows of q
    behind the last sequence are left as they were in `out`. Forward only, like every call of this package.

    Sums, maxima and lse are fp32; the weights are rounded to 16 bits for their product with v: bf16 over a bf16 cache, else f16,
    where a weight times its v row's power of two counts down to 2^-25 of the largest at the least. e4m3 values are multiplied
    exactly; a bf16 q over them goes to f16 row by row, where its values 2^-28 below the row's largest lose bits.
    A key that a query does not see has no part in its result. There is one exception: an infinite or NaN value of v may reach
    every query of its sequence in the call, through a weight of zero; an infinite or NaN key reaches the queries that see it."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
    _attention(out, lse, q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, q_starts,
               q.shape[-1] ** -0.5 if scale is None else float(scale), causal, window)
    return (out, lse) if return_lse else out
