"""Operators for exported modules that ATen has none for.

``torch.ops.chroma_amd.paged_attention`` and ``paged_chunk_attention`` (the functions here) can be called in any module that is
exported and compiled; eager calls and other devices compute the plain forms below. Importing this module
registers them (the compiler does, so exported files that hold them load there).
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor


@torch.library.custom_op("chroma_amd::paged_attention", mutates_args=())
def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, k_new: Optional[Tensor], v_new: Optional[Tensor], table: Tensor,
                    lengths: Tensor, sinks: Optional[Tensor], scale: float, window: int = 0, first: int = 0) -> Tensor:
    """Attention of one new token per sequence over its cached keys and values, which lie in pages.

    q [S, KV, G, D]; k_pages and v_pages [P, R, KV, D]; k_new and v_new [S, KV, D], the token's own row at
    position ``lengths``, or None; table [S, N] and lengths [S] int64; sinks [KV * G], a learned logit per query
    head, or None. Row j < lengths[b] of sequence b is row j % R of page table[b, j // R]. ``window`` > 0 leaves
    out the rows at least ``window`` before the token's position, but for the ``first`` first ones. Lengths
    below 0 count as 0 and above N * R as N * R, rows on pages outside [0, P) are not seen, and a token that
    sees no row gets zeros. Scores and sums are float's, the result is rounded once; compiled with bfloat16, a weight
    meets the values as two bfloat16 halves (within 2^-16 of it)."""
    _check(q, k_pages, v_pages, k_new, v_new, table, lengths, sinks, window, first)
    sequences, kv_heads, group, dim = q.shape
    pages, rows = k_pages.shape[:2]
    span = table.shape[1] * rows
    held = lengths.clamp(0, span)
    j = torch.arange(span, device=q.device)[None, :]
    seen = (j < held[:, None]) & ((table >= 0) & (table < pages)).repeat_interleave(rows, 1)
    if window:
        position = held[:, None] - (0 if k_new is not None else 1)
        seen = seen & ((j > position - window) | (j < first))
    where = table.clamp(0, pages - 1)

    def cached(values: Tensor) -> Tensor:  # [S, KV, span, D], zero where nothing is seen
        gathered = values[where].float().reshape(sequences, span, kv_heads, dim)
        return torch.where(seen[:, :, None, None], gathered, 0.0).transpose(1, 2).contiguous()

    k, v = cached(k_pages), cached(v_pages)
    scaled = q.float() * scale
    scores = (scaled[:, :, :, None, :] * k[:, :, None]).sum(-1).masked_fill(~seen[:, None, None, :], -math.inf)
    if k_new is not None:
        scores = torch.cat([scores, (scaled * k_new.float()[:, :, None, :]).sum(-1, keepdim=True)], -1)
        v = torch.cat([v, v_new.float()[:, :, None, :]], 2)
    joined = scores
    if sinks is not None:
        joined = torch.cat([scores, sinks.float().reshape(1, kv_heads, group, 1).expand(sequences, -1, -1, 1)], -1)
    top = joined.amax(-1, keepdim=True) if joined.shape[-1] else joined.new_zeros(sequences, kv_heads, group, 1)
    top = torch.where(top == -math.inf, 0.0, top)
    total = torch.exp(joined - top).sum(-1, keepdim=True)
    mixed = (torch.exp(scores - top)[..., None] * v[:, :, None]).sum(-2)
    return torch.where(total == 0, 0.0, mixed / total).to(q.dtype)


@paged_attention.register_fake
def _(q, k_pages, v_pages, k_new, v_new, table, lengths, sinks, scale, window=0, first=0):
    _check(q, k_pages, v_pages, k_new, v_new, table, lengths, sinks, window, first)
    return q.new_empty(q.shape)


def _check(q, k_pages, v_pages, k_new, v_new, table, lengths, sinks, window, first) -> None:
    if q.dim() != 4 or k_pages.dim() != 4 or tuple(v_pages.shape) != tuple(k_pages.shape):
        raise ValueError("paged_attention wants q [sequences, KV heads, group, dim] and pages [pages, rows, KV heads, dim]")
    sequences, kv_heads, group, dim = q.shape
    if 0 in q.shape or 0 in k_pages.shape:
        raise ValueError(f"empty q {tuple(q.shape)} or pages {tuple(k_pages.shape)}")
    if tuple(k_pages.shape[2:]) != (kv_heads, dim):
        raise ValueError(f"pages of {tuple(k_pages.shape[2:])} heads and dimensions, q of {(kv_heads, dim)}")
    if (k_new is None) != (v_new is None) or (k_new is not None and not tuple(k_new.shape) == tuple(v_new.shape) == (sequences, kv_heads, dim)):
        raise ValueError("k_new and v_new come together, [sequences, KV heads, dim]")
    if table.dim() != 2 or table.shape[0] != sequences or tuple(lengths.shape) != (sequences,):
        raise ValueError("paged_attention wants table [sequences, pages of the longest] and lengths [sequences]")
    if table.dtype != torch.int64 or lengths.dtype != torch.int64:
        raise TypeError("table and lengths must be int64")
    if sinks is not None and tuple(sinks.shape) != (kv_heads * group,):
        raise ValueError("sinks must hold one value per query head")
    if any(x is not None and x.dtype != q.dtype for x in (k_pages, v_pages, k_new, v_new, sinks)):
        raise TypeError("q, pages, new rows and sinks must have one dtype")
    if window < 0 or first < 0:
        raise ValueError("window and first must not be negative")


@torch.library.custom_op("chroma_amd::paged_chunk_attention", mutates_args=())
def paged_chunk_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, k_new: Optional[Tensor], v_new: Optional[Tensor], table: Tensor, lengths: Tensor,
                          starts: Tensor, sinks: Optional[Tensor], scale: float, window: int = 0, first: int = 0) -> Tensor:
    """Attention of a chunk of new tokens of every sequence over its cached keys and values, which lie in pages.

    q [T, KV, G, D], rows starts[b] .. starts[b + 1] - 1 of it sequence b's tokens; starts [S + 1] int64, ascending within
    [0, T] (entries outside count as the nearest bound, a range that descends as empty). k_new and v_new [T, KV, D] are the tokens' own
    rows, token i of a sequence at position lengths[b] + i; or None, where they are the last of the lengths[b] cached rows. A
    token sees the rows up to its position, cached or new, less what ``window`` leaves out. Pages, table [S, N], lengths, sinks,
    window and first are as for ``paged_attention``. A token that sees no row and a row of q that no sequence has get zeros. Scores
    and sums are float's, the result is rounded once; compiled with bfloat16, a weight meets the values as two bfloat16 halves
    (within 2^-16 of it), or, where there are 64 query heads of a KV head or more for each sequence, rounded to bfloat16."""
    _check_chunk(q, k_pages, v_pages, k_new, v_new, table, lengths, starts, sinks, window, first)
    tokens, kv_heads, group, dim = q.shape
    pages, rows = k_pages.shape[:2]
    out = torch.zeros_like(q)
    for b in range(len(lengths)):
        begin = min(max(int(starts[b]), 0), tokens)
        end = min(max(int(starts[b + 1]), begin), tokens)
        if begin == end:
            continue
        length = min(max(int(lengths[b]), 0), table.shape[1] * rows)
        j = torch.arange(length, device=q.device)
        page = table[b][j // rows]
        held = (page >= 0) & (page < pages)
        j, place = j[held], (page * rows + j % rows)[held]
        k, v = (x.reshape(-1, kv_heads, dim)[place].float() for x in (k_pages, v_pages))
        now = torch.arange(end - begin, device=q.device) + length
        if k_new is None:
            now = now - (end - begin)
        else:
            k, v, j = torch.cat([k, k_new[begin:end].float()]), torch.cat([v, v_new[begin:end].float()]), torch.cat([j, now])
        seen = j[None, :] <= now[:, None]
        if window:
            seen = seen & ((j[None, :] > now[:, None] - window) | (j[None, :] < first))
        # head by head: [tokens, G, rows]
        for h in range(kv_heads):
            scores = torch.mm((q[begin:end, h].float() * scale).reshape(-1, dim), k[:, h].t().contiguous()).reshape(end - begin, group, -1)
            scores = scores.masked_fill(~seen[:, None, :], -math.inf)
            joined = scores
            if sinks is not None:
                joined = torch.cat([scores, sinks.float()[h * group : (h + 1) * group].reshape(1, group, 1).expand(end - begin, -1, -1)], -1)
            top = joined.amax(-1, keepdim=True) if joined.shape[-1] else joined.new_zeros(end - begin, group, 1)
            top = torch.where(top == -math.inf, 0.0, top)
            weights, total = torch.exp(scores - top), torch.exp(joined - top).sum(-1, keepdim=True)
            mixed = torch.mm(weights.reshape(-1, weights.shape[-1]), v[:, h]).reshape(end - begin, group, dim)
            out[begin:end, h] = torch.where(total == 0, 0.0, mixed / total).to(q.dtype)
    return out


@paged_chunk_attention.register_fake
def _(q, k_pages, v_pages, k_new, v_new, table, lengths, starts, sinks, scale, window=0, first=0):
    _check_chunk(q, k_pages, v_pages, k_new, v_new, table, lengths, starts, sinks, window, first)
    return q.new_empty(q.shape)


def _check_chunk(q, k_pages, v_pages, k_new, v_new, table, lengths, starts, sinks, window, first) -> None:
    if q.dim() != 4 or table.dim() != 2 or lengths.dim() != 1 or len(lengths) == 0:
        raise ValueError("paged_chunk_attention wants q [tokens, KV heads, group, dim], table [sequences, pages of the longest] and lengths [sequences]")
    tokens, kv_heads, _, dim = q.shape
    if (k_new is None) != (v_new is None) or (k_new is not None and not tuple(k_new.shape) == tuple(v_new.shape) == (tokens, kv_heads, dim)):
        raise ValueError("k_new and v_new come together, [tokens, KV heads, dim]")
    # the rest is as for a token of each sequence
    _check(q.new_empty((len(lengths), *q.shape[1:])) if tokens else q, k_pages, v_pages, None, None, table, lengths, sinks, window, first)
    if k_new is not None and (k_new.dtype != q.dtype or v_new.dtype != q.dtype):
        raise TypeError("q, pages, new rows and sinks must have one dtype")
    if tuple(starts.shape) != (len(lengths) + 1,):
        raise ValueError("starts must hold one entry more than lengths")
    if starts.dtype != torch.int64:
        raise TypeError("starts must be int64")


__all__ = ["paged_attention", "paged_chunk_attention"]
