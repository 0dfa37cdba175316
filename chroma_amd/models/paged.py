"""Batched steps of the GPT-OSS workload over one paged key-value cache.

``export_paged(model, sequences, pages, page_rows, span)`` exports one step that consumes a token of each of
``sequences`` sequences: token ids [sequences] int64, positions [sequences] fp32, keys and values [layers,
pages, page_rows, kv_heads, head_dim], the page table [sequences, span] int64 (row j of a sequence is row
j % page_rows of page table[j // page_rows]) and the sequences' cached rows [sequences] int64. It returns the
logits [sequences, vocab] and the new key and value rows [layers, sequences, kv_heads, head_dim]: the
``export_cached`` graph with a batch of sequences in place of a prompt's steps, and
``chroma_amd.ops.paged_attention`` in place of attention over one contiguous cache.

``export_paged_chunk(model, tokens, sequences, pages, page_rows, span)`` exports a step in which every sequence takes any
number of tokens, ``tokens`` in all: token ids and positions [tokens], the cache, table and lengths as above, where each
sequence's tokens begin [sequences + 1] int64 and which row its last one is [sequences] int64. It returns the logits after
those [sequences, vocab] and the new rows [layers, tokens, kv_heads, head_dim]. (No counterparts in the reference, whose
decoder holds one sequence.)
"""

from __future__ import annotations

from typing import List, Tuple

import torch
from torch import Tensor, nn

from chroma_amd.models.gpt_oss import Transformer
from chroma_amd.ops import paged_attention, paged_chunk_attention


class PagedTransformer(nn.Module):
    def __init__(self, model: Transformer) -> None:
        super().__init__()
        self.model = model

    def forward(self, tokens: Tensor, positions: Tensor, keys: Tensor, values: Tensor, table: Tensor, lengths: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
        x = self.model.embedding(tokens)
        new_keys: List[Tensor] = []
        new_values: List[Tensor] = []
        pages = keys.shape[1:]
        for layer, block in enumerate(self.model.block):
            attention = block.attn
            q, k, v = attention.project(x, positions)
            new_keys.append(k.unsqueeze(0))
            new_values.append(v.unsqueeze(0))
            attended = paged_attention(q, keys[layer : layer + 1].reshape(pages), values[layer : layer + 1].reshape(pages), k, v, table, lengths,
                                       attention.sinks, attention.sm_scale, attention.sliding_window)
            x = block.mlp(x + attention.out(attended.reshape(tokens.shape[0], -1)))
        return self.model.unembedding(self.model.norm(x)), torch.cat(new_keys, dim=0), torch.cat(new_values, dim=0)


class ChunkedTransformer(nn.Module):
    def __init__(self, model: Transformer) -> None:
        super().__init__()
        self.model = model

    def forward(self, tokens: Tensor, positions: Tensor, keys: Tensor, values: Tensor, table: Tensor, lengths: Tensor, starts: Tensor,
                last: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
        x = self.model.embedding(tokens)
        new_keys: List[Tensor] = []
        new_values: List[Tensor] = []
        pages = keys.shape[1:]
        for layer, block in enumerate(self.model.block):
            attention = block.attn
            q, k, v = attention.project(x, positions)
            new_keys.append(k.unsqueeze(0))
            new_values.append(v.unsqueeze(0))
            attended = paged_chunk_attention(q, keys[layer : layer + 1].reshape(pages), values[layer : layer + 1].reshape(pages), k, v, table, lengths,
                                             starts, attention.sinks, attention.sm_scale, attention.sliding_window)
            x = block.mlp(x + attention.out(attended.reshape(tokens.shape[0], -1)))
        return self.model.unembedding(self.model.norm(x[last])), torch.cat(new_keys, dim=0), torch.cat(new_values, dim=0)


def export_paged(model: Transformer, sequences: int, pages: int, page_rows: int, span: int) -> torch.export.ExportedProgram:
    if min(sequences, pages, page_rows, span) < 1:
        raise ValueError(f"{sequences} sequences, {pages} pages of {page_rows} rows, {span} pages a sequence")
    examples = (torch.zeros(sequences, dtype=torch.int64), torch.zeros(sequences, dtype=torch.float32),
                *_cache_examples(model, sequences, pages, page_rows, span))
    with torch.no_grad():
        return torch.export.export(PagedTransformer(model).eval(), examples)


def export_paged_chunk(model: Transformer, tokens: int, sequences: int, pages: int, page_rows: int, span: int) -> torch.export.ExportedProgram:
    if min(tokens, sequences, pages, page_rows, span) < 1:
        raise ValueError(f"{tokens} tokens, {sequences} sequences, {pages} pages of {page_rows} rows, {span} pages a sequence")
    examples = (torch.zeros(tokens, dtype=torch.int64), torch.zeros(tokens, dtype=torch.float32),
                *_cache_examples(model, sequences, pages, page_rows, span), torch.zeros(sequences + 1, dtype=torch.int64),
                torch.zeros(sequences, dtype=torch.int64))
    with torch.no_grad():
        return torch.export.export(ChunkedTransformer(model).eval(), examples)


def _cache_examples(model: Transformer, sequences: int, pages: int, page_rows: int, span: int) -> Tuple[Tensor, ...]:
    """Keys, values, table and lengths."""
    first = model.block[0].attn
    cache_shape = (len(model.block), pages, page_rows, first.num_key_value_heads, first.head_dim)
    dtype = first.qkv.weight.dtype
    return (torch.zeros(cache_shape, dtype=dtype), torch.zeros(cache_shape, dtype=dtype), torch.zeros(sequences, span, dtype=torch.int64),
            torch.zeros(sequences, dtype=torch.int64))
