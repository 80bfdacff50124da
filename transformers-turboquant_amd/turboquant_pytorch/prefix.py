"""Attention of sequences that share a long prefix, over pages of a compressed cache.

Sequences that were forked from one prompt have the prompt's pages in common.  Tree attention reads them for every
sequence; the operators here for up to 32 query columns of a group at a time: the shared positions against the queries of
several sequences, each sequence's own positions against its own, and both joined.  No counterpart in the
reference, which keeps no cache between steps (patch.py:81).
"""

from __future__ import annotations

import torch

from ._ops import ops
from .compressors import TurboQuantCompressorMSE, TurboQuantCompressorV2
from .drafts import _both_tables, _tree_args
from .pages import PagePool

__all__ = ["append_prefix_attention", "prefix_attention", "prefix_groups"]


def prefix_groups(sizes, shared, device="cuda") -> torch.Tensor:
    """Groups of a batch as `prefix_attention` takes them, int32 [sum(sizes), 2]: the first sizes[0] sequences share
    their first shared[0] positions, the next sizes[1] theirs, and so on (0: nothing is shared)."""
    sizes, shared = [int(n) for n in sizes], [int(n) for n in shared]
    if len(sizes) != len(shared):
        raise ValueError(f"{len(sizes)} group sizes and {len(shared)} numbers of shared positions")
    if any(n < 1 for n in sizes) or any(not 0 <= n < 2 ** 31 for n in shared):
        raise ValueError(f"groups have at least one sequence and share 0 positions or more, got sizes {sizes} and shared {shared}")
    rows = [[i, n] for i, (size, n) in enumerate(zip(sizes, shared)) for _ in range(size)]
    return torch.tensor(rows, dtype=torch.int32).reshape(-1, 2).to(device)


def prefix_attention(queries: torch.Tensor, key_compressor: TurboQuantCompressorV2, val_compressor: TurboQuantCompressorMSE,
                     pool: PagePool, layer: int, block_table: torch.Tensor, lengths: torch.Tensor, groups: torch.Tensor,
                     parents: torch.Tensor | None = None, scale: float | None = None,
                     out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """`tree_attention` ([B, T, Hq, D] from queries [B, Hq, T, D]) of sequences that share their first positions.

    groups int32 [B, 2] on the GPU: sequences that follow one another with the same id ``groups[b, 0] >= 0`` and
    the same ``groups[b, 1]`` have the rows of positions ``[0, groups[b, 1])`` in common (`prefix_groups` makes it); an id of
    -1 or 0 shared positions: alone.  The table row of every sequence of a group that has a length holds pages with the
    shared rows; through which of these table rows they are read depends on the shape.  Whole slabs of 32 shared positions are
    read for several sequences together (64 at most: a batch is cut at every 64th sequence).  A sequence shorter than what it
    shares gets zeros, as one without room for its tokens does."""
    tk, tv = _both_tables(key_compressor, val_compressor, queries.device)
    args = _tree_args(tk, tv, queries.shape[-1], key_compressor, val_compressor, pool, layer, block_table, lengths, parents,
                      scale, out_dtype or queries.dtype, (groups,))
    return ops().prefix_attend(queries, tk.pi_split, tk.s_eff16, *args)


def append_prefix_attention(k: torch.Tensor, v: torch.Tensor, queries: torch.Tensor, key_compressor, val_compressor,
                            pool: PagePool, layer: int, block_table: torch.Tensor, lengths: torch.Tensor, groups: torch.Tensor,
                            parents: torch.Tensor | None = None, scale: float | None = None,
                            out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """`append_tree_attention` of sequences that share their first positions: the T new tokens' keys and values k, v
    [B, Hkv, T, D] into their pages (positions ``lengths[b] + i``, none of them shared), then prefix_attention."""
    tk, tv = _both_tables(key_compressor, val_compressor, queries.device)
    args = _tree_args(tk, tv, queries.shape[-1], key_compressor, val_compressor, pool, layer, block_table, lengths, parents,
                      scale, out_dtype or queries.dtype, (groups,))
    return ops().prefix_page_attend(k, v, queries, tk.pi_split, tk.seff_split, tk.cent32, tk.bounds32, tv.pi_split,
                                    tv.bounds32, tk.s_eff16, *args)
