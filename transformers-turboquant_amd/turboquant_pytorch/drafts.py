"""Drafted tokens: attention of a token tree over pages of a compressed cache, and verification.

Node i of a sequence's tree was drafted as a child of ``parents[i] < i``; -1 continues the cached text.
Without parents the tokens form a chain.  No counterpart in the reference, which generates one
token at a time without a cache (patch.py:81).
"""

from __future__ import annotations

import math

import torch

from ._ops import ops
from .compressors import TurboQuantCompressorMSE, TurboQuantCompressorV2, _scaled_tables, _tables
from .pages import PagePool

__all__ = ["append_tree_attention", "tree_attention", "tree_attention_from_prepared", "verify_drafts"]


def tree_attention(queries: torch.Tensor, key_compressor: TurboQuantCompressorV2,
                   val_compressor: TurboQuantCompressorMSE, pool: PagePool, layer: int, block_table: torch.Tensor,
                   lengths: torch.Tensor, parents: torch.Tensor | None = None, scale: float | None = None,
                   out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Attention output [B, T, Hq, D] of T drafted tokens per sequence (T = 1: a decoding step).

    queries [B, Hq, T, D] on the GPU, T up to 64.  ``lengths[b]`` positions are cached, and the drafted tokens'
    own rows stand at ``lengths[b] + i`` (``pool.write``).  Node i sees the cached positions, its
    ancestors and itself.  parents int32 [T] (one tree for all sequences) or [B, T]; a value that is
    neither -1 nor an earlier node leaves the node without a place: its output is zero and no node
    sees it (padding of smaller trees).  A sequence with a negative length, or whose table has no room for
    lengths[b] + T positions, gets zeros.  head_dim 64 or 128, 2 to 4 bits.
    """
    tk, tv = _both_tables(key_compressor, val_compressor, queries.device)
    return ops().tree_attend(queries, tk.pi_split, tk.s_eff16,
                             *_tree_args(tk, tv, queries.shape[-1], key_compressor, val_compressor, pool, layer, block_table,
                                         lengths, parents, scale, out_dtype or queries.dtype))


def tree_attention_from_prepared(q_rot: torch.Tensor, q_proj: torch.Tensor, key_compressor, val_compressor,
                                 pool: PagePool, layer: int, block_table: torch.Tensor, lengths: torch.Tensor,
                                 parents: torch.Tensor | None = None, scale: float | None = None,
                                 out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """tree_attention on queries already prepared by ``key_compressor.prepare_queries``."""
    tk, tv = _both_tables(key_compressor, val_compressor, q_rot.device)
    return ops().tree_attention(q_rot, q_proj,
                                *_tree_args(tk, tv, q_rot.shape[-1], key_compressor, val_compressor, pool, layer, block_table,
                                            lengths, parents, scale, out_dtype))


def append_tree_attention(k: torch.Tensor, v: torch.Tensor, queries: torch.Tensor, key_compressor, val_compressor,
                          pool: PagePool, layer: int, block_table: torch.Tensor, lengths: torch.Tensor,
                          parents: torch.Tensor | None = None, scale: float | None = None,
                          out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """One layer's decoding or speculation step: the T new tokens' keys and values k, v [B, Hkv, T, D]
    compressed into their pages (positions ``lengths[b] + i``) and the queries prepared in one launch,
    then tree_attention.  A new row whose page is missing is not written.  k, v and queries of different
    types run as the separate operators (compress, ``pool.write``, tree_attention), each in its own type."""
    tk, tv = _both_tables(key_compressor, val_compressor, queries.device)
    return ops().page_attend(k, v, queries, tk.pi_split, tk.seff_split, tk.cent32, tk.bounds32, tv.pi_split, tv.bounds32,
                             tk.s_eff16, *_tree_args(tk, tv, queries.shape[-1], key_compressor, val_compressor, pool, layer,
                                                     block_table, lengths, parents, scale, out_dtype or queries.dtype))


def _both_tables(key_compressor, val_compressor, dev):
    return _tables(key_compressor, dev, with_qjl=True), _tables(val_compressor, dev, with_qjl=False)


def _tree_args(tk, tv, D, key_compressor, val_compressor, pool, layer, block_table, lengths, parents, scale, out_dtype):
    if key_compressor.S.shape[0] != D:
        raise ValueError("tree attention needs a square QJL matrix")
    if val_compressor.bits != key_compressor.mse_bits + 1:
        raise ValueError(f"tree attention needs keys and values of one bit width, got {key_compressor.mse_bits + 1} "
                         f"and {val_compressor.bits}")
    vcent, vpit = _scaled_tables(val_compressor, tv)
    kcodes, ksigns, krn, kvn, vcodes, vvn = pool._layer[layer]
    if out_dtype not in (torch.float32, torch.float16, torch.bfloat16):
        out_dtype = torch.float32
    return (kcodes, ksigns, krn, kvn, tk.cent16, val_compressor.bits, vcodes, vvn, vcent, vpit, block_table,
            lengths, parents, math.sqrt(math.pi / 2) / key_compressor.S.shape[0],
            float(scale if scale is not None else 1.0 / math.sqrt(D)), out_dtype)


def verify_drafts(tokens: torch.Tensor, target_probs: torch.Tensor, uniforms: torch.Tensor,
                  parents: torch.Tensor | None = None, draft_probs: torch.Tensor | None = None
                  ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accept drafted tokens against the target's probabilities: (path, count, next_token).

    tokens int64 [B, T]: node 0 is the last emitted token, the others were drafted (T up to 64; T = 1
    only draws the next token).  target_probs [B, T, V]: the target's distribution after each
    node.  uniforms float32 [B, T] in [0, 1): ``[:, i]`` decides node i, ``[:, 0]`` draws the next token.

    Without draft_probs the drafted tokens are chosen candidates in a chain, or in the tree that
    parents (int32 [T] or [B, T]) gives; a node's children are tried in index order, each against
    what the earlier ones left.  draft_probs [B, T - 1, V], of target_probs' type: the drafted tokens
    form a chain, token i + 1 drawn from ``draft_probs[:, i]``; token x is accepted iff u q(x) < p(x),
    and a rejection leaves (p - q)+.  Either way the emitted tokens are distributed as the target's.

    path int32 [B, T]: the accepted nodes from the root on, then -1; count int32 [B]: how many;
    next_token int64 [B]: drawn from what is left after the last of them (-1 where a row has no
    positive probability).
    """
    return ops().verify_drafts(tokens, target_probs, uniforms, parents, draft_probs)
