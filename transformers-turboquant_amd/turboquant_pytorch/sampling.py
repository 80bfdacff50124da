"""Sampling from logits by temperature, top-k, top-p and min-p, from given uniforms.

Tokens are ranked by falling logit, equal ones by index.  With the weights ``w = exp((l - max l) / temperature)``:
top_k keeps the first top_k in rank; top_p, of those, the ones whose predecessors weigh less than top_p of
their total, and the first one in any case; min_p, of those, the ones that weigh min_p of the likeliest or more.  A setting
is a number, or a tensor with one value per row (float32, top_k int32, on the logits' device): top_k 0, top_p 1 and
min_p 0 filter nothing, temperature 0 keeps the likeliest token alone.  A logit that is -inf or NaN is never
kept.  No counterpart in the reference, which leaves generation to transformers.
"""

from __future__ import annotations

import torch

from ._ops import ops

__all__ = ["filter_probs", "sample_tokens"]


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """A token of every row: int64 [...] from logits [..., V] and uniforms float32 [...] in [0, 1).

    The first token x, in index order, at which the kept tokens' weights up to x exceed the uniform times their
    total; -1 for a row without a logit above -inf.  Weights are float64 (3e-13), sums float64 or integers of 2^-62 of
    the total: what is kept and drawn is that of the exact distribution, unless a border lies within 2^-40 of the total of a
    token's edge (2^-37 for more than 2^20 tokens) or min_p within 3e-13 of a weight, and a call gives the same tokens every
    time."""
    if uniforms.shape != logits.shape[:-1]:
        raise ValueError(f"uniforms must be {list(logits.shape[:-1])}, one per row of the logits, got {list(uniforms.shape)}")
    settings = _settings(logits, temperature, top_k, top_p, min_p)
    if logits.dim() == 2:
        return ops().sample_tokens(_rows(logits), uniforms.contiguous(), *settings)
    return ops().sample_tokens(_rows(logits), uniforms.reshape(-1).contiguous(), *settings).reshape(logits.shape[:-1])


def filter_probs(logits: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """The distributions that `sample_tokens` draws from, float32 [..., V]: zero where a token is not kept (a whole
    row of zeros where no logit is above -inf).  `verify_drafts` takes them as target or draft probabilities."""
    settings = _settings(logits, temperature, top_k, top_p, min_p)
    probs = ops().filter_probs(_rows(logits), *settings)
    return probs if logits.dim() == 2 else probs.reshape(logits.shape)


def _rows(logits):
    """Logits as [N, V], copied where they are strided along the vocabulary."""
    rows = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    return rows if rows.stride(1) == 1 else rows.contiguous()


def _settings(logits, temperature, top_k, top_p, min_p):
    """Each setting as (values of the rows or None, number)."""
    out = []
    for name, x, off in (("temperature", temperature, 1.0), ("top_k", top_k, 0), ("top_p", top_p, 1.0), ("min_p", min_p, 0.0)):
        if isinstance(x, torch.Tensor):
            if x.shape != logits.shape[:-1]:
                raise ValueError(f"{name} must be a number or {list(logits.shape[:-1])}, one per row of the logits, got {list(x.shape)}")
            out += [x.reshape(-1).contiguous(), off]
        else:
            out += [None, x]
    return out
