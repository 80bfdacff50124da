"""One step of speculative decoding over a paged compressed cache.

No counterpart in the reference, which generates one token at a time without a cache (patch.py:81).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from .paged_cache import MAX_DRAFT, TurboQuantPagedCache

__all__ = ["speculative_step"]


@torch.no_grad()
def speculative_step(model, cache: TurboQuantPagedCache, tokens: torch.Tensor, parents=None,
                     draft_probs: torch.Tensor | None = None, uniforms: torch.Tensor | None = None,
                     temperature: float = 1.0) -> list[list[int]]:
    """Run a patched model over drafted tokens of the cache's active sequences, verify them, keep the
    accepted path in the cache, and return each sequence's emitted tokens: the accepted drafted
    ones and one more, which is the next step's root.

    tokens int64 [B, T] (T up to 64): tokens[:, 0] is the last emitted token, whose keys and values
    are not cached yet; the others were drafted after it.  parents (a list, [T] or [B, T]) gives
    their tree in index order: node 0 is -1, another node's parent an earlier node, -2 pads a smaller
    tree; None is a chain.  draft_probs [B, T - 1, V]: a chain's tokens were drawn from these
    distributions (`turboquant_pytorch.verify_drafts`).  temperature 0 takes the likeliest token
    instead of drawing.  uniforms float32 [B, T] default to torch.rand."""
    from turboquant_pytorch import verify_drafts

    if tokens.dim() != 2 or not 1 <= tokens.shape[1] <= MAX_DRAFT:
        raise ValueError(f"tokens must be [B, 1 to {MAX_DRAFT}], got {tuple(tokens.shape)}")
    if temperature < 0:
        raise ValueError(f"temperature must not be negative, got {temperature}")
    B, T = tokens.shape
    dev = tokens.device
    tree, depth = _depths(parents, B, T)
    if tree is not None:
        if draft_probs is not None:
            raise ValueError("tokens drawn from a draft distribution form a chain; a tree (parents) holds chosen candidates")
        tree = tree.to(dev)
    lengths = cache.lengths()
    if len(lengths) != B:
        raise ValueError(f"tokens of {B} sequences for {len(lengths)} active ones (cache.use)")
    positions = (torch.tensor(lengths)[:, None] + depth).to(dev)
    with cache.draft(tree):
        logits = model(input_ids=tokens, position_ids=positions, past_key_values=cache, use_cache=True).logits.float()
    if temperature == 0:
        probs = F.one_hot(logits.argmax(-1), logits.shape[-1]).float()
    else:
        probs = torch.softmax(logits / temperature, -1)
    if uniforms is None:
        uniforms = torch.rand(B, T, device=dev)
    if draft_probs is not None:
        draft_probs = draft_probs.to(probs.dtype)
    path, count, nxt = verify_drafts(tokens, probs, uniforms, parents=tree, draft_probs=draft_probs)
    # one transfer, and before anything is kept: a step that cannot be finished leaves the cache as it was
    got = torch.cat([path, count[:, None], nxt[:, None]], 1).tolist()
    if any(row[-1] < 0 for row in got):
        cache.drop_draft()
        raise RuntimeError("the model's distribution after the accepted tokens has no positive probability")
    cache.accept(path, count)
    drafted = tokens.tolist()
    return [[drafted[b][i] for i in row[1:row[T]]] + [row[T + 1]] for b, row in enumerate(got)]


def _depths(parents, B: int, T: int):
    """Checked parents as an int32 tensor (None: a chain), and every node's depth [1 or B, T]."""
    if parents is None:
        return None, torch.arange(T)[None]
    tree = torch.as_tensor(parents, dtype=torch.int32).cpu()
    if tuple(tree.shape) not in ((T,), (B, T)):
        raise ValueError(f"parents must be [{T}] or [{B}, {T}], got {tuple(tree.shape)}")
    rows = tree.reshape(-1, T).tolist()
    depth = []
    for row in rows:
        d = [0] * T
        for i, p in enumerate(row):
            if (p != -1) if i == 0 else not (p == -2 or 0 <= p < i):
                raise ValueError(f"node {i} has parent {p}: node 0 is the root (-1), another node's parent an earlier "
                                 "node, or -2 for none")
            d[i] = d[p] + 1 if p >= 0 else 0
        depth.append(d)
    return tree, torch.tensor(depth)
