"""What a patched model checks before a forward over a TurboQuantPagedCache.

A paged cache decides by itself what a token sees, so what the decoder would have told its attention layers in a
mask has to be looked at before the mask is made.  No counterpart in the reference, which
disables the KV cache (patch.py:81).
"""

from __future__ import annotations

import inspect

import torch

from .paged_cache import TurboQuantPagedCache

__all__ = ["PagedCall", "attention_window"]


def attention_window(original) -> int | None:
    """Positions that a transformers attention module's token sees, itself among them (None: all before it)."""
    if hasattr(original, "sliding_window"):
        return original.sliding_window
    cfg = getattr(original, "config", None)
    types = getattr(cfg, "layer_types", None)
    layer = getattr(original, "layer_idx", None)
    if getattr(cfg, "use_sliding_window", True) is False:
        return None
    if types is not None and layer is not None and types[layer] != "sliding_attention":
        return None
    return getattr(cfg, "sliding_window", None)


def check_window(window: int | None, cached: int, new: int) -> None:
    """Refuse `new` tokens behind `cached` positions where a token would be past its window: pages are attended whole."""
    if window is not None and cached + new > window:
        raise ValueError(f"a paged cache attends to every cached position: {cached} cached and {new} new tokens do not fit the "
                         f"model's sliding window of {window}")


class PagedCall:
    """Forward pre-hook of a patched model's decoder; does nothing with other caches."""

    def __init__(self, names: list[str], window: int | None):
        self.names = names  # of forward's parameters, in order
        self.window = window  # the smallest of the attention layers'

    @classmethod
    def install(cls, model) -> None:
        decoder = getattr(model, "base_model", model)  # the module that makes masks and positions
        for key, hook in list(decoder._forward_pre_hooks.items()):
            if isinstance(hook, cls):  # patched before
                del decoder._forward_pre_hooks[key]
                decoder._forward_pre_hooks_with_kwargs.pop(key, None)
        windows = [w for m in decoder.modules() if hasattr(m, "causal_mode")
                   for w in [getattr(m, "sliding_window", None)] if w is not None]
        decoder.register_forward_pre_hook(cls(list(inspect.signature(decoder.forward).parameters), min(windows, default=None)),
                                          with_kwargs=True)

    def __call__(self, module, args, kwargs):
        given = {**dict(zip(self.names, args)), **kwargs}
        cache = given.get("past_key_values")
        if not isinstance(cache, TurboQuantPagedCache):
            return None
        tokens = given.get("input_ids")
        if tokens is None:
            tokens = given.get("inputs_embeds")
        if tokens is None:
            return None
        check_window(self.window, cache.get_seq_length(), tokens.shape[1])
        mask = given.get("attention_mask")
        # over a cache that masks by itself the decoder reduces a 2-D mask to its first columns, and to None
        # where those are ones: padding is only seen here (masks of other forms reach the layers, which refuse them)
        if isinstance(mask, torch.Tensor) and mask.dim() == 2 and not bool(mask.all()):
            raise ValueError("a paged cache masks by itself and takes no padding: run prompts unpadded, in batches of one length")
        return self._place(cache, tokens, mask, given.get("position_ids"), args, kwargs)

    def _place(self, cache, tokens, mask, positions, args, kwargs):
        """The arguments with the tokens' positions where the decoder would make wrong ones: from the longest
        sequence, one after another."""
        B, T = tokens.shape[:2]
        lengths, tree = cache.lengths(), cache.draft_parents
        unequal = len(set(lengths)) > 1
        if len(lengths) not in (0, B) or (tree is not None and tuple(tree.shape) not in ((T,), (B, T))):
            return None  # the cache refuses the step
        if unequal and isinstance(mask, torch.Tensor) and mask.dim() == 2 and mask.shape[1] > T:
            # generate() counts positions along such a mask
            raise ValueError(f"a mask of {mask.shape[1]} positions for sequences of {sorted(set(lengths))} cached ones and {T} new "
                             "tokens: pass none, and position_ids or none")
        if positions is not None:
            if unequal and positions.shape[0] != B:
                raise ValueError(f"position_ids {tuple(positions.shape)} for {B} sequences of unequal length")
            return None
        if not unequal and tree is None or "position_ids" not in self.names:
            return None
        behind = torch.arange(T)[None] if tree is None else tree_depths(tree)
        positions = (torch.tensor(lengths or [0] * B)[:, None] + behind).to(tokens.device)
        at = self.names.index("position_ids")
        if at < len(args):
            return (*args[:at], positions, *args[at + 1:]), kwargs
        return args, {**kwargs, "position_ids": positions}


def tree_depths(parents: torch.Tensor) -> torch.Tensor:
    """How far behind the cached text each node of the trees [T] or [B, T] stands: [1 or B, T] (0 without a place)."""
    rows = []
    for row in parents.reshape(-1, parents.shape[-1]).tolist():
        depth = []
        for i, p in enumerate(row):
            depth.append(depth[p] + 1 if 0 <= p < i else 0)
        rows.append(depth)
    return torch.tensor(rows)
