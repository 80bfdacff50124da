"""Paged compressed KV cache: sequences of unequal length over one pool of pages.

Where :class:`TurboQuantCache` holds capacity planes of one length for a whole batch, a
``TurboQuantPagedCache`` keeps each sequence as a list of pages of a :class:`PagePool`:

* sequences come and go (``add``, ``free``), and ``use`` picks which of them the next forward's batch
  rows are;
* a fork (``fork``, beam search's ``reorder_cache``) shares its pages with the sequence it came from; a
  shared page is copied before a position in it is written; with ``shared_prefix=True`` attention reads the pages
  that active sequences next to one another share for several of them together;
* drafted tokens (``draft``) are appended as a tree that is not part of the text yet; after verification
  ``accept`` keeps one path of it, moved down behind the cached positions, and frees the rest.

The compressed rows and the estimator are those of the compressors; what a token sees is decided
by the cache (every cached position, then causally or along the tree), so it takes no attention
mask: prompts are not padded but run sequence by sequence, or in batches of one length.
No counterpart in the reference, which disables the KV cache (patch.py:81).

    cache = TurboQuantPagedCache(num_pages=4096, num_layers=model.config.num_hidden_layers)
    out = model.generate(ids, past_key_values=cache, use_cache=True)
"""

from __future__ import annotations

import contextlib
import math

import torch
from transformers.cache_utils import Cache
from turboquant_pytorch.drafts import append_tree_attention
from turboquant_pytorch.prefix import append_prefix_attention

__all__ = ["TurboQuantPagedCache"]

MAX_DRAFT = 64  # nodes of a tree; longer appends are prompts


def _best_runs(common: list[int]) -> list[tuple[int, int]]:
    """len(common) + 1 sequences cut into runs (size, pages that all of it share) that save the most pages of
    reading, (size - 1) * shared each; common[i]: pages that i and i + 1 share.  Where these are not all the same, runs
    are of 64 at most, as the operator reads them."""
    n = len(common) + 1
    if len(set(common)) <= 1:
        return [(n, common[0])] if common and common[0] else [(1, 0)] * n
    best = [(0, 0, 0)]  # of the first j sequences: pages saved, the last run's begin and what it shares
    for j in range(1, n + 1):
        top, least = (best[j - 1][0], j - 1, 0), None
        for i in range(j - 2, max(-1, j - 65), -1):
            least = common[i] if least is None else min(least, common[i])
            if not least:
                break
            saved = best[i][0] + (j - i - 1) * least
            if saved > top[0]:
                top = (saved, i, least)
        best.append(top)
    runs, j = [], n
    while j:
        _, i, shared = best[j]
        runs.append((j - i, shared))
        j = i
    return runs[::-1]


class _Sequence:
    __slots__ = ("pages", "length")

    def __init__(self, pages=(), length: int = 0):
        self.pages = list(pages)
        self.length = length


class TurboQuantPagedCache(Cache):
    """A transformers ``Cache`` over pages, for models patched by ``apply_turboquant`` on the GPU."""

    def __init__(self, num_pages: int, num_layers: int, page_size: int = 64, shared_prefix: bool = False):
        super().__init__(layers=[])
        if num_pages < 1 or num_layers < 1:
            raise ValueError("a paged cache needs at least one page and one layer")
        if page_size < 32 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 32 on, got {page_size}")
        self.num_pages, self.num_layers, self.page_size = num_pages, num_layers, page_size
        self.shared_prefix = shared_prefix
        self.pool = None  # made by the first append, which knows heads, head_dim and bits
        self._free = list(range(num_pages - 1, -1, -1))
        self._refs = [0] * num_pages
        self._seqs: dict[int, _Sequence] = {}
        self._next_id = 0
        self._active: list[int] = []
        self._codec: dict[int, tuple] = {}  # per layer: bits and seeds of the compressors that filled it
        self._tree = None  # inside draft(): (parents,)
        self._drafted = False  # the step's rows are drafted tokens that accept() may keep
        self._written: set[int] = set()  # layers of the step under way that hold its rows
        self._step = 0  # tokens of the step under way
        self._device_state = None  # (block table, lengths) of the active sequences; None: to be made
        self._groups = None  # of the active sequences that share pages, on the device (None: attended alone)
        self._made: list[int] = []  # sequences that the step under way made
        self._made_pool = False  # it made the pool, too

    # ------------------------------------------------------------------ sequences
    def add(self, n: int = 1) -> list[int]:
        """Ids of n new, empty sequences (not yet active)."""
        ids = list(range(self._next_id, self._next_id + n))
        self._next_id += n
        for i in ids:
            self._seqs[i] = _Sequence()
        return ids

    def fork(self, seq: int, n: int = 1) -> list[int]:
        """Ids of n new sequences with the contents of `seq`, sharing its pages."""
        self._abandon()
        src = self._seq(seq)
        ids = self.add(n)
        for i in ids:
            self._seqs[i] = self._share(src)
        return ids

    def free(self, *seqs: int) -> None:
        """Forget sequences; pages that no other sequence shares are free again."""
        seqs = tuple(dict.fromkeys(seqs))
        for i in seqs:
            self._seq(i)
        if any(i in self._active for i in seqs):
            self._abandon()
        for i in seqs:
            self._drop(self._seqs.pop(i), 0)
        self._active = [i for i in self._active if i not in seqs]

    def use(self, seqs) -> None:
        """The sequences that the batch rows of the next forwards are, in order."""
        seqs = list(seqs)
        for i in seqs:
            self._seq(i)
        if len(set(seqs)) != len(seqs):
            raise ValueError(f"a sequence can be active once, got {seqs}")
        self._abandon()
        self._active = seqs

    @property
    def active(self) -> list[int]:
        return list(self._active)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def lengths(self, seqs=None) -> list[int]:
        """Cached positions of the given (default: the active) sequences."""
        return [self._seq(i).length for i in (self._active if seqs is None else seqs)]

    def _seq(self, i: int) -> _Sequence:
        if i not in self._seqs:
            raise ValueError(f"no sequence {i} in this cache")
        return self._seqs[i]

    def _share(self, src: _Sequence) -> _Sequence:
        for p in src.pages:
            self._refs[p] += 1
        return _Sequence(src.pages, src.length)

    def _drop(self, seq: _Sequence, keep: int) -> None:
        """Give back the pages behind the first `keep`."""
        for p in seq.pages[keep:]:
            self._refs[p] -= 1
            if not self._refs[p]:
                self._free.append(p)
        del seq.pages[keep:]

    def _pages_for(self, positions: int) -> int:
        return -(-positions // self.page_size)

    # ------------------------------------------------------------------ transformers' Cache
    def __len__(self) -> int:
        return self.num_layers

    def __repr__(self) -> str:
        return (f"{type(self).__name__}({len(self._seqs)} sequences, {self.num_pages - len(self._free)} of "
                f"{self.num_pages} pages of {self.page_size})")

    def get_seq_length(self, layer_idx: int = 0) -> int:
        """Length of the longest active sequence."""
        return max(self.lengths(), default=0)

    def get_query_offset(self, layer_idx: int = 0) -> int:
        return self.get_seq_length()

    def get_mask_sizes(self, query_length: int, layer_idx: int = 0) -> tuple[int, int]:
        # the cache masks by itself: no mask over cached positions is wanted, and models build
        # none where the keys of a mask would be the queries
        return query_length, 0

    def get_max_cache_shape(self, layer_idx: int = 0) -> int:
        return -1

    @property
    def is_compileable(self) -> bool:
        return False

    @property
    def is_initialized(self) -> bool:
        return self.pool is not None

    @property
    def is_sliding(self) -> list[bool]:
        return [False] * self.num_layers

    def update(self, *args, **kwargs):
        raise NotImplementedError("TurboQuantPagedCache holds compressed pages; it is filled by attention modules "
                                  "patched with apply_turboquant, not by uncompressed key/value updates")

    def reset(self) -> None:
        """Forget every sequence."""
        self._abandon()
        self.free(*list(self._seqs))

    def crop(self, tokens_to_remove: int) -> None:
        """Drop the last -tokens_to_remove positions of the active sequences (a positive value is the
        length to keep)."""
        self._abandon()
        for i in self._active:
            seq = self._seqs[i]
            keep = tokens_to_remove if tokens_to_remove > 0 else seq.length + tokens_to_remove
            seq.length = max(0, min(seq.length, keep))
            self._drop(seq, self._pages_for(seq.length))

    def reorder_cache(self, beam_idx: torch.Tensor) -> None:
        """Active sequence i becomes a fork of what active sequence beam_idx[i] was."""
        self._select(beam_idx.tolist())

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        self._select(indices.tolist())

    def batch_repeat_interleave(self, repeats: int) -> None:
        self._select([i for i in range(len(self._active)) for _ in range(repeats)])

    def _select(self, rows: list[int]) -> None:
        if any(not 0 <= r < len(self._active) for r in rows):
            raise ValueError(f"rows {rows} of a batch of {len(self._active)}")
        self._abandon()
        old = self._active
        new = [self._share(self._seqs[old[r]]) for r in rows]
        for i in old:
            self._drop(self._seqs[i], 0)
        ids = old[:len(rows)] + self.add(max(0, len(rows) - len(old)))
        for i in old[len(rows):]:
            del self._seqs[i]
        for i, seq in zip(ids, new):
            self._seqs[i] = seq
        self._active = ids

    def nbytes(self) -> int:
        """Bytes of the pages in use."""
        return 0 if self.pool is None else self.pool.nbytes() // self.num_pages * (self.num_pages - len(self._free))

    # ------------------------------------------------------------------ drafted tokens
    @contextlib.contextmanager
    def draft(self, parents=None):
        """The forward inside appends drafted tokens of the active sequences: up to 64 per sequence, as the
        tree that parents gives (int32 [T] or [B, T] on the GPU, see `tree_attention`; None: a
        chain).  They are not part of the text until accept(); anything else done with the cache
        drops them."""
        if self._tree is not None:
            raise RuntimeError("draft() inside draft()")
        self._abandon()
        if parents is not None and (parents.dtype != torch.int32 or parents.dim() not in (1, 2)):
            raise ValueError(f"parents must be int32 [T] or [B, T], got {parents.dtype} {tuple(parents.shape)}")
        self._tree = (parents,)
        try:
            yield self
            self._drafted = len(self._written) == self.num_layers
        finally:
            self._tree = None
            if not self._drafted:
                self._abandon()

    @property
    def draft_parents(self) -> torch.Tensor | None:
        """The tree of the draft under way (None: no draft, or a chain)."""
        return self._tree[0] if self._tree else None

    def accept(self, path: torch.Tensor, count: torch.Tensor) -> list[int]:
        """Keep the first count[b] nodes of path[b] (`verify_drafts`) of the drafted tokens, in every
        layer; the others are dropped and their pages freed.  Returns the new lengths."""
        if not self._drafted:
            raise RuntimeError("accept() needs drafted tokens: run the model inside cache.draft() first")
        if tuple(path.shape) != (len(self._active), self._step):
            raise ValueError(f"path must be [{len(self._active)}, {self._step}], got {tuple(path.shape)}")
        table, lengths = self._device_state
        new = self.pool.keep(table, lengths, path, count).tolist()
        for i, n in zip(self._active, new):
            self._seqs[i].length = n
        self._abandon()
        return new

    def drop_draft(self) -> None:
        """Forget drafted tokens that are not accepted, and give their pages back."""
        if self._drafted:
            self._abandon()

    def _abandon(self) -> None:
        """Drop a step under way (drafted tokens, a forward that did not finish): its rows are behind
        the lengths and get overwritten; its pages are given back."""
        for i in self._active:
            seq = self._seqs[i]
            self._drop(seq, self._pages_for(seq.length))
        self._written.clear()
        self._step = 0
        self._drafted = False
        self._device_state = self._groups = None
        self._made, self._made_pool = [], False

    def _undo(self) -> None:
        """Drop a step that failed, with the sequences and the pool that it made."""
        made, made_pool = self._made, self._made_pool
        self._abandon()
        for i in made:
            self._drop(self._seqs.pop(i), 0)
        self._active = [i for i in self._active if i not in made]
        if made_pool:
            self.pool = None

    # ------------------------------------------------------------------ compressed storage
    def append_attend(self, layer_idx: int, key_compressor, val_compressor, k: torch.Tensor, v: torch.Tensor,
                      q: torch.Tensor, scale: float | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """Compress one layer's new keys and values [B, Hkv, T, D] into the active sequences' pages and
        attend from q [B, Hq, T, D] over everything cached and the new tokens (causally, or along the
        drafted tree).  Returns [B, T, Hq, D].

        The first layer of a forward reserves its pages (copying shared ones first); when every
        layer has written, the tokens are part of the text, unless they are drafted."""
        if k.device.type != "cuda":
            raise ValueError("TurboQuantPagedCache runs on the GPU")
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            raise ValueError(f"layer {layer_idx} of a cache of {self.num_layers} layers")
        B, _, T, D = k.shape
        if T < 1:
            raise ValueError("no tokens to append")
        bits = val_compressor.bits
        fast = T <= MAX_DRAFT and D in (64, 128) and 2 <= bits <= 4
        if self._tree is not None and not fast:
            raise ValueError(f"drafted tokens: at most {MAX_DRAFT} per sequence, head_dim 64 or 128 and 2 to 4 bits; got "
                             f"{T} tokens, head_dim {D}, {bits} bits")
        self._check_codec(layer_idx, key_compressor, val_compressor)
        self._begin(layer_idx, k, bits)
        table, lengths = self._device_state
        try:
            if fast and self._groups is not None:
                out = append_prefix_attention(k, v, q, key_compressor, val_compressor, self.pool, layer_idx, table, lengths,
                                              self._groups, self.draft_parents, scale, out_dtype)
            elif fast:
                out = append_tree_attention(k, v, q, key_compressor, val_compressor, self.pool, layer_idx, table, lengths,
                                            self.draft_parents, scale, out_dtype)
            else:
                out = self._attend_prompt(layer_idx, key_compressor, val_compressor, k, v, q, table, lengths, scale, out_dtype)
        except BaseException:
            if not self._written:  # else the next forward finds a step that is not finished
                self._undo()
            raise
        self._finish(layer_idx)
        return out

    def _finish(self, layer_idx: int) -> None:
        self._written.add(layer_idx)
        if len(self._written) == self.num_layers and self._tree is None:
            for i in self._active:
                self._seqs[i].length += self._step
            table, lengths = self._device_state
            self._device_state = (table, lengths + self._step)  # stands until a page is added
            self._written.clear()
            self._step = 0
            self._made, self._made_pool = [], False

    def _check_codec(self, layer_idx, key_compressor, val_compressor) -> None:
        if val_compressor.bits != key_compressor.mse_bits + 1:
            raise ValueError(f"a paged cache holds keys and values of one bit width, got {key_compressor.mse_bits + 1} and "
                             f"{val_compressor.bits}")
        codec = (key_compressor.bits, val_compressor.bits, getattr(key_compressor, "seed", None),
                 getattr(val_compressor, "seed", None))
        held = self._codec.get(layer_idx)
        if held is not None and held != codec and any(s.length for s in self._seqs.values()):
            raise ValueError(f"layer {layer_idx} holds positions compressed with other settings (cached, new): {held}, {codec}")
        self._codec[layer_idx] = codec

    def _begin(self, layer_idx: int, k: torch.Tensor, bits: int) -> None:
        from turboquant_pytorch.pages import PagePool

        B, H, T, D = k.shape
        done = len(self._written)
        if layer_idx in self._written and done < self.num_layers:
            self._undo()
            raise RuntimeError(f"the forward before this one wrote {done} of the cache's {self.num_layers} layers; its "
                               "tokens were dropped")
        if self._active or self._seqs:
            if B != len(self._active):
                raise ValueError(f"a batch of {B} for {len(self._active)} active sequences (cache.use)")
        if self.pool is None:
            self.pool = PagePool(self.num_pages, self.page_size, H, D, bits, self.num_layers, k.device)
            self._made_pool = True
        pool = self.pool
        if (H, D, bits) != (pool.num_kv_heads, pool.head_dim, pool.bits) or k.device != pool.device:
            raise ValueError(f"the cache's pages hold {pool.num_kv_heads} heads of {pool.head_dim} at {pool.bits} bits on "
                             f"{pool.device}, got {H} of {D} at {bits} bits on {k.device}")
        if layer_idx in self._written:  # a draft that was not accepted
            self._abandon()
        if self._written:
            if T != self._step:
                raise ValueError(f"layer {layer_idx} appends {T} tokens in a step of {self._step}")
            return
        try:
            if not self._active and not self._seqs:
                self._active = self._made = self.add(B)
            parents = self.draft_parents
            if parents is not None and tuple(parents.shape) not in ((T,), (B, T)):
                raise ValueError(f"parents {tuple(parents.shape)} for {B} sequences of {T} drafted tokens")
            self._reserve(T)
        except BaseException:
            self._undo()
            raise
        self._step = T

    def _reserve(self, T: int) -> None:
        """Pages for T more positions of every active sequence, none of them shared."""
        P, seqs = self.page_size, [self._seqs[i] for i in self._active]
        refs = dict.fromkeys((p for s in seqs for p in s.pages[s.length // P:]))
        refs = {p: self._refs[p] for p in refs}
        plan, need = [], 0
        for s in seqs:  # which pages are copied, how many are new
            shared = []
            for at in range(s.length // P, len(s.pages)):
                if refs[s.pages[at]] > 1:
                    refs[s.pages[at]] -= 1
                    shared.append(at)
            fresh = self._pages_for(s.length + T) - len(s.pages)
            plan.append((shared, max(0, fresh)))
            need += len(shared) + max(0, fresh)
        if need > len(self._free):
            raise RuntimeError(f"the paged cache is full: {need} more pages of {P} positions wanted, {len(self._free)} of "
                               f"{self.num_pages} free")
        src, dst = [], []
        for s, (shared, fresh) in zip(seqs, plan):
            for at in shared:
                new = self._take()
                if at * P < s.length:  # the page holds cached positions
                    src.append(s.pages[at])
                    dst.append(new)
                self._refs[s.pages[at]] -= 1
                s.pages[at] = new
            s.pages.extend(self._take() for _ in range(fresh))
        if self._device_state is not None and not need:
            return
        dev = self.pool.device
        width = max(len(s.pages) for s in seqs)
        groups = self._shared(seqs) if self.shared_prefix else [(-1, 0)] * len(seqs)
        state = torch.tensor([s.pages + [-1] * (width - len(s.pages)) + [s.length, *g] for s, g in zip(seqs, groups)],
                             dtype=torch.int32)
        state = state.to(dev)  # one copy for all
        self._device_state = (state[:, :-3].contiguous(), state[:, -3].contiguous())
        self._groups = state[:, -2:].contiguous() if any(n for _, n in groups) else None
        if src:
            pairs = torch.tensor([src, dst], dtype=torch.int32).to(dev)
            self.pool.copy(pairs[0], pairs[1])

    def _shared(self, seqs) -> list[tuple[int, int]]:
        """(id, shared positions) of each sequence, as `prefix_attention` takes them."""
        common = []  # leading pages that a sequence and the next one have in common
        for a, b in zip(seqs, seqs[1:]):
            lo, hi = 0, min(len(a.pages), len(b.pages))
            while lo < hi:  # behind the first page that differs, all do
                mid = (lo + hi) // 2
                lo, hi = (mid + 1, hi) if a.pages[mid] == b.pages[mid] else (lo, mid)
            common.append(lo)
        runs = _best_runs(common)
        # Worth it from a fifth of all pages on: 16 sequences with 8192 positions of their own, 32/8 heads, behind 64 shared
        # ones 46.5 us against 42 apart, 1024 (a tenth saved) 46 and 44, 4096 (0.3) 50 and 53; 2 sequences of 12k, 4096
        # of them shared (a sixth), 30 and 29.5.
        if 5 * sum((size - 1) * n for size, n in runs) < sum(len(s.pages) for s in seqs):
            runs = [(1, 0)] * len(seqs)
        return [(i, n * self.page_size) for i, (size, n) in enumerate(runs) for _ in range(size)]

    def _take(self) -> int:
        p = self._free.pop()
        self._refs[p] = 1
        return p

    def _attend_prompt(self, layer_idx, key_compressor, val_compressor, k, v, q, table, lengths, scale, out_dtype):
        """Many tokens, or rows that tree attention does not take: attention over contiguous rows, the
        new ones alone for a fresh batch, else gathered out of the pages, per length."""
        from turboquant_pytorch.fused import compressed_attention

        B, H, T, D = k.shape
        ck, cv = key_compressor.compress(k), val_compressor.compress(v)
        self.pool.write(layer_idx, ck, cv, table, lengths)
        scale = 1.0 / math.sqrt(D) if scale is None else scale
        lens = self.lengths()
        if not any(lens):
            return compressed_attention(q, key_compressor, val_compressor, ck, cv, causal=True, scale=scale,
                                        out_dtype=out_dtype)
        out = torch.empty((B, T) + (q.shape[1], D), dtype=out_dtype or q.dtype, device=q.device)
        for n in sorted(set(lens)):
            rows = torch.tensor([b for b in range(B) if lens[b] == n], device=q.device)
            ak, av = self.pool.read(layer_idx, table.index_select(0, rows), lengths.index_select(0, rows) + T, n + T)
            out[rows] = compressed_attention(q.index_select(0, rows), key_compressor, val_compressor, ak, av, causal=True,
                                             scale=scale, out_dtype=out.dtype)
        return out
