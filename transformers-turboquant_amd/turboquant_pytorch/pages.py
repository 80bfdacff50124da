"""Pages of a compressed KV cache on the GPU.

A :class:`PagePool` holds, for every layer, the packed planes of ``num_pages`` pages of
``page_size`` positions: key codes, QJL signs, residual and vector norms, value codes and norms, laid out
``[layers, num_pages, Hkv, page_size, ...]``.  Which pages a sequence has is the caller's: position j of
sequence b is row ``j % page_size`` of page ``block_table[b, j // page_size]`` in every layer.
Sequences of unequal length share a pool, a forked sequence shares its pages with the one it
came from, and pages of a finished one serve the next.

Tables, lengths and page indices are int32 tensors on the pool's device; kernels check them
there, and leave out rows whose page is outside the pool (-1: no page).  No counterpart in the
reference, which keeps no cache between steps (patch.py:81).
"""

from __future__ import annotations

import torch

from ._ops import ops

__all__ = ["PagePool"]

_NAMES = ("kcodes", "ksigns", "krn", "kvn", "vcodes", "vvn")


class PagePool:
    """Compressed pages of `layers` attention layers, and the operators that move their rows."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, bits: int, layers: int = 1,
                 device="cuda"):
        if bits < 2 or bits > 8:
            raise ValueError(f"bits must be 2 to 8, got {bits}")
        if head_dim % 8 or not 8 <= head_dim <= 256:
            raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {head_dim}")
        if min(num_pages, num_kv_heads, layers) < 1:
            raise ValueError("a pool needs at least one page, head and layer")
        shape = (layers, num_pages, num_kv_heads, page_size)
        widths = ((head_dim * (bits - 1) + 7) // 8, head_dim // 8, 0, 0, (head_dim * bits + 7) // 8, 0)
        self._set(*(torch.zeros(*shape, w, dtype=torch.uint8, device=device) if w
                    else torch.zeros(shape, dtype=torch.float16, device=device) for w in widths))

    @classmethod
    def over(cls, kcodes: torch.Tensor, ksigns: torch.Tensor, krn: torch.Tensor, kvn: torch.Tensor,
             vcodes: torch.Tensor, vvn: torch.Tensor) -> "PagePool":
        """A pool over existing planes ``[layers, num_pages, Hkv, page_size, (bytes)]``."""
        pool = cls.__new__(cls)
        pool._set(kcodes, ksigns, krn, kvn, vcodes, vvn)
        return pool

    def _set(self, *planes: torch.Tensor) -> None:
        norms = planes[3]
        if norms.dim() != 4:
            raise ValueError(f"norm planes must be [layers, num_pages, Hkv, page_size], got {tuple(norms.shape)}")
        self.layers, self.num_pages, self.num_kv_heads, self.page_size = norms.shape
        if self.page_size < 32 or self.page_size & (self.page_size - 1):
            raise ValueError(f"page_size must be a power of two from 32 on, got {self.page_size}")
        self.head_dim = planes[1].shape[-1] * 8
        self.bits = planes[4].shape[-1] * 8 // self.head_dim
        self.device = norms.device
        self._planes = planes
        self._layer = [tuple(p[i] for p in planes) for i in range(self.layers)]

    def planes(self, layer: int) -> dict[str, torch.Tensor]:
        """The planes of one layer, by name (views of the pool)."""
        return dict(zip(_NAMES, self._layer[layer]))

    def write(self, layer: int, compressed_k: dict, compressed_v: dict, block_table: torch.Tensor,
              start: torch.Tensor) -> None:
        """Compressed rows [B, Hkv, S, D] (the compressors' packed dicts, contiguous) to positions
        ``start[b] + s`` of a layer.  A negative start writes nothing for that sequence."""
        if "packed_key_indices" not in compressed_k or "packed_indices" not in compressed_v:
            raise ValueError("PagePool.write takes the packed (GPU) formats")
        B, H, S, D = compressed_k["shape"]
        if (H, D) != (self.num_kv_heads, self.head_dim) or compressed_v["shape"] != compressed_k["shape"]:
            raise ValueError(f"rows of {compressed_k['shape']} keys and {compressed_v['shape']} values do not go into "
                             f"pages of {self.num_kv_heads} heads of {self.head_dim}")
        if B != block_table.shape[0]:
            raise ValueError(f"block_table has {block_table.shape[0]} rows for {B} sequences")
        ops().page_write(compressed_k["packed_key_indices"], compressed_k["packed_qjl_signs"],
                         compressed_k["residual_norm"], compressed_k["vec_norms"], compressed_v["packed_indices"],
                         compressed_v["vec_norms"], *self._layer[layer], block_table, start, S)

    def read(self, layer: int, block_table: torch.Tensor, lengths: torch.Tensor, S: int) -> tuple[dict, dict]:
        """The first S positions of each sequence as contiguous packed dicts [B, Hkv, S, D];
        positions from ``lengths[b]`` on are zeros."""
        kc, ks, rn, kn, vc, vn = ops().page_read(*self._layer[layer], block_table, lengths, S)
        shape = (block_table.shape[0], self.num_kv_heads, S, self.head_dim)
        return ({"packed_key_indices": kc, "packed_qjl_signs": ks, "residual_norm": rn, "vec_norms": kn, "shape": shape},
                {"packed_indices": vc, "vec_norms": vn, "shape": shape})

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page ``dst[i]`` := page ``src[i]`` in every layer.  No page may be both a source and a
        target, and none a target twice."""
        ops().page_copy(*self._planes, src, dst)

    def keep(self, block_table: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor,
             count: torch.Tensor) -> torch.Tensor:
        """Move an accepted path of drafted tokens behind the cached positions, in every layer:
        position ``lengths[b] + path[b, i]`` to ``lengths[b] + i`` for ``i < count[b]``.  Returns the new
        lengths, ``lengths + count``."""
        return ops().page_keep(*self._planes, block_table, lengths, path, count)

    def nbytes(self) -> int:
        return sum(p.numel() * p.element_size() for p in self._planes)
