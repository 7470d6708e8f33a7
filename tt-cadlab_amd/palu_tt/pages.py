"""The page table of a server over paged caches: rows forked, ended, cut and grown, pools compacted.

The paged ops (fused.palu_sdpa_decode, flash_decode, flash_prefill, paged_update_cache, paged_fill_cache) read a page table
[B, max_pages] int32 and page pools [n_pages, n_groups, page_size, width], one table for the K and V pools of all layers.
``PagePools`` holds the pools of a server and changes the table, with the copies of pages in all pools that this asks for, on
the device and without a synchronisation. The reference has no counterpart (its caches are contiguous).

A page is in use where one of a row's first ceil(length / page_size) table entries names it. Nothing else is kept: no
reference counts and no free list, so a row is freed by giving it the length 0. Rows may share pages that they only read
(a common prefix, the siblings of a beam); ``update`` gives every row its own copy of the page that it writes next.
"""
import ctypes
from typing import Optional, Sequence, Tuple

import torch

from palu_tt import _native
from palu_tt.cache import LatentCache


def _ints(t, name: str, shape, device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.is_floating_point() or tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{name} must be an integer tensor {list(shape)}, got {tuple(getattr(t, 'shape', ()))}")
    if t.device != device or t.dtype != torch.int32:
        t = t.to(device=device, dtype=torch.int32)
    return t.contiguous()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    ends = lambda t: (t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
    (a0, a1), (b0, b1) = ends(a), ends(b)
    return a0 < b1 and b0 < a1


class PagePools:
    """The page pools that share a page table: row-major [n_pages, n_groups, page_size, width] bf16 tensors or LatentCache
    pools (of any group counts and widths)."""

    def __init__(self, pools: Sequence):
        if not pools:
            raise RuntimeError("PagePools needs at least one pool")
        self.pools = list(pools)
        self._take()

    def _look(self) -> None:
        """Takes the pools anew if one is not what it was: a LatentCache's ``data`` may be another tensor than at the last
        call, and a tensor may have been given other memory or another size."""
        for cache, store, place, size in self._seen:
            if (cache is not None and cache.data is not store) or store.data_ptr() != place or store.numel() != size:
                self._take()
                return

    def _take(self) -> None:
        """Checks the pools as they are now and takes their storage, which is held for as long as its address is."""
        stores = [p.data if isinstance(p, LatentCache) else p for p in self.pools]
        for p, s in zip(self.pools, stores):
            if not (isinstance(s, torch.Tensor) and len(p.shape) == 4 and s.is_cuda and s.dtype == torch.bfloat16 and
                    s.is_contiguous() and s.data_ptr() % 16 == 0 and s.numel()):
                raise RuntimeError("a pool is a contiguous, 16-byte aligned bf16 [n_pages, n_groups, page_size, width] tensor, "
                                   "not empty, on the GPU or a LatentCache")
            if (p.shape[0], p.shape[2], s.device) != (self.pools[0].shape[0], self.pools[0].shape[2], stores[0].device):
                raise RuntimeError("pools must agree in pages, page size and device: "
                                   f"{tuple(p.shape)}, {tuple(self.pools[0].shape)}")
        if any(_overlap(a, b) for i, a in enumerate(stores) for b in stores[:i]):
            raise RuntimeError("pools must not overlap")
        self.n_pages, self.page_size = int(self.pools[0].shape[0]), int(self.pools[0].shape[2])
        self.device = stores[0].device
        n = len(stores)
        self._ptrs = (ctypes.c_void_p * n)(*[s.data_ptr() for s in stores])
        self._bytes = (ctypes.c_longlong * n)(*[s.numel() * 2 // self.n_pages for s in stores])
        self._seen = [(p if isinstance(p, LatentCache) else None, s, s.data_ptr(), s.numel()) for p, s in zip(self.pools, stores)]
        self._stores = stores

    def _args(self, page_table, lengths):
        self._look()
        if not (isinstance(page_table, torch.Tensor) and page_table.dim() == 2):
            raise RuntimeError("page_table must be [B, max_pages] int32")
        B, slots = page_table.shape
        return (_ints(page_table, "page_table", (B, slots), self.device), _ints(lengths, "lengths", (B,), self.device), B, slots)

    def _workspace(self, B: int, workspace: Optional[torch.Tensor]):
        need = _native.load().palu_pages_workspace_bytes(B, self.n_pages)
        if workspace is None:
            return torch.empty(need, dtype=torch.uint8, device=self.device), need
        _native.workspace_bytes(workspace, need, self.device)
        return workspace, need

    def update(self, page_table, lengths, *, parents=None, new_lengths=None, out=None,
               workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(page_table, lengths) in which row b is a copy of row parents[b] as it was (None: of itself; an index outside the batch,
        such as -1: of an empty row), cut or grown to new_lengths[b] positions (None: as long as its parent). So a step of
        every row is new_lengths = lengths + 1, a fork parents[b] = a with b a free row, beam search parents = the beams
        picked, the end of a request new_lengths[b] = 0, the rejection of drafted tokens a shorter length.

        Whole pages are shared; the page that a row writes next is its own: the first row that would write it keeps it, unless
        another holds it whole, the others get a copy in every pool. New pages are the lowest free ones. Where the pool has
        no more, the returned length of a row is what its pages hold: compare with what was asked for, and go on from the new table
        (pages that it does not name may hold other rows' copies already, so the old one is done with). All integers are
        int32 [B] and [B, max_pages] on the device; entries past a row's pages are -1. out: (page_table, lengths) to
        write, memory of their own. Do not share a workspace (uint8, palu_pages_workspace_bytes) between calls that may overlap."""
        pt, ln, B, slots = self._args(page_table, lengths)
        ws, need = self._workspace(B, workspace) if B else (None, 0)
        par = None if parents is None else _ints(parents, "parents", (B,), self.device)
        new = None if new_lengths is None else _ints(new_lengths, "new_lengths", (B,), self.device)
        if out is None:
            out = torch.empty_like(pt), torch.empty_like(ln)
        else:
            for t, like, name in zip(out, (pt, ln), ("page_table", "lengths")):
                if t.shape != like.shape or t.dtype != torch.int32 or t.device != self.device or not t.is_contiguous():
                    raise RuntimeError(f"out: {name} must be a contiguous int32 {list(like.shape)} tensor on {self.device}")
                if any(i is not None and _overlap(t, i) for i in (pt, ln, par, new, workspace, *self._stores)):
                    raise RuntimeError(f"out: {name} must be memory of its own")
            if _overlap(*out):
                raise RuntimeError("out: page_table and lengths must not overlap")
        if B:
            _native.launch("pages_update", self.device, pt.data_ptr(), ln.data_ptr(), _native.ptr(par), _native.ptr(new),
                           out[0].data_ptr(), out[1].data_ptr(), self._ptrs, self._bytes, len(self.pools), B, self.n_pages,
                           self.page_size, slots, ws.data_ptr(), need)
        return out[0], out[1]

    def compact(self, page_table, lengths, *, workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(page_table, n): the n pages in use moved to pages 0 .. n - 1 of every pool, those at n or above in order to the free
        ones below n, and the table over the new places (entries past a row's pages -1); n is an int32 [1] tensor."""
        pt, ln, B, slots = self._args(page_table, lengths)
        if B < 1:
            raise RuntimeError("page_table must have at least one row")
        table = torch.empty_like(pt)
        n = torch.empty(1, dtype=torch.int32, device=self.device)
        ws, need = self._workspace(B, workspace)
        _native.launch("pages_compact", self.device, pt.data_ptr(), ln.data_ptr(), table.data_ptr(), n.data_ptr(), self._ptrs,
                       self._bytes, len(self.pools), B, self.n_pages, self.page_size, slots, ws.data_ptr(), need)
        return table, n
