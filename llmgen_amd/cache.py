"""Other forms of the paged KV cache (include/llmgen_cache.h): pools of 4-bit pages, the scratch of the attention over
them and over sliding windows, and page copies in every layer's pools.

The kernels themselves are called as every other one of the library, through :func:`~llmgen_amd._lib.lib`
(``hip_store_kv4``, ``hip_attn_decode_kv4``, ...), or by the attention node for a layer that has such a form
(:class:`~llmgen_amd.attention.PagedAttentionManager`).
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from ._lib import lib


def kv4_pool(num_blocks: int, nkv: int, block_size: int, hd: int = 128, device="cuda") -> torch.Tensor:
    """A pool of 4-bit pages, [num_blocks, bytes a page] uint8: all values 0."""
    nbytes = lib().hip_kv4_block_bytes(nkv, hd, block_size)
    if nbytes == 0 or num_blocks <= 0:
        raise ValueError(f"no 4-bit pages of {nkv} heads of {hd} values and {block_size} tokens (heads have 128 values)")
    return torch.zeros((num_blocks, nbytes), dtype=torch.uint8, device=device)


def attn_work(device="cuda") -> torch.Tensor:
    """Scratch for the attention calls of one stream, ready for use there: it is cleared before this returns, as that
    stream need not be torch's current one (while that is capturing, the graph clears it)."""
    work = torch.zeros(lib().hip_attn_work_bytes(), dtype=torch.uint8, device=device)
    if work.is_cuda and not torch.cuda.is_current_stream_capturing():
        torch.cuda.current_stream(work.device).synchronize()
    return work


class BlockCopies:
    """Copies of pages inside a list of pools that share their block ids (the K and V pools of every layer)."""

    def __init__(self, pools):
        pools = list(pools)
        if not pools:
            raise ValueError("no pools")
        first = pools[0]
        for p in pools:
            if not p.is_cuda or not p.is_contiguous() or p.device != first.device:
                raise ValueError("pools must be contiguous tensors of one device")
            if p.dim() < 2 or p.shape[0] != first.shape[0] or self._page_bytes(p) != self._page_bytes(first):
                raise ValueError("pools must have the same number of pages and the same page size")
            if self._page_bytes(p) % 16 or p.data_ptr() % 16:
                raise ValueError("pages must be multiples of 16 bytes, and pools 16-byte aligned")
        self.pools, self.num_blocks, self.page_bytes = pools, first.shape[0], self._page_bytes(first)
        self._ptrs = (ctypes.c_void_p * len(pools))(*[p.data_ptr() for p in pools])
        self._call = lib().hip_copy_blocks

    @staticmethod
    def _page_bytes(pool) -> int:
        return pool[0].numel() * pool.element_size()

    @staticmethod
    def _ids(ids):
        if getattr(ids, "dtype", None) != np.int32:
            a = np.asarray(ids)
            if a.size and (a.dtype.kind not in "iu" or a.min() < -(1 << 31) or a.max() >= 1 << 31):
                raise ValueError("page ids are whole numbers of 32 bits")
            ids = a.astype(np.int32)
        return np.ascontiguousarray(ids)

    def run(self, src, dst) -> None:
        """Page src[i] onto page dst[i] in every pool; ids as :meth:`Blocks.compact <llmgen_amd.host.Blocks.compact>`
        returns them (int32 arrays) or any sequences of whole numbers.  The pairs have no order."""
        src, dst = self._ids(src), self._ids(dst)
        if src.shape != dst.shape or src.ndim != 1:
            raise ValueError("one destination for each source")
        self._call(self._ptrs, len(self.pools), self.page_bytes, self.num_blocks, src.__array_interface__["data"][0],
                   dst.__array_interface__["data"][0], src.size)
