"""Block-sparse decode: attention over the cache blocks that a cheap score selects (``nvk_block_index_*``, ``nvk_sparse_decode*``).

What ``Attention::paged_attention`` (``include/core/attention.hpp:82-159``) computes, over the first, the last and the best-scored
blocks of each sequence and kv-head.  A :class:`BlockIndex` beside a :class:`PagedKVPool` keeps the bounds of every
block's keys that the scores are made of; :meth:`BlockIndex.update` brings it up to date behind an append."""
from __future__ import annotations

import ctypes as C
from typing import Tuple

import numpy as np

from . import _capi
from .kv_pool import PagedKVPool, _address, _f32, _i32, _ptr


class BlockIndex:
    def __init__(self, pool: PagedKVPool):
        h = C.c_void_p()
        _capi.check(_capi.lib.nvk_block_index_create(pool.handle, C.byref(h)))
        self._h, self.pool = h, pool  # keeps the pool alive

    def close(self) -> None:
        if getattr(self, "_h", None) and _capi.lib is not None:  # (None: the interpreter is going down)
            _capi.lib.nvk_block_index_destroy(self._h)
            self._h = None

    __del__ = close

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def handle(self) -> C.c_void_p:
        if not self._h:
            raise RuntimeError("index is closed")
        self.pool.handle  # (a closed pool's memory is gone)
        return self._h

    def layer_ptr(self, layer: int) -> int:
        """Device address of a layer's bounds, [num_blocks, n_kv_heads, 2 (least, largest), head_dim] fp32."""
        p = C.c_void_p()
        _capi.check(_capi.lib.nvk_block_index_layer_ptr(self.handle, int(layer), C.byref(p)))
        return int(p.value)

    @property
    def workspace_generation(self) -> int:
        return int(_capi.lib.nvk_block_index_workspace_generation(self.handle))

    def reserve_workspace(self, num_seqs: int, n_heads: int, max_ctx: int, top_blocks: int) -> None:
        """Room for later decode calls of up to this shape (needed before capturing them)."""
        _capi.check(_capi.lib.nvk_block_index_reserve_workspace(self.handle, int(num_seqs), int(n_heads), int(max_ctx), int(top_blocks)))

    def update(self, layer: int, block_tables, starts, ctx_lens) -> None:
        """Brings the blocks of tokens [starts[s], ctx_lens[s]) up to date, host arrays."""
        tabs, st, ctx = _i32(block_tables), _i32(starts).reshape(-1), _i32(ctx_lens).reshape(-1)
        if tabs.ndim != 2 or st.size != tabs.shape[0] or ctx.size != tabs.shape[0]:
            raise ValueError("block_tables must be [num_seqs, max_blocks], starts and ctx_lens [num_seqs]")
        _capi.check(_capi.lib.nvk_block_index_update(self.handle, int(layer), ctx.size, _ptr(tabs), tabs.shape[1], _ptr(st), _ptr(ctx), 0,
                                                     _capi.PTR_HOST, None))

    def update_device(self, layer: int, num_seqs: int, block_tables_dev, max_blocks: int, starts_dev, ctx_lens_dev, max_new: int,
                      stream=None) -> None:
        _capi.check(_capi.lib.nvk_block_index_update(self.handle, int(layer), int(num_seqs), _address(block_tables_dev), int(max_blocks),
                                                     _address(starts_dev), _address(ctx_lens_dev), int(max_new), _capi.PTR_DEVICE,
                                                     _address(stream)))


def sparse_decode(index: BlockIndex, layer: int, q, block_tables, ctx_lens, top_blocks: int, first_blocks: int = 1,
                  last_blocks: int = 1) -> Tuple[np.ndarray, np.ndarray]:
    """One layer-call from host arrays: (out [num_seqs, n_heads, head_dim], the blocks read [num_seqs, n_kv_heads, top_blocks],
    ascending and filled up with -1)."""
    tabs, ctx, qh = _i32(block_tables), _i32(ctx_lens).reshape(-1), _f32(q)
    if tabs.ndim != 2 or ctx.size != tabs.shape[0]:
        raise ValueError("block_tables must be [num_seqs, max_blocks] and ctx_lens [num_seqs]")
    if qh.ndim != 3 or qh.shape[0] != ctx.size or qh.shape[2] != index.pool.head_dim:
        raise ValueError("q must be [num_seqs, n_heads, head_dim]")
    out = np.empty_like(qh)
    got = np.empty((ctx.size, index.pool.n_kv_heads, max(int(top_blocks), 0)), np.int32)
    _capi.check(_capi.lib.nvk_sparse_decode(index.handle, int(layer), ctx.size, int(qh.shape[1]), _ptr(qh), _ptr(tabs), tabs.shape[1],
                                            _ptr(ctx), int(top_blocks), int(first_blocks), int(last_blocks), _ptr(out), _ptr(got)))
    return out, got


def sparse_decode_device(index: BlockIndex, layer: int, num_seqs: int, n_heads: int, q_dev, block_tables_dev, max_blocks: int,
                         ctx_lens_dev, max_ctx: int, top_blocks: int, first_blocks: int, last_blocks: int, out_dev, selected_dev=None,
                         stream=None) -> None:
    """Asynchronous layer-call on device pointers; selected_dev (int32, may be None) receives the blocks read."""
    _capi.check(_capi.lib.nvk_sparse_decode_device(index.handle, int(layer), int(num_seqs), int(n_heads), _address(q_dev),
                                                   _address(block_tables_dev), int(max_blocks), _address(ctx_lens_dev), int(max_ctx),
                                                   int(top_blocks), int(first_blocks), int(last_blocks), _address(out_dev),
                                                   _address(selected_dev), _address(stream)))
