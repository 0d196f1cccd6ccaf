"""Mx4KVPool: a paged KV cache held in 4 bits a value, and attention over it.

The cache of ``PagedKVPool`` (``include/core/model.hpp:94-97``) with every value as sign * {0, .5, 1, 1.5, 2, 3, 4, 6} * 2^e, one e for
each 32 channels of a row: 17/32 byte instead of 4.  Rows come in through :func:`norm_rope_append` /
:func:`norm_rope_append_device`; block tables, positions and lengths are those of the fp32 pool."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import numpy as np

from . import _capi
from .kv_pool import _address, _f32, _i32, _ptr


class Mx4KVPool:
    def __init__(self, n_layers: int, num_blocks: int, block_size: int, n_kv_heads: int, head_dim: int, device: int = 0):
        handle = C.c_void_p()
        _capi.check(_capi.lib.nvk_mx4_pool_create(int(n_layers), int(num_blocks), int(block_size), int(n_kv_heads), int(head_dim),
                                                  int(device), C.byref(handle)))
        self._h = handle
        self.n_layers, self.num_blocks, self.block_size = int(n_layers), int(num_blocks), int(block_size)
        self.n_kv_heads, self.head_dim, self.device = int(n_kv_heads), int(head_dim), int(device)

    def close(self) -> None:
        if getattr(self, "_h", None) and _capi.lib is not None:  # (None: the interpreter is going down)
            _capi.lib.nvk_mx4_pool_destroy(self._h)
            self._h = None

    __del__ = close

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def handle(self) -> C.c_void_p:
        if not self._h:
            raise RuntimeError("pool is closed")
        return self._h

    @property
    def layer_bytes(self) -> int:
        return int(_capi.lib.nvk_mx4_pool_layer_bytes(self.handle))

    def layer_ptr(self, layer: int) -> int:
        p = C.c_void_p()
        _capi.check(_capi.lib.nvk_mx4_pool_layer_ptr(self.handle, int(layer), C.byref(p)))
        return int(p.value)

    @property
    def stream(self) -> int:
        s = C.c_void_p()
        _capi.check(_capi.lib.nvk_mx4_pool_stream(self.handle, C.byref(s)))
        return int(s.value or 0)

    @property
    def workspace_generation(self) -> int:
        return int(_capi.lib.nvk_mx4_pool_workspace_generation(self.handle))

    def synchronize(self) -> None:
        _capi.check(_capi.lib.nvk_mx4_pool_synchronize(self.handle))

    def reserve_workspace(self, num_seqs: int, n_heads: int, max_rows: int, max_ctx: int, total_rows: Optional[int] = None) -> None:
        """Room for later attention calls of up to this shape (needed before capturing them); total_rows: all sequences'
        query rows, num_seqs * max_rows unless given."""
        total = int(num_seqs) * int(max_rows) if total_rows is None else int(total_rows)
        _capi.check(_capi.lib.nvk_mx4_pool_reserve_workspace(self.handle, int(num_seqs), int(n_heads), total, int(max_rows),
                                                             int(max_ctx)))

    def read_rows(self, layer: int, block_tables, positions, row_seqs=None) -> Tuple[np.ndarray, np.ndarray]:
        """The values held for the given rows: (k, v), each [rows, n_kv_heads, head_dim]; zeros for rows of padding."""
        tabs, pos = _i32(block_tables), _i32(positions).reshape(-1)
        if tabs.ndim != 2:
            raise ValueError("block_tables must be [num_seqs, max_blocks]")
        seqs = None if row_seqs is None else _i32(row_seqs).reshape(-1)
        if (seqs is not None and seqs.size != pos.size) or (seqs is None and pos.size > tabs.shape[0]):
            raise ValueError("every row needs a table row")
        k = np.zeros((pos.size, self.n_kv_heads, self.head_dim), np.float32)
        v = np.zeros_like(k)
        _capi.check(_capi.lib.nvk_mx4_pool_read_rows(self.handle, int(layer), pos.size, _ptr(seqs), _ptr(pos), _ptr(tabs), tabs.shape[0],
                                                     tabs.shape[1], _ptr(k), _ptr(v), _capi.PTR_HOST, None))
        return k, v

    def read_rows_device(self, layer: int, rows: int, row_seqs_dev, positions_dev, block_tables_dev, num_seqs: int, max_blocks: int,
                         k_out_dev, v_out_dev, stream=None) -> None:
        _capi.check(_capi.lib.nvk_mx4_pool_read_rows(self.handle, int(layer), int(rows), _address(row_seqs_dev), _address(positions_dev),
                                                     _address(block_tables_dev), int(num_seqs), int(max_blocks), _address(k_out_dev),
                                                     _address(v_out_dev), _capi.PTR_DEVICE, _address(stream)))


def _lens(pool, block_tables, ctx_lens):
    tabs, ctx = _i32(block_tables), _i32(ctx_lens).reshape(-1)
    if tabs.ndim != 2 or ctx.size != tabs.shape[0]:
        raise ValueError("block_tables must be [num_seqs, max_blocks] and ctx_lens [num_seqs]")
    return tabs, ctx


def mx4_decode(pool: Mx4KVPool, layer: int, q, block_tables, ctx_lens) -> np.ndarray:
    """One layer-call from host arrays: q [num_seqs, n_heads, head_dim] -> out of the same shape."""
    tabs, ctx = _lens(pool, block_tables, ctx_lens)
    qh = _f32(q)
    if qh.ndim != 3 or qh.shape[0] != ctx.size or qh.shape[2] != pool.head_dim:
        raise ValueError("q must be [num_seqs, n_heads, head_dim]")
    out = np.empty_like(qh)
    _capi.check(_capi.lib.nvk_mx4_decode(pool.handle, int(layer), ctx.size, int(qh.shape[1]), _ptr(qh), _ptr(tabs), tabs.shape[1],
                                         _ptr(ctx), _ptr(out)))
    return out


def mx4_prefill(pool: Mx4KVPool, layer: int, q, block_tables, chunk_lens, ctx_lens) -> np.ndarray:
    """Causal attention of each sequence's newest chunk_lens[s] tokens over its ctx_lens[s] cached ones (the chunk included):
    q [sum(chunk_lens), n_heads, head_dim] -> out of the same shape."""
    tabs, ctx = _lens(pool, block_tables, ctx_lens)
    lens, qh = _i32(chunk_lens).reshape(-1), _f32(q)
    if lens.size != ctx.size or qh.ndim != 3 or qh.shape[0] != int(lens.astype(np.int64).sum()) or qh.shape[2] != pool.head_dim:
        raise ValueError("q must be [sum(chunk_lens), n_heads, head_dim], chunk_lens [num_seqs]")
    out = np.empty_like(qh)
    _capi.check(_capi.lib.nvk_mx4_prefill(pool.handle, int(layer), ctx.size, int(qh.shape[1]), _ptr(qh), _ptr(tabs), tabs.shape[1],
                                          _ptr(lens), _ptr(ctx), _ptr(out)))
    return out


def mx4_decode_device(pool: Mx4KVPool, layer: int, num_seqs: int, n_heads: int, q_dev, block_tables_dev, max_blocks: int, ctx_lens_dev,
                      max_ctx: int, out_dev, stream=None) -> None:
    """Asynchronous layer-call on device pointers."""
    _capi.check(_capi.lib.nvk_mx4_decode_device(pool.handle, int(layer), int(num_seqs), int(n_heads), _address(q_dev),
                                                _address(block_tables_dev), int(max_blocks), _address(ctx_lens_dev), int(max_ctx),
                                                _address(out_dev), _address(stream)))


def mx4_prefill_device(pool: Mx4KVPool, layer: int, num_seqs: int, n_heads: int, total_rows: int, q_dev, row_offsets_dev, max_rows: int,
                       block_tables_dev, max_blocks: int, ctx_lens_dev, max_ctx: int, out_dev, stream=None) -> None:
    """Asynchronous form; row_offsets_dev [num_seqs + 1] are the first rows of the sequences' chunks."""
    _capi.check(_capi.lib.nvk_mx4_prefill_device(pool.handle, int(layer), int(num_seqs), int(n_heads), int(total_rows), _address(q_dev),
                                                 _address(row_offsets_dev), int(max_rows), _address(block_tables_dev), int(max_blocks),
                                                 _address(ctx_lens_dev), int(max_ctx), _address(out_dev), _address(stream)))
