"""RMS norm of query and key heads, rotary positions and the append to a paged cache, in one launch.

The reference rotates adjacent pairs over the whole head, unscaled and without a norm (``Ops::apply_rope``,
``include/ops/positional.hpp:13-39``, then the append at ``include/core/model.hpp:190-207``); a :class:`RotaryTable` also knows
the half layout, a rotated part of the head, and contexts stretched beyond the trained length.  The cache may be a
:class:`PagedKVPool` or an :class:`Mx4KVPool`."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np

from . import _capi
from .kv_pool import PagedKVPool, _address, _f32, _i32, _ptr

ROPE_INTERLEAVED = _capi.ROPE_INTERLEAVED
ROPE_HALF = _capi.ROPE_HALF
ROPE_SCALE_NONE = _capi.ROPE_SCALE_NONE
ROPE_SCALE_LINEAR = _capi.ROPE_SCALE_LINEAR
ROPE_SCALE_NTK = _capi.ROPE_SCALE_NTK
ROPE_SCALE_YARN = _capi.ROPE_SCALE_YARN


class RotaryTable:
    """Angles per position of the rotated pairs of a head (``nvk_rope_*``); made once, usable from any stream."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, layout: int = ROPE_INTERLEAVED, theta: float = 10000.0,
                 scaling: int = ROPE_SCALE_NONE, factor: float = 1.0, original_len: int = 0, device: int = 0):
        h = C.c_void_p()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        _capi.check(_capi.lib.nvk_rope_create(int(head_dim), int(rotary_dim), int(layout), float(theta), int(scaling),
                                              float(factor), int(original_len), int(device), C.byref(h)))
        self._h = h
        self.head_dim, self.rotary_dim, self.layout, self.device = int(head_dim), int(rotary_dim), int(layout), int(device)

    def close(self) -> None:
        if getattr(self, "_h", None) and _capi.lib is not None:  # (None: the interpreter is going down)
            _capi.lib.nvk_rope_destroy(self._h)
            self._h = None

    __del__ = close

    @property
    def handle(self) -> C.c_void_p:
        if not self._h:
            raise RuntimeError("rotary table is closed")
        return self._h

    def frequencies(self):
        """(angle per position of every pair, factor on cos and sin), both in 64 bits."""
        freq = np.empty(self.rotary_dim // 2, np.float64)
        factor = C.c_double()
        _capi.check(_capi.lib.nvk_rope_frequencies(self.handle, freq.ctypes.data_as(C.POINTER(C.c_double)), freq.size,
                                                   C.byref(factor)))
        return freq, float(factor.value)


def _entry(pool):
    return _capi.lib.nvk_pool_norm_rope_append if isinstance(pool, PagedKVPool) else _capi.lib.nvk_mx4_pool_norm_rope_append


def norm_rope_append_device(pool, layer: int, rope: Optional[RotaryTable], rows: int, n_heads: int, q_dev, q_out_dev, k_rows_dev,
                            v_rows_dev, q_weight_dev, k_weight_dev, eps: float, row_seqs_dev, positions_dev, block_tables_dev,
                            num_seqs: int, max_blocks: int, stream=None) -> None:
    """Asynchronous form on device pointers; see ``nvk_pool_norm_rope_append`` for what may be None."""
    _capi.check(_entry(pool)(pool.handle, int(layer), rope.handle if rope is not None else None, int(rows), int(n_heads),
                             _address(q_dev), _address(q_out_dev), _address(k_rows_dev), _address(v_rows_dev), _address(q_weight_dev),
                             _address(k_weight_dev), float(eps), _address(row_seqs_dev), _address(positions_dev),
                             _address(block_tables_dev), int(num_seqs), int(max_blocks), _capi.PTR_DEVICE, _address(stream)))


def norm_rope_append(pool, layer: int, rope: Optional[RotaryTable], q, k_rows, v_rows, block_tables, positions, row_seqs=None,
                     q_weight=None, k_weight=None, eps: float = 1e-5) -> Optional[np.ndarray]:
    """The same from host arrays: q [rows, n_heads, head_dim] or None, k_rows / v_rows [rows, n_kv_heads, head_dim] or None.
    Returns the normed and rotated q (rows of padding, position < 0, as they came), or None without q."""
    tabs, pos = _i32(block_tables), _i32(positions).reshape(-1)
    if tabs.ndim != 2:
        raise ValueError("block_tables must be [num_seqs, max_blocks]")
    n, hd = pos.size, pool.head_dim
    seqs = None if row_seqs is None else _i32(row_seqs).reshape(-1)
    if seqs is not None and seqs.size != n:
        raise ValueError("row_seqs must be [rows], like positions")
    if seqs is None and n > tabs.shape[0] and k_rows is not None:
        raise ValueError("without row_seqs every row needs a table row of its own")
    qh = None if q is None else _f32(q)
    if qh is not None and (qh.ndim != 3 or qh.shape[0] != n or qh.shape[2] != hd):
        raise ValueError("q must be [rows, n_heads, head_dim]")
    if (k_rows is None) != (v_rows is None):
        raise ValueError("k_rows and v_rows come in pairs")
    k = None if k_rows is None else _f32(k_rows, (n, pool.n_kv_heads, hd))
    v = None if v_rows is None else _f32(v_rows, (n, pool.n_kv_heads, hd))
    wq = None if q_weight is None else _f32(q_weight, (hd,))
    wk = None if k_weight is None else _f32(k_weight, (hd,))
    out = None if qh is None else np.empty_like(qh)
    heads = pool.n_kv_heads if qh is None else qh.shape[1]
    _capi.check(_entry(pool)(pool.handle, int(layer), rope.handle if rope is not None else None, n, int(heads), _ptr(qh), _ptr(out),
                             _ptr(k), _ptr(v), _ptr(wq), _ptr(wk), float(eps), _ptr(seqs), _ptr(pos), _ptr(tabs), tabs.shape[0],
                             tabs.shape[1], _capi.PTR_HOST, None))
    return out
