"""Edges of the paged-cache operators that their own files leave out."""
import ctypes as C

import numpy as np
import pytest

import nano_vllm_amd as nv
import operator_oracles as oo
from hipmem import DeviceArray
from nano_vllm_amd import _capi
from test_gpu_sparse import filled as filled_index

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("geom", [(2, 2, 64), (4, 2, 128), (8, 2, 32), (12, 2, 64), (12, 2, 128), (4, 2, 256), (14, 2, 256)],
                         ids=lambda g: "x".join(map(str, g)))
def test_a_query_that_holds_no_number_has_infinite_scores(geom):
    """max(q, 0) and min(q, 0) of a NaN are no number, so no block's score is one: all count as infinite, and the lowest blocks are read
    beside the first and the last.  The other kv-head's queries choose as ever."""
    H, KV, hd = geom
    bs, top, first, last, ctx = 16, 9, 1, 2, [40 * 16 - 3]
    pool, tabs, held = filled_index(ctx, bs, KV, hd, seed=71)
    q = np.random.default_rng(72).normal(size=(1, H, hd)).astype(np.float32)
    q[0, H - 1, hd - 3] = np.nan  # the last head of the second kv-head
    with pool, nv.BlockIndex(pool) as index:
        index.update(1, tabs, [0], ctx)
        got, sel = nv.sparse_decode(index, 1, q, tabs, ctx, top, first, last)
    score = oo.block_scores(q[0], held[0][0], ctx[0], bs, KV)
    assert sel[0, 0].tolist() == oo.choose(score[0], 40, top, first, last)
    assert sel[0, 1].tolist() == oo.choose(np.full(40, np.inf), 40, top, first, last)
    assert np.isfinite(got[0, :H - 1]).all() and np.isnan(got[0, H - 1]).all()


@pytest.mark.parametrize("cache", ["fp32", "mx4"])
@pytest.mark.parametrize("kind", [_capi.PTR_HOST, _capi.PTR_DEVICE], ids=["host", "device"])
def test_rotation_alone_reads_positions_alone(cache, kind):
    """Without rows to append, tables and sequences are not looked at: neither an address where nothing is nor a size that no array has."""
    rows, H, hd = 5, 4, 64
    q = np.random.default_rng(73).normal(size=(rows, H, hd)).astype(np.float32)
    pos = np.array([0, 7, -1, 900, 3], np.int32)
    nowhere = C.c_void_p(4096)
    entry = _capi.lib.nvk_pool_norm_rope_append if cache == "fp32" else _capi.lib.nvk_mx4_pool_norm_rope_append
    rope = nv.RotaryTable(hd)
    with (nv.PagedKVPool if cache == "fp32" else nv.Mx4KVPool)(1, 2, 16, 1, hd) as pool:
        want = nv.norm_rope_append(pool, 0, rope, q, None, None, np.zeros((rows, 1), np.int32), pos)
        for seqs, max_blocks in ((1 << 20, 1 << 10), (3, -1), (0, 0)):
            out = np.zeros_like(q)
            if kind == _capi.PTR_HOST:
                a = [C.c_void_p(x.ctypes.data) for x in (q, out, pos)]
            else:
                d = [DeviceArray(x) for x in (q, out, pos)]
                a = [x.ptr for x in d]
            assert entry(pool.handle, 0, rope.handle, rows, H, a[0], a[1], None, None, None, None, 1e-5, nowhere, a[2], nowhere, seqs, max_blocks,
                         kind, None) == 0
            if kind == _capi.PTR_DEVICE:
                pool.synchronize()
                out = d[1].numpy()
                want[2] = 0  # (the row of padding: left alone here, returned as it came there)
            assert (out == want).all()
    rope.close()
