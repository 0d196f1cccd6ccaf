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


@pytest.mark.parametrize("case", [(16, 128, 90, 40), (16, 64, 3000, 40), (2, 32, 6000, 2000), (16, 256, 2000, 300)], ids=str)
def test_scores_that_are_all_minus_infinity_are_no_answer(case):
    """Every key holds -inf in a channel where the query is positive: 0 / 0, which is nvk_decode's answer too and not the zeros of an
    empty context.  Written directly, joined by the attention kernel, joined by a kernel of its own; beside it a context of which one
    token is left, and an empty one."""
    bs, hd, n, top = case
    rng = np.random.default_rng(74)
    ctx = [n, n, 0]
    tabs, blocks = oo.tables_for(ctx, bs, seed=75)
    k, v = (rng.normal(size=(2, n, 1, hd)).astype(np.float32) for _ in range(2))
    k[:, :, 0, 5] = -np.inf
    k[1, n - 1, 0, 5] = 0.25
    q = rng.normal(size=(3, 4, hd)).astype(np.float32)
    q[:, :, 5] = 1.0
    with nv.PagedKVPool(1, blocks, bs, 1, hd) as pool, nv.BlockIndex(pool) as index:
        for s in range(2):
            nv.norm_rope_append(pool, 0, None, None, k[s], v[s], tabs, np.arange(n), np.full(n, s))
        index.update(0, tabs, [0, 0, 0], ctx)
        got, _ = nv.sparse_decode(index, 0, q, tabs, ctx, top, 1, 1)
        dense = nv.decode(pool, 0, q, np.where(tabs < 0, 0, tabs), ctx)
    for out in (got, dense):
        assert np.isnan(out[0]).all() and (out[1] == v[1, n - 1, 0]).all() and (out[2] == 0).all()


@pytest.mark.parametrize("hd", [48, 128, 256])
@pytest.mark.parametrize("n", [40, 1500, 9000])
def test_scores_of_the_4_bit_cache_that_pass_fp32_are_no_answer(hd, n):
    """Every score below the least fp32 number: 0 / 0 as above, decode and chunks of a few and of many rows; an empty context beside it."""
    bs, rows = 16, (1, 3, 70)
    tabs, blocks = oo.tables_for([n, 0], bs, seed=76)
    v = np.random.default_rng(77).normal(size=(n, 1, hd)).astype(np.float32)
    with nv.Mx4KVPool(1, blocks, bs, 1, hd) as pool:
        nv.norm_rope_append(pool, 0, None, None, np.full((n, 1, hd), -1e38, np.float32), v, tabs, np.arange(n), np.zeros(n, np.int32))
        q = np.full((80, 4, hd), 3e38, np.float32)
        one = nv.mx4_decode(pool, 0, q[:2], tabs, [n, 0])
        assert np.isnan(one[0]).all() and (one[1] == 0).all()
        for r in rows:
            if r <= n:
                assert np.isnan(nv.mx4_prefill(pool, 0, q[:r], tabs, [r, 0], [n, 0])).all(), r
