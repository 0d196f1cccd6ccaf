"""The block index and block-sparse decode against their definitions in 64 bits (operator_oracles.py)."""
import ctypes as C

import numpy as np
import pytest

import nano_vllm_amd as nv
import operator_oracles as oo
from hipmem import D2H, H2D, DeviceArray, Stream, _hip

pytestmark = pytest.mark.gpu


def filled(ctx_lens, bs, kv, hd, seed):
    rng = np.random.default_rng(seed)
    tabs, blocks = oo.tables_for(ctx_lens, bs, seed)
    pool = nv.PagedKVPool(2, blocks, bs, kv, hd)
    held = []
    for s, n in enumerate(ctx_lens):
        nb = (n + bs - 1) // bs
        k = (np.repeat(rng.normal(size=(nb, kv, hd)), bs, 0)[:n] + 0.5 * rng.normal(size=(n, kv, hd))).astype(np.float32)
        v = rng.normal(size=(n, kv, hd)).astype(np.float32)
        if n:
            nv.norm_rope_append(pool, 1, None, None, k, v, tabs, np.arange(n), np.full(n, s))
        held.append((k, v))
    return pool, tabs, held


def bounds_of(index, layer):
    p = index.pool
    out = np.empty((p.num_blocks, p.n_kv_heads, 2, p.head_dim), np.float32)
    assert _hip.hipDeviceSynchronize() == 0
    assert _hip.hipMemcpy(C.c_void_p(out.ctypes.data), C.c_void_p(index.layer_ptr(layer)), out.nbytes, D2H) == 0
    return out


def check(pool, index, tabs, held, ctx, H, top, first, last, seed):
    KV, bs = pool.n_kv_heads, pool.block_size
    q = np.random.default_rng(seed).normal(size=(len(ctx), H, pool.head_dim)).astype(np.float32)
    got, sel = nv.sparse_decode(index, 1, q, tabs, ctx, top, first, last)
    g = H // KV
    for s, n in enumerate(ctx):
        nb = (n + bs - 1) // bs
        score = oo.block_scores(q[s], held[s][0], n, bs, KV)
        for j in range(KV):
            want_sel = oo.choose(score[j], nb, top, first, last)
            assert sel[s, j].tolist() == want_sel + [-1] * (top - len(want_sel)), f"sequence {s} of {n} tokens, kv-head {j}"
            tok = np.array([t for b in want_sel for t in range(b * bs, min(n, (b + 1) * bs))], int)
            want, bound = oo.attention(q[s:s + 1, j * g:(j + 1) * g], held[s][0][tok, j:j + 1], held[s][1][tok, j:j + 1], [len(tok)])
            err = np.abs(got[s, j * g:(j + 1) * g] - want[0])
            assert (err <= bound[0]).all(), f"sequence {s} of {n} tokens, kv-head {j}: {err.max():.3e}"
    return got


GEOMS = [(8, 2, 128, 16), (4, 4, 128, 16), (6, 6, 48, 16), (6, 2, 64, 8), (5, 1, 128, 5), (16, 1, 256, 16), (2, 2, 256, 32), (7, 1, 32, 1),
         (3, 1, 4, 3), (10, 5, 80, 64), (24, 2, 96, 16)]


@pytest.mark.parametrize("geom", GEOMS, ids=lambda g: "x".join(map(str, g)))
@pytest.mark.parametrize("picks", [(4, 1, 1), (9, 0, 2), (1, 0, 1), (40, 2, 3)], ids=str)
def test_against_definition(geom, picks):
    H, KV, hd, bs = geom
    top, first, last = picks
    ctx = [0, 1, bs, bs + 1, 3 * bs, 5 * bs - 1, 37 * bs + bs // 2, 50 * bs]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=hd + H)
    with pool, nv.BlockIndex(pool) as index:
        index.update(1, tabs, [0] * len(ctx), ctx)
        check(pool, index, tabs, held, ctx, H, top, first, last, seed=top)


def test_long_context():
    """Thousands of blocks: several score workgroups, several passes of the selection, chunks of the chosen blocks."""
    H, KV, hd, bs = 4, 2, 32, 4
    ctx = [30000, 9001, 16]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=1)
    with pool, nv.BlockIndex(pool) as index:
        index.update(1, tabs, [0] * 3, ctx)
        for top, first, last in ((700, 1, 4), (64, 0, 1)):
            check(pool, index, tabs, held, ctx, H, top, first, last, seed=2)


def test_index_follows_appends():
    """Updates cover exactly the blocks of the new tokens; a block's bounds come from all its tokens below the context."""
    H, KV, hd, bs = 4, 2, 64, 16
    rng = np.random.default_rng(3)
    ctx_end = [70, 35]
    tabs, blocks = oo.tables_for(ctx_end, bs)
    k, v = [[rng.normal(size=(n, KV, hd)).astype(np.float32) for n in ctx_end] for _ in range(2)]
    with nv.PagedKVPool(2, blocks, bs, KV, hd) as pool, nv.BlockIndex(pool) as index:
        have = [0, 0]
        want = np.zeros((blocks, KV, 2, hd), np.float32)
        for new in ((20, 1), (0, 15), (12, 0), (1, 1), (37, 18)):
            start = list(have)
            for s in range(2):
                if new[s]:
                    p = np.arange(have[s], have[s] + new[s])
                    nv.norm_rope_append(pool, 1, None, None, k[s][p], v[s][p], tabs, p, np.full(len(p), s))
                    have[s] += new[s]
                    for b in range(start[s] // bs, (have[s] + bs - 1) // bs):
                        rows = k[s][b * bs:min(have[s], (b + 1) * bs)]
                        want[tabs[s, b], :, 0], want[tabs[s, b], :, 1] = rows.min(0), rows.max(0)
            index.update(1, tabs, start, have)
            assert (bounds_of(index, 1) == want).all()
        assert (bounds_of(index, 0) == 0).all(), "another layer"


def test_everything_read_is_dense_decode():
    """top_blocks at or above the number of blocks: nvk_decode's result, within both sides' bounds."""
    H, KV, hd, bs = 8, 2, 128, 16
    ctx = [100, 16, 333]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=4)
    with pool, nv.BlockIndex(pool) as index:  # (never updated: no score is asked for)
        q = np.random.default_rng(5).normal(size=(3, H, hd)).astype(np.float32)
        got, sel = nv.sparse_decode(index, 1, q, tabs, ctx, 21)
        dense = nv.decode(pool, 1, q, np.where(tabs < 0, 0, tabs), ctx)
        for s, n in enumerate(ctx):
            _, bound = oo.attention(q[s:s + 1], *held[s], [n])
            assert (np.abs(got[s] - dense[s]) <= 2 * bound[0]).all()
            assert (sel[s] == [list(range((n + 15) // 16)) + [-1] * (21 - (n + 15) // 16)] * KV).all()


def test_ties_and_odd_scores():
    """Blocks with the same bounds: the lowest are read.  A block whose keys hold a NaN is read, and answers NaN."""
    KV, hd, bs, n = 1, 64, 16, 40 * 16
    rng = np.random.default_rng(6)
    same = rng.normal(size=(bs, KV, hd)).astype(np.float32)
    k = np.tile(same, (40, 1, 1))
    v = rng.normal(size=(n, KV, hd)).astype(np.float32)
    k[17 * bs:18 * bs] *= 2  # one block above the others for q = its own keys' direction
    tabs, blocks = oo.tables_for([n], bs)
    with nv.PagedKVPool(1, blocks, bs, KV, hd) as pool, nv.BlockIndex(pool) as index:
        nv.norm_rope_append(pool, 0, None, None, k, v, tabs, np.arange(n), np.zeros(n, np.int32))
        index.update(0, tabs, [0], [n])
        q = same[:1].copy()
        _, sel = nv.sparse_decode(index, 0, q, tabs, [n], 9, 1, 2)
        assert sel[0, 0].tolist() == [0, 1, 2, 3, 4, 5, 17, 38, 39]
        _, sel = nv.sparse_decode(index, 0, np.zeros_like(q), tabs, [n], 5, 0, 1)  # every score 0
        assert sel[0, 0].tolist() == [0, 1, 2, 3, 39]
        k[30 * bs + 3, 0, 5] = np.nan
        nv.norm_rope_append(pool, 0, None, None, k, v, tabs, np.arange(n), np.zeros(n, np.int32))
        index.update(0, tabs, [0], [n])
        out, sel = nv.sparse_decode(index, 0, q, tabs, [n], 4, 1, 1)
        assert 30 in sel[0, 0].tolist() and np.isnan(out).all()
        out, _ = nv.sparse_decode(index, 0, q, tabs, [30 * bs + 3], 4, 1, 1)  # the NaN lies behind this context
        assert np.isfinite(out).all()


def test_refusals():
    with nv.PagedKVPool(1, 4, 16, 2, 64) as pool, nv.BlockIndex(pool) as index:
        q, t = np.zeros((1, 4, 64), np.float32), np.array([[0, 1]], np.int32)
        nv.sparse_decode(index, 0, q, t, [20], 2)
        for kw in (dict(ctx=[33]), dict(ctx=[-1]), dict(tabs=[[0, 4]]), dict(layer=1), dict(top=0), dict(top=1), dict(last=0), dict(first=-1),
                   dict(q=np.zeros((1, 3, 64), np.float32))):
            a = dict(layer=0, q=q, tabs=t, ctx=[20], top=2, first=1, last=1)
            a.update(kw)
            with pytest.raises(nv.NvkError):
                nv.sparse_decode(index, a["layer"], a["q"], np.array(a["tabs"], np.int32), a["ctx"], a["top"], a["first"], a["last"])
        for start, ctx in (([-1], [20]), ([21], [20]), ([0], [40])):
            with pytest.raises(nv.NvkError):
                index.update(0, t, start, ctx)
        index.update(0, t, [20], [20])  # nothing new
        with pytest.raises(nv.NvkError):
            index.reserve_workspace(1, 3, 16, 4)
        with pytest.raises(ValueError):
            nv.sparse_decode(index, 0, q[0], t, [20], 2)
        lib, d = nv._capi.lib, DeviceArray(np.zeros(4096, np.float32))
        odd = C.c_void_p(d.ptr.value + 4)
        for p in ((None, d.ptr, d.ptr), (odd, d.ptr, d.ptr), (d.ptr, None, d.ptr), (d.ptr, d.ptr, None)):
            assert lib.nvk_sparse_decode_device(index.handle, 0, 1, 4, p[0], p[1], 1, p[2], 16, 2, 1, 1, d.ptr, None, None) == nv._capi.ERR_INVALID_ARG
    with nv.PagedKVPool(1, 4, 16, 2, 64) as pool:
        index = nv.BlockIndex(pool)
    with pytest.raises(RuntimeError):
        nv.sparse_decode(index, 0, np.zeros((1, 4, 64), np.float32), np.zeros((1, 1), np.int32), [1], 2)


def test_decode_loop_together_and_captured():
    """append -> update -> sparse decode as a serving loop runs them, one captured graph replayed over growing contexts, each
    step against the definition; a capture that has to grow the workspace is refused."""
    H, KV, hd, bs, n, steps = 8, 2, 64, 16, 3, 5
    start = [150, 64, 300]
    room = [s + steps for s in start]
    rng = np.random.default_rng(50)
    tabs, blocks = oo.tables_for(room, bs)
    k, v = [[rng.normal(size=(m, KV, hd)).astype(np.float32) for m in room] for _ in range(2)]
    rope = nv.RotaryTable(hd)
    freq, fm = oo.frequencies(hd, 10000.0)
    kr = [oo.norm_rope(k[s], None, 0, np.arange(room[s]), freq, fm, False).astype(np.float32) for s in range(n)]
    top, first, last = 6, 1, 2
    st = Stream()
    with nv.PagedKVPool(2, blocks, bs, KV, hd) as pool, nv.BlockIndex(pool) as index:
        for s in range(n):
            p = np.arange(start[s])
            nv.norm_rope_append(pool, 1, rope, None, k[s][p], v[s][p], tabs, p, np.full(len(p), s))
        index.update(1, tabs, [0] * n, start)
        zero = lambda *shape: DeviceArray(np.zeros(shape, np.float32))  # noqa: E731
        dq, do, dk, dv = zero(n, H, hd), zero(n, H, hd), zero(n, KV, hd), zero(n, KV, hd)
        dpos, dctx, dt, dsel = (DeviceArray(np.zeros(x, np.int32)) for x in (n, n, tabs.shape, (n, KV, top)))
        put = lambda a, b: _hip.hipMemcpy(a.ptr, C.c_void_p(b.ctypes.data), b.nbytes, H2D)  # noqa: E731
        put(dt, tabs)

        def step():
            nv.norm_rope_append_device(pool, 1, rope, n, H, dq, dq, dk, dv, None, None, 1e-5, None, dpos, dt, n, tabs.shape[1], st)
            index.update_device(1, n, dt, tabs.shape[1], dpos, dctx, 1, st)
            nv.sparse_decode_device(index, 1, n, H, dq, dt, tabs.shape[1], dctx, max(room), top, first, last, do, dsel, st)

        def refused():
            with pytest.raises(nv.NvkError):
                step()

        st.capture(refused)
        index.reserve_workspace(n, H, max(room), top)
        exe = st.capture(step)
        for i in range(steps):
            pos = np.array([s + i for s in start], np.int32)
            ctx = pos + 1
            q = rng.normal(size=(n, H, hd)).astype(np.float32)
            for a, b in ((dq, q), (dk, np.stack([k[s][pos[s]] for s in range(n)])), (dv, np.stack([v[s][pos[s]] for s in range(n)])),
                         (dpos, pos), (dctx, ctx)):
                assert put(a, np.ascontiguousarray(b)) == 0
            st.launch(exe)
            st.synchronize()
            got, sel, qr = do.numpy(), dsel.numpy(), dq.numpy()
            eager, esel = nv.sparse_decode(index, 1, qr, np.where(tabs < 0, 0, tabs), ctx, top, first, last)
            assert (got == eager).all() and (sel == esel).all(), f"step {i}"
            for s in range(n):
                score = oo.block_scores(qr[s], kr[s], int(ctx[s]), bs, KV)
                for j in range(KV):
                    want_sel = oo.choose(score[j], (int(ctx[s]) + bs - 1) // bs, top, first, last)
                    assert sel[s, j].tolist() == want_sel + [-1] * (top - len(want_sel))
                    tok = np.array([t for b in want_sel for t in range(b * bs, min(ctx[s], (b + 1) * bs))], int)
                    g = H // KV
                    want, bound = oo.attention(qr[s:s + 1, j * g:(j + 1) * g], kr[s][tok, j:j + 1], v[s][tok, j:j + 1], [len(tok)])
                    assert (np.abs(got[s, j * g:(j + 1) * g] - want[0]) <= bound[0]).all()
    st.close()


def test_a_pool_and_an_index_of_more_than_32_bits():
    """Blocks whose keys and whose bounds lie beyond 2^31 floats of a layer answer what the first ones do."""
    KV, hd, bs, H, n = 8, 128, 4, 16, 41
    blocks = 1_060_000  # 4096 floats of keys, 2048 of bounds each
    rng = np.random.default_rng(60)
    k, v = (rng.normal(size=(n, KV, hd)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(1, H, hd)).astype(np.float32)
    low = np.random.default_rng(61).permutation(11).astype(np.int32)[None]
    high = (blocks - 1 - low).astype(np.int32)
    got = []
    with nv.PagedKVPool(1, blocks, bs, KV, hd) as pool, nv.BlockIndex(pool) as index:
        for tabs in (low, high):
            nv.norm_rope_append(pool, 0, None, None, k, v, tabs, np.arange(n), np.zeros(n, np.int32))
            index.update(0, tabs, [0], [n])
            got.append(nv.sparse_decode(index, 0, q, tabs, [n], 5, 1, 1))
    assert (got[0][0] == got[1][0]).all() and (got[0][1] == got[1][1]).all()
    score = oo.block_scores(q[0], k, n, bs, KV)
    for j in range(KV):
        assert got[0][1][0, j].tolist() == oo.choose(score[j], 11, 5, 1, 1)


def test_without_a_list_and_at_any_float():
    """The list left out (also with top_blocks far above the blocks there are), a result 4 bytes behind a line, other streams,
    and what is refused."""
    KV, hd, bs, H = 2, 32, 4, 4
    ctx = [9001, 37, 0]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=62)
    q = np.random.default_rng(63).normal(size=(3, H, hd)).astype(np.float32)
    st = Stream()
    with pool, nv.BlockIndex(pool) as index:
        index.update(1, tabs, [0] * 3, ctx)
        dq, dt, dc, do = (DeviceArray(x) for x in (q, tabs, np.array(ctx, np.int32), np.zeros(3 * H * hd + 1, np.float32)))
        for top, n in ((64, 3), (700, 3), (5000, 3), (2 ** 31 - 1, 3), (4, 1)):
            want, _ = nv.sparse_decode(index, 1, q[:n], tabs[:n], ctx[:n], min(top, 5000))
            nv.sparse_decode_device(index, 1, n, H, dq, dt, tabs.shape[1], dc, max(ctx), top, 1, 1, do.data_ptr() + 4, None, st)
            st.synchronize()
            assert (do.numpy()[1:1 + n * H * hd].reshape(n, H, hd) == want).all(), top
        for kw in (dict(out=do.data_ptr() + 2), dict(ctx=2 ** 31 - 1)):
            with pytest.raises(nv.NvkError):
                nv.sparse_decode_device(index, 1, 3, H, dq, dt, tabs.shape[1], dc, kw.get("ctx", max(ctx)), 9, 1, 1, kw.get("out", do.data_ptr()))
    st.close()


@pytest.mark.parametrize("blocks", [(256, 257, 9, 500), (1025, 600, 40, 1), (2048, 1500, 2047, 513), (2049, 2048, 300, 41)], ids=str)
@pytest.mark.parametrize("levels", [0, 3])
def test_selections_of_every_size(blocks, levels):
    """One to eight blocks a thread and the kernel for more, beside contexts that are read whole; scores of a few levels (many
    ties) or all different, some of them negative."""
    KV, hd, bs, H, top = 2, 4, 2, 4, 40
    ctx = [b * bs - (i % 2) for i, b in enumerate(blocks)]
    tabs, n = oo.tables_for(ctx, bs, seed=64)
    rng = np.random.default_rng(65 + levels)
    held = []
    with nv.PagedKVPool(2, n, bs, KV, hd) as pool, nv.BlockIndex(pool) as index:
        for s, c in enumerate(ctx):
            k = (rng.integers(-levels, levels + 1, (c, KV, hd)) if levels else rng.normal(size=(c, KV, hd))).astype(np.float32)
            v = rng.normal(size=(c, KV, hd)).astype(np.float32)
            nv.norm_rope_append(pool, 1, None, None, k, v, tabs, np.arange(c), np.full(c, s))
            held.append((k, v))
        index.update(1, tabs, [0] * len(ctx), ctx)
        for first, last in ((1, 2), (0, 1), (20, 20)):
            check(pool, index, tabs, held, ctx, H, top, first, last, seed=66)


@pytest.mark.parametrize("geom", [(16, 2, 128, 16), (10, 2, 64, 4), (7, 1, 32, 2), (21, 1, 36, 3), (40, 1, 128, 2), (9, 1, 80, 8), (12, 2, 4, 1)],
                         ids=lambda g: "x".join(map(str, g)))
def test_large_groups(geom):
    """Groups of 5 to 40 heads: bounds on matrix instructions, sixteen heads and blocks at a time, more blocks than a wave takes;
    a block whose keys hold an infinity counts as highest."""
    H, KV, hd, bs = geom
    ctx = [700 * bs - 1, 17 * bs, 16 * bs + 1, 0, 131 * bs]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=hd + H)
    with pool, nv.BlockIndex(pool) as index:
        index.update(1, tabs, [0] * len(ctx), ctx)
        for top, first, last in ((9, 1, 2), (16, 0, 1)):
            check(pool, index, tabs, held, ctx, H, top, first, last, seed=top)
        k = held[0][0][:500 * bs].copy()
        k[300 * bs, 0, 1] = np.inf
        k[310 * bs, 0, 2] = np.nan
        nv.norm_rope_append(pool, 1, None, None, k, held[0][1][:500 * bs], tabs, np.arange(500 * bs), np.zeros(500 * bs, np.int32))
        index.update(1, tabs[:1], [0], [500 * bs])
        q = np.abs(np.random.default_rng(1).normal(size=(1, H, hd))).astype(np.float32)
        _, sel = nv.sparse_decode(index, 1, q, tabs[:1], [500 * bs], 4, 0, 1)
        assert {300, 310, 499} <= set(sel[0, 0].tolist())


@pytest.mark.parametrize("blocks", [(2049, 5000, 30), (16385, 2100, 41), (32768, 16000, 40), (32769, 32768, 39)], ids=str)
@pytest.mark.parametrize("levels", [0, 2])
def test_selections_of_long_contexts(blocks, levels):
    """Up to 32 blocks a thread of the selection kernel, and the one for more; scores of a few levels or all different."""
    KV, hd, bs, H, top = 1, 4, 1, 2, 40
    tabs, n = oo.tables_for(blocks, bs, seed=67)
    rng = np.random.default_rng(68 + levels)
    held = []
    with nv.PagedKVPool(2, n, bs, KV, hd) as pool, nv.BlockIndex(pool) as index:
        for s, c in enumerate(blocks):
            k = (rng.integers(-levels, levels + 1, (c, KV, hd)) if levels else rng.normal(size=(c, KV, hd))).astype(np.float32)
            v = rng.normal(size=(c, KV, hd)).astype(np.float32)
            nv.norm_rope_append(pool, 1, None, None, k, v, tabs, np.arange(c), np.full(c, s))
            held.append((k, v))
        index.update(1, tabs, [0] * len(blocks), blocks)
        for first, last in ((1, 2), (0, 1)):
            check(pool, index, tabs, held, blocks, H, top, first, last, seed=69)


@pytest.mark.parametrize("geom", [(3, 96, 64), (1, 4, 33), (16, 128, 5), (9, 256, 16), (2, 260 - 4, 7)], ids=lambda g: "x".join(map(str, g)))
@pytest.mark.parametrize("many", [False, True])
def test_bounds_of_rows_of_any_width(geom, many):
    """Few long blocks and many short ones: rows that end inside a workgroup's run of channels, blocks that are full, begun and
    untouched; a NaN in a key stays in its channel."""
    KV, hd, bs = geom
    ctx = [7 * bs + 1, 3 * bs, 1, 0, 2 * bs - 1] + ([bs + 1] * 300 if many else [])
    rng = np.random.default_rng(70)
    tabs, blocks = oo.tables_for(ctx, bs, seed=70)
    want = np.zeros((blocks, KV, 2, hd), np.float32)
    with nv.PagedKVPool(1, blocks, bs, KV, hd) as pool, nv.BlockIndex(pool) as index:
        rows, seqs, pos = [], [], []
        for s, n in enumerate(ctx):
            k = rng.normal(size=(n, KV, hd)).astype(np.float32)
            if s == 1:
                k[bs, KV - 1, hd - 1] = np.nan
            for b in range((n + bs - 1) // bs):
                part = k[b * bs:min(n, (b + 1) * bs)]
                want[tabs[s, b], :, 0], want[tabs[s, b], :, 1] = part.min(0), part.max(0)
            rows.append(k), seqs.append(np.full(n, s)), pos.append(np.arange(n))
        k = np.concatenate(rows)
        nv.norm_rope_append(pool, 0, None, None, k, k, tabs, np.concatenate(pos), np.concatenate(seqs))
        index.update(0, tabs, [0] * len(ctx), ctx)
        assert np.array_equal(bounds_of(index, 0), want, equal_nan=True)


def test_a_reservation_holds_for_every_smaller_call():
    for KV, group, hd, bs in ((1, 4, 32, 16), (2, 7, 64, 4), (2, 3, 256, 16), (1, 20, 128, 1)):
        H = KV * group
        for seqs, ctx, top in ((64, 3000, 300), (5, 9000, 4000), (300, 400, 20)):
            width = (ctx + bs - 1) // bs
            with nv.PagedKVPool(1, 4, bs, KV, hd) as pool, nv.BlockIndex(pool) as index:
                index.reserve_workspace(seqs, H, ctx, top)
                gen = index.workspace_generation
                tabs = DeviceArray(np.zeros((seqs, width), np.int32))
                q, out = (DeviceArray(np.zeros((seqs, H, hd), np.float32)) for _ in range(2))
                for n in sorted({1, 2, 3, 7, 13, seqs // 2, seqs} & set(range(1, seqs + 1))):
                    lens = DeviceArray(np.full(n, 1, np.int32))  # (what counts is the bound given)
                    for c in sorted({1, 100, ctx // 2, ctx}):
                        for t in sorted({1, 5, 16, 65, top // 2, top}):
                            if t <= top:
                                nv.sparse_decode_device(index, 0, n, H, q, tabs, width, lens, c, t, 0, 1, out)
                    pool.synchronize()
                assert index.workspace_generation == gen, (KV, group, hd, bs, seqs, ctx, top)
