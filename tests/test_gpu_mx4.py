"""Attention over the 4-bit cache against its definition in 64 bits, on the values that the cache holds (operator_oracles.py)."""
import ctypes as C

import numpy as np
import pytest

import nano_vllm_amd as nv
import operator_oracles as oo
from hipmem import H2D, DeviceArray, Stream, _hip

pytestmark = pytest.mark.gpu


def filled(ctx_lens, bs, kv, hd, seed, spread=0.7):
    """(pool, tables, [(k, v) values of each sequence])"""
    rng = np.random.default_rng(seed)
    tabs, blocks = oo.tables_for(ctx_lens, bs, seed)
    pool = nv.Mx4KVPool(2, blocks, bs, kv, hd)
    held = []
    for s, n in enumerate(ctx_lens):
        k = (rng.normal(size=(n, kv, hd)) * np.exp(spread * rng.normal(size=(1, kv, hd)))).astype(np.float32)
        v = rng.normal(size=(n, kv, hd)).astype(np.float32)
        if n:
            nv.norm_rope_append(pool, 1, None, None, k, v, tabs, np.arange(n), np.full(n, s))
        held.append((oo.round4(k), oo.round4(v)))
    return pool, tabs, held


def check_decode(pool, tabs, held, ctx, H, seed, layer=1):
    q = np.random.default_rng(seed + 1).normal(size=(len(ctx), H, pool.head_dim)).astype(np.float32)
    got = nv.mx4_decode(pool, layer, q, tabs, ctx)
    for s, n in enumerate(ctx):
        want, bound = oo.attention(q[s:s + 1], held[s][0][:n], held[s][1][:n], [n])
        err = np.abs(got[s] - want[0])
        assert (err <= bound[0]).all(), f"sequence {s} of {n} tokens: {err.max():.3e}, allowed {bound[0].max():.3e}"
        norm = np.linalg.norm(want)
        assert norm == 0 or np.linalg.norm(got[s] - want[0]) <= 2e-6 * norm  # what sums of exact products come to


GEOMS = [(8, 2, 128, 16), (8, 8, 128, 16), (5, 1, 128, 32), (6, 6, 48, 16), (32, 2, 64, 16), (3, 1, 32, 48), (2, 2, 8, 16), (20, 1, 96, 16),
         (14, 2, 80, 64), (4, 1, 256, 16), (17, 1, 256, 32), (8, 2, 160, 16), (7, 1, 24, 16), (40, 1, 128, 16)]


@pytest.mark.parametrize("geom", GEOMS, ids=lambda g: "x".join(map(str, g)))
def test_decode_lengths(geom):
    H, KV, hd, bs = geom
    ctx = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 511, 700]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=hd + H)
    with pool:
        check_decode(pool, tabs, held, ctx, H, hd)


@pytest.mark.parametrize("geom", [(8, 2, 128, 16), (6, 6, 48, 16), (4, 1, 256, 16)], ids=lambda g: "x".join(map(str, g)))
def test_decode_long(geom):
    """Contexts that are cut into chunks, ragged beside each other."""
    H, KV, hd, bs = geom
    ctx = [6000, 1, 4097, 0, 2500]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=3)
    with pool:
        check_decode(pool, tabs, held, ctx, H, 4)


def test_decode_wide_batch():
    ctx = [int(x) for x in np.random.default_rng(0).integers(0, 90, 300)]
    pool, tabs, held = filled(ctx, 16, 2, 64, seed=9)
    with pool:
        check_decode(pool, tabs, held, ctx, 8, 10)


@pytest.mark.parametrize("geom", GEOMS, ids=lambda g: "x".join(map(str, g)))
@pytest.mark.parametrize("rows", [(1, 3, 0, 17), (40, 129, 1, 64)], ids=str)
def test_prefill(geom, rows):
    H, KV, hd, bs = geom
    ctx = [rows[0], rows[1] + 100, 50, rows[3] + 13]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=hd + 2 * H)
    q = np.random.default_rng(1).normal(size=(sum(rows), H, hd)).astype(np.float32)
    with pool:
        got = nv.mx4_prefill(pool, 1, q, tabs, rows, ctx)
    at = 0
    for s, n in enumerate(rows):
        want, bound = oo.attention(q[at:at + n], *held[s], [ctx[s] - n + i + 1 for i in range(n)])
        err = np.abs(got[at:at + n] - want)
        assert (err <= bound).all(), f"sequence {s}: {err.max():.3e}"
        at += n


def test_prefill_long_context_few_rows():
    """A short chunk behind a long context: columns of one workgroup, tokens cut into chunks."""
    rows, ctx = [9, 33], [3000, 5001]
    pool, tabs, held = filled(ctx, 16, 1, 128, seed=12)
    q = np.random.default_rng(1).normal(size=(sum(rows), 4, 128)).astype(np.float32)
    with pool:
        got = nv.mx4_prefill(pool, 1, q, tabs, rows, ctx)
    at = 0
    for s, n in enumerate(rows):
        want, bound = oo.attention(q[at:at + n], *held[s], [ctx[s] - n + i + 1 for i in range(n)])
        assert (np.abs(got[at:at + n] - want) <= bound).all()
        at += n


def test_large_scores_and_scales():
    """Scores of hundreds (one token takes all) and rows of 1e-18 and 1e18 beside each other."""
    hd, bs, n = 64, 16, 70
    rng = np.random.default_rng(2)
    k, v = rng.normal(size=(n, 1, hd)) * 30, rng.normal(size=(n, 1, hd))
    v[::3] *= 1e18
    v[1::3] *= 1e-18
    k, v = k.astype(np.float32), v.astype(np.float32)
    tabs, blocks = oo.tables_for([n], bs)
    with nv.Mx4KVPool(1, blocks, bs, 1, hd) as pool:
        nv.norm_rope_append(pool, 0, None, None, k, v, tabs, np.arange(n), np.zeros(n, np.int32))
        q = (rng.normal(size=(1, 4, hd)) * 5).astype(np.float32)
        got = nv.mx4_decode(pool, 0, q, tabs, [n])
    want, bound = oo.attention(q, oo.round4(k), oo.round4(v), [n])
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("hd", [48, 128, 256])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_no_number_reaches_only_the_rows_that_see_it(hd, what, bad):
    """A token whose key or value holds no number: rows before it stay clean, rows behind it get NaN (a value: in the channels of
    its group only)."""
    bs, n, at, c = 16, 90, 41, 37
    rng = np.random.default_rng(3)
    k, v = (rng.normal(size=(n, 2, hd)).astype(np.float32) for _ in range(2))
    (k if what == "k" else v)[at, 1, c] = bad
    tabs, blocks = oo.tables_for([n], bs)
    with nv.Mx4KVPool(1, blocks, bs, 2, hd) as pool:
        nv.norm_rope_append(pool, 0, None, None, k, v, tabs, np.arange(n), np.zeros(n, np.int32))
        q = rng.normal(size=(n, 4, hd)).astype(np.float32)
        full = nv.mx4_prefill(pool, 0, q, tabs, [n], [n])
        one = np.stack([nv.mx4_decode(pool, 0, q[i:i + 1], tabs, [i + 1])[0] for i in (at - 1, at, n - 1)])
    for got, pos in ((full, range(n)), (one, (at - 1, at, n - 1))):
        nan = np.isnan(got)
        for r, p in enumerate(pos):
            assert not nan[r, :2].any(), "the other kv-head's queries"
            if p < at:
                assert not nan[r].any(), f"row {p} does not see token {at}"
            elif what == "k":
                assert nan[r, 2:].all()
            else:
                lo, hi = c // 32 * 32, min(c // 32 * 32 + 32, hd)
                assert nan[r, 2:, lo:hi].all() and not nan[r, 2:, :lo].any() and not nan[r, 2:, hi:].any()


def test_stale_blocks_are_not_seen():
    """Tokens behind the context, in the last page and in its tile, hold NaN; table entries behind it point anywhere."""
    bs, hd = 32, 64
    rng = np.random.default_rng(4)
    tabs = np.array([[0, 1, 2]], np.int32)
    with nv.Mx4KVPool(1, 3, bs, 1, hd) as pool:
        k, v = (rng.normal(size=(96, 1, hd)).astype(np.float32) for _ in range(2))
        k[37:], v[37:] = np.nan, np.nan
        nv.norm_rope_append(pool, 0, None, None, k, v, tabs, np.arange(96), np.zeros(96, np.int32))
        q = rng.normal(size=(1, 2, hd)).astype(np.float32)
        for n in (1, 16, 31, 33, 37):
            got = nv.mx4_decode(pool, 0, q, tabs, [n])
            want, bound = oo.attention(q, oo.round4(k[:n]), oo.round4(v[:n]), [n])
            assert (np.abs(got - want) <= bound).all()
        d = [DeviceArray(x) for x in (q, np.array([[0, 1, 1 << 30]], np.int32), np.array([37], np.int32), np.zeros_like(q))]
        nv.mx4_decode_device(pool, 0, 1, 2, d[0], d[1], 3, d[2], 96, d[3])
        pool.synchronize()
        assert (d[3].numpy() == got).all()


def test_device_form_bounds():
    """max_ctx and max_rows above what the lengths need, rows behind the last sequence, bad table entries."""
    bs, hd, KV, H = 16, 128, 2, 8
    ctx, rows = [70, 0, 40], [5, 0, 20]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=21)
    rng = np.random.default_rng(22)
    q = rng.normal(size=(30, H, hd)).astype(np.float32)
    off = np.array([0, 5, 5, 25], np.int32)
    wide = np.full((3, 9), -7, np.int32)
    wide[:, :tabs.shape[1]] = tabs
    with pool:
        dq, do, dw, dc, dof = (DeviceArray(x) for x in (q, np.full_like(q, 5), wide, np.array(ctx, np.int32), off))
        nv.mx4_prefill_device(pool, 1, 3, H, 30, dq, dof, 29, dw, 9, dc, 144, do)
        pool.synchronize()
        got = do.numpy()
        assert (got[25:] == 5).all(), "rows behind the last sequence"
        for s, lo, hi in ((0, 0, 5), (2, 5, 25)):
            n = hi - lo
            want, bound = oo.attention(q[lo:hi], *held[s], [ctx[s] - n + i + 1 for i in range(n)])
            assert (np.abs(got[lo:hi] - want) <= bound).all()
        dd = DeviceArray(np.full((3, H, hd), 5, np.float32))
        nv.mx4_decode_device(pool, 1, 3, H, dq, dw, 9, dc, 2000, dd)
        pool.synchronize()
        got = dd.numpy()
        assert (got[1] == 0).all()
        for s in (0, 2):
            want, bound = oo.attention(q[s:s + 1], *held[s], [ctx[s]])
            assert (np.abs(got[s] - want[0]) <= bound[0]).all()


def test_refusals():
    with nv.Mx4KVPool(2, 4, 16, 2, 64) as pool:
        q = np.zeros((1, 4, 64), np.float32)
        t = np.array([[0, 1]], np.int32)
        nv.mx4_decode(pool, 0, q, t, [20])
        for kw in (dict(ctx=[33]), dict(ctx=[-1]), dict(tabs=[[0, 4]]), dict(tabs=[[-1, 0]]), dict(layer=2), dict(layer=-1),
                   dict(q=np.zeros((1, 3, 64), np.float32))):
            a = dict(layer=0, q=q, tabs=t, ctx=[20])
            a.update(kw)
            with pytest.raises(nv.NvkError):
                nv.mx4_decode(pool, a["layer"], a["q"], np.array(a["tabs"], np.int32), a["ctx"])
        nv.mx4_decode(pool, 0, q, np.array([[0, 99]], np.int32), [16])  # an entry behind the context is not looked at
        with pytest.raises(nv.NvkError):
            nv.mx4_prefill(pool, 0, np.zeros((21, 4, 64), np.float32), t, [21], [20])  # more rows than tokens
        with pytest.raises(nv.NvkError):
            nv.mx4_prefill(pool, 0, q, t, [1], [40])
        for bad in (np.zeros((2, 4, 64), np.float32), np.zeros((1, 4, 32), np.float32), np.zeros((4, 64), np.float32)):
            with pytest.raises(ValueError):
                nv.mx4_decode(pool, 0, bad, t, [20])
        for args in ((0, -1, 4, 1, 1, 16), (0, 1, 3, 1, 1, 16)):
            with pytest.raises(nv.NvkError):
                nv.Mx4KVPool.reserve_workspace(pool, args[1], args[2], args[3], args[5])
        assert nv.mx4_prefill(pool, 0, np.zeros((0, 4, 64), np.float32), t, [0], [20]).shape == (0, 4, 64)
        lib = nv._capi.lib
        d = DeviceArray(np.zeros(4096, np.float32))
        for a in ((0, 1, 4, None, d, 1, d, 16, d), (0, 1, 4, d, None, 1, d, 16, d), (0, 1, 4, d, d, 0, d, 16, d), (0, 1, 4, d, d, 1, d, -1, d),
                  (0, 1, 4, d, d, 2 ** 30, d, 16, d)):
            p = [x.ptr if isinstance(x, DeviceArray) else x for x in a]
            assert lib.nvk_mx4_decode_device(pool.handle, *p, None) == nv._capi.ERR_INVALID_ARG


def test_captured_calls_share_the_workspace():
    """Two graphs (a cut decode, a cut prefill) of one pool, replayed in turn with eager calls between: every replay the eager
    result.  A capture that would have to grow the workspace is refused and leaves the pool usable."""
    bs, hd, KV, H, n = 16, 128, 1, 4, 3
    ctx = [2600, 1700, 900]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=30)
    rng = np.random.default_rng(31)
    rows = [4, 2, 5]
    off = np.array([0, 4, 6, 11], np.int32)
    st = Stream()
    with pool:
        dt, dc, dof = DeviceArray(tabs), DeviceArray(np.array(ctx, np.int32)), DeviceArray(off)
        dq, d1 = DeviceArray(np.zeros((n, H, hd), np.float32)), DeviceArray(np.zeros((n, H, hd), np.float32))
        dp, d2 = DeviceArray(np.zeros((11, H, hd), np.float32)), DeviceArray(np.zeros((11, H, hd), np.float32))
        decode = lambda: nv.mx4_decode_device(pool, 1, n, H, dq, dt, tabs.shape[1], dc, max(ctx), d1, st)  # noqa: E731
        prefill = lambda: nv.mx4_prefill_device(pool, 1, n, H, 11, dp, dof, 5, dt, tabs.shape[1], dc, max(ctx), d2, st)  # noqa: E731
        gen = pool.workspace_generation

        def refused():
            with pytest.raises(nv.NvkError):
                decode()

        st.capture(refused)
        assert pool.workspace_generation == gen
        pool.reserve_workspace(n, H, 1, max(ctx))
        pool.reserve_workspace(n, H, 5, max(ctx), 11)
        gen = pool.workspace_generation
        g1, g2 = st.capture(decode), st.capture(prefill)
        assert pool.workspace_generation == gen
        for step in range(3):
            q1, q2 = (rng.normal(size=(m, H, hd)).astype(np.float32) for m in (n, 11))
            for a, b in ((dq, q1), (dp, q2)):
                assert _hip.hipMemcpy(a.ptr, C.c_void_p(b.ctypes.data), b.nbytes, H2D) == 0
            st.launch(g1)
            st.launch(g2)
            st.synchronize()
            r1, r2 = d1.numpy(), d2.numpy()
            assert (r1 == nv.mx4_decode(pool, 1, q1, tabs, ctx)).all()
            assert (r2 == nv.mx4_prefill(pool, 1, q2, tabs, rows, ctx)).all()
            for s in range(n):
                want, bound = oo.attention(q1[s:s + 1], *held[s], [ctx[s]])
                assert (np.abs(r1[s] - want[0]) <= bound[0]).all()
    st.close()


def test_generation_together():
    """A prompt in two chunks, then decode steps, all through the 4-bit cache: rows normed, rotated, stored and attended to as
    a model's layer does it, against the same in 64 bits."""
    H, KV, hd, bs, prompt, steps = 8, 2, 128, 16, (37, 50), 12
    rng = np.random.default_rng(40)
    total = prompt[1] + steps
    q, k, v = (rng.normal(size=(total, n, hd)).astype(np.float32) for n in (H, KV, KV))
    wq, wk = (rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2))
    rope = nv.RotaryTable(hd, 64, nv.ROPE_HALF, scaling=nv.ROPE_SCALE_YARN, factor=4.0, original_len=64)
    freq, m = oo.frequencies(64, 10000.0, "yarn", 4.0, 64)
    pos = np.arange(total)
    q64 = oo.norm_rope(q, wq, 1e-5, pos, freq, m, True)
    k4, v4 = oo.round4(oo.norm_rope(k, wk, 1e-5, pos, freq, m, True)), oo.round4(v)
    tabs, blocks = oo.tables_for([total], bs)
    want, bound = oo.attention(q64, k4, v4, pos + 1)
    # q arrives rounded to fp32: half a step of each element, in the scores
    bound = bound + 2 * oo.U * np.abs(q64).max() * np.abs(k4).max() * hd ** 0.5 * np.abs(v4).max()
    got = np.zeros_like(want)
    with nv.Mx4KVPool(1, blocks, bs, KV, hd) as pool:
        for lo, hi in ((0, prompt[0]), (prompt[0], prompt[1])):
            qr = nv.norm_rope_append(pool, 0, rope, q[lo:hi], k[lo:hi], v[lo:hi], tabs, pos[lo:hi], np.zeros(hi - lo, np.int32), wq, wk)
            got[lo:hi] = nv.mx4_prefill(pool, 0, qr, tabs, [hi - lo], [hi])
        for t in range(prompt[1], total):
            qr = nv.norm_rope_append(pool, 0, rope, q[t:t + 1], k[t:t + 1], v[t:t + 1], tabs, [t], None, wq, wk)
            got[t:t + 1] = nv.mx4_decode(pool, 0, qr, tabs, [t + 1])
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()


@pytest.mark.parametrize("geom", [(2, 2, 128, 16), (4, 2, 64, 32), (6, 2, 48, 16), (1, 1, 256, 16), (8, 2, 128, 16)], ids=lambda g: "x".join(map(str, g)))
@pytest.mark.parametrize("most", [2, 4])
def test_prefill_of_a_few_rows(geom, most):
    """Chunks of up to 16 columns, rows behind short and long contexts beside each other (whole and cut into pieces)."""
    H, KV, hd, bs = geom
    rows, ctx = [1, most, 0, 2, most], [1, most, 9, 700, 2001]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=hd + H)
    q = np.random.default_rng(most).normal(size=(sum(rows), H, hd)).astype(np.float32)
    with pool:
        got = nv.mx4_prefill(pool, 1, q, tabs, rows, ctx)
    at = 0
    for s, n in enumerate(rows):
        want, bound = oo.attention(q[at:at + n], *held[s], [ctx[s] - n + i + 1 for i in range(n)])
        err = np.abs(got[at:at + n] - want)
        assert (err <= bound).all(), f"sequence {s}: {err.max():.3e}"
        at += n


def test_more_pieces_than_one_workgroup_joins():
    """Contexts of about 100 pieces beside contexts of one and of none, decode and two rows each."""
    ctx = [9300, 40, 8200, 0, 1000]
    pool, tabs, held = filled(ctx, 16, 1, 32, seed=33)
    with pool:
        check_decode(pool, tabs, held, ctx, 4, 34)
        rows = [2, 2, 1, 0, 2]
        q = np.random.default_rng(35).normal(size=(sum(rows), 4, 32)).astype(np.float32)
        got = nv.mx4_prefill(pool, 1, q, tabs, rows, ctx)
    at = 0
    for s, n in enumerate(rows):
        want, bound = oo.attention(q[at:at + n], *held[s], [ctx[s] - n + i + 1 for i in range(n)])
        assert (np.abs(got[at:at + n] - want) <= bound).all()
        at += n


def test_stale_values_of_any_size_are_not_seen():
    """Behind the context the last page holds the largest fp32 numbers: stored as finite ones, and none reaches a row."""
    bs, hd, n = 32, 64, 96
    rng = np.random.default_rng(5)
    big = np.float32(3.4028234e38)
    tabs = np.array([[0, 1, 2]], np.int32)
    with nv.Mx4KVPool(1, 3, bs, 1, hd) as pool:
        k, v = (rng.normal(size=(n, 1, hd)).astype(np.float32) for _ in range(2))
        k[37:], v[37:] = big, -big
        nv.norm_rope_append(pool, 0, None, None, k, v, tabs, np.arange(n), np.zeros(n, np.int32))
        kc, vc = pool.read_rows(0, tabs, np.arange(n), np.zeros(n, np.int32))
        assert (kc[37:] == np.float32(6 * 2.0 ** 125)).all() and (vc[37:] == np.float32(-6 * 2.0 ** 125)).all()
        q = rng.normal(size=(17, 2, hd)).astype(np.float32)
        for c in (1, 31, 33, 37):
            got = nv.mx4_decode(pool, 0, q[:1], tabs, [c])
            want, bound = oo.attention(q[:1], oo.round4(k[:c]), oo.round4(v[:c]), [c])
            assert (np.abs(got - want) <= bound).all()
        got = nv.mx4_prefill(pool, 0, q, tabs, [17], [37])
        want, bound = oo.attention(q, oo.round4(k[:37]), oo.round4(v[:37]), np.arange(21, 38))
        assert (np.abs(got - want) <= bound).all()


def test_operands_at_any_float():
    """q, results and rows that start 4 bytes behind a line: whole contexts, joined pieces, many rows; addresses that are refused."""
    KV, hd, bs, H = 2, 128, 16, 8
    ctx, rows = [700, 3, 90], [1, 2, 30]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=36)
    rng = np.random.default_rng(37)
    q = rng.normal(size=(33, H, hd)).astype(np.float32)
    shifted = lambda x: DeviceArray(np.concatenate([np.zeros(1, x.dtype), x.reshape(-1)]))  # noqa: E731
    dq, do, dk, dv = shifted(q), shifted(np.zeros_like(q)), shifted(np.zeros((5, KV, hd), np.float32)), shifted(np.zeros((5, KV, hd), np.float32))
    dt, dc, dof, dp = (DeviceArray(x) for x in (tabs, np.array(ctx, np.int32), np.array([0, 1, 3, 33], np.int32), np.arange(5, dtype=np.int32)))
    ds = DeviceArray(np.zeros(5, np.int32))
    p = lambda x: x.data_ptr() + 4  # noqa: E731
    back = lambda x, shape: x.numpy()[1:1 + int(np.prod(shape))].reshape(shape)  # noqa: E731
    with pool:
        for n in (1, 3):  # one sequence: pieces joined inside
            nv.mx4_decode_device(pool, 1, n, H, p(dq), dt, tabs.shape[1], dc, max(ctx), p(do))
            pool.synchronize()
            assert (back(do, (n, H, hd)) == nv.mx4_decode(pool, 1, q[:n], tabs[:n], ctx[:n])).all()
        nv.mx4_prefill_device(pool, 1, 3, H, 33, p(dq), dof, 30, dt, tabs.shape[1], dc, max(ctx), p(do))
        pool.synchronize()
        assert (back(do, (33, H, hd)) == nv.mx4_prefill(pool, 1, q, tabs, rows, ctx)).all()
        pool.read_rows_device(1, 5, ds, dp, dt, 3, tabs.shape[1], p(dk), p(dv))
        pool.synchronize()
        assert (back(dk, (5, KV, hd)) == held[0][0][:5]).all() and (back(dv, (5, KV, hd)) == held[0][1][:5]).all()
        for a, b in ((p(dq) + 1, p(do)), (p(dq), p(do) + 2)):
            with pytest.raises(nv.NvkError):
                nv.mx4_decode_device(pool, 1, 3, H, a, dt, tabs.shape[1], dc, max(ctx), b)
            with pytest.raises(nv.NvkError):
                nv.mx4_prefill_device(pool, 1, 3, H, 33, a, dof, 30, dt, tabs.shape[1], dc, max(ctx), b)
            with pytest.raises(nv.NvkError):
                pool.read_rows_device(1, 5, ds, dp, dt, 3, tabs.shape[1], a, b)
        with pytest.raises(nv.NvkError):
            nv.mx4_decode_device(pool, 1, 3, H, dq, dt, tabs.shape[1], dc, 2 ** 31 - 1, do)


def test_a_layer_of_more_than_32_bits():
    """Blocks that lie beyond 4 GiB of a layer hold and answer what the first ones do."""
    KV, hd, bs, H, n = 8, 128, 16, 16, 75
    blocks = 260_000  # 17408 bytes each
    rng = np.random.default_rng(38)
    k, v = (rng.normal(size=(n, KV, hd)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(n, H, hd)).astype(np.float32)
    low = np.array([[3, 0, 4, 1, 2]], np.int32)
    high = blocks - 1 - low
    got = []
    with nv.Mx4KVPool(1, blocks, bs, KV, hd) as pool:
        assert pool.layer_bytes > 2 ** 32
        for tabs in (low, high):
            nv.norm_rope_append(pool, 0, None, None, k, v, tabs, np.arange(n), np.zeros(n, np.int32))
            got.append((pool.read_rows(0, tabs, np.arange(n), np.zeros(n, np.int32)), nv.mx4_decode(pool, 0, q[:1], tabs, [n]),
                        nv.mx4_prefill(pool, 0, q, tabs, [n], [n])))
    (r0, d0, p0), (r1, d1, p1) = got
    assert (r0[0] == oo.round4(k)).all() and (r1[0] == r0[0]).all() and (r1[1] == r0[1]).all()
    assert (d0 == d1).all() and (p0 == p1).all()


def test_two_pools_at_once_and_shared_blocks():
    """Calls on two pools, each on a stream of its own, overlap; sequences of one batch share their first blocks."""
    KV, hd, bs, H, n = 1, 128, 16, 4, 3
    rng = np.random.default_rng(39)
    streams = [Stream(), Stream()]
    sets = []
    for i in range(2):
        k, v = (rng.normal(size=(2600, KV, hd)).astype(np.float32) for _ in range(2))
        base, blocks = oo.tables_for([2600], bs, seed=i)
        tabs, ctx = np.repeat(base, n, 0), np.array([2600, 1333, 16 * 50], np.int32)
        pool = nv.Mx4KVPool(1, blocks, bs, KV, hd)
        nv.norm_rope_append(pool, 0, None, None, k, v, base, np.arange(2600), np.zeros(2600, np.int32))
        q = rng.normal(size=(n, H, hd)).astype(np.float32)
        want = nv.mx4_decode(pool, 0, q, tabs, ctx)
        for s in range(n):
            w, bound = oo.attention(q[s:s + 1], oo.round4(k), oo.round4(v), [ctx[s]])
            assert (np.abs(want[s] - w[0]) <= bound[0]).all()
        d = [DeviceArray(x) for x in (q, tabs, ctx, np.zeros_like(q))]
        sets.append((pool, d, want, tabs))
    for turn in range(20):
        for (pool, d, _, tabs), st in zip(sets, streams):
            nv.mx4_decode_device(pool, 0, n, H, d[0], d[1], tabs.shape[1], d[2], 2600, d[3], st)
    for (pool, d, want, _), st in zip(sets, streams):
        st.synchronize()
        assert (d[3].numpy() == want).all()
        pool.close()
        st.close()


def test_a_reservation_holds_for_every_smaller_call():
    """Fewer sequences are cut into more pieces: after one reservation nothing up to that shape moves the workspace."""
    for KV, group, hd in ((1, 4, 32), (2, 7, 64), (2, 1, 256), (1, 20, 128)):
        H = KV * group
        for seqs, rows, ctx in ((64, 1, 3000), (40, 6, 9000), (6, 500, 2000)):
            with nv.Mx4KVPool(1, 600, 16, KV, hd) as pool:
                pool.reserve_workspace(seqs, H, rows, ctx, seqs * rows)
                gen = pool.workspace_generation
                tabs = DeviceArray(np.zeros((seqs, 600), np.int32))
                q, out = (DeviceArray(np.zeros((seqs * rows, H, hd), np.float32)) for _ in range(2))
                for n in sorted({1, 2, 3, 7, 13, seqs // 2, seqs} & set(range(1, seqs + 1))):
                    for c in sorted({1, 100, 700, ctx // 2, ctx}):
                        lens = DeviceArray(np.full(n, 1, np.int32))  # (what counts is the bound given)
                        nv.mx4_decode_device(pool, 0, n, H, q, tabs, 600, lens, c, out)
                        for r in sorted({1, 2, 5, rows // 2, rows} & set(range(1, rows + 1))):
                            off = DeviceArray(np.arange(n + 1, dtype=np.int32))
                            nv.mx4_prefill_device(pool, 0, n, H, n * r, q, off, r, tabs, 600, lens, c, out)
                            pool.synchronize()
                assert pool.workspace_generation == gen, (KV, group, hd, seqs, rows, ctx)


def test_a_padded_batch_of_rows():
    """Far more rows than the sequences' chunks can hold: they are left as they were and take no workspace."""
    KV, H, hd, bs = 1, 4, 128, 16
    ctx, rows = [2500, 900], [3, 5]
    pool, tabs, held = filled(ctx, bs, KV, hd, seed=41)
    q = np.random.default_rng(42).normal(size=(4000, H, hd)).astype(np.float32)
    dq, do, dt, dc, dof = (DeviceArray(x) for x in (q, np.full_like(q, 5), tabs, np.array(ctx, np.int32), np.array([0, 3, 8], np.int32)))
    with pool:
        pool.reserve_workspace(2, H, 5, max(ctx), 4000)
        gen = pool.workspace_generation
        nv.mx4_prefill_device(pool, 1, 2, H, 4000, dq, dof, 5, dt, tabs.shape[1], dc, max(ctx), do)
        pool.synchronize()
        assert pool.workspace_generation == gen
        got = do.numpy()
    assert (got[8:] == 5).all()
    for s, lo, hi in ((0, 0, 3), (1, 3, 8)):
        n = hi - lo
        want, bound = oo.attention(q[lo:hi], *held[s], [ctx[s] - n + i + 1 for i in range(n)])
        assert (np.abs(got[lo:hi] - want) <= bound).all()
