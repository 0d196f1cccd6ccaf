"""norm_rope_append into both caches against its definition in 64 bits (operator_oracles.py)."""
import numpy as np
import pytest

import nano_vllm_amd as nv
import operator_oracles as oo
from hipmem import DeviceArray, Stream

pytestmark = pytest.mark.gpu

EPS = 1e-5


def make_pool(cache, blocks, bs, kv, hd):
    return (nv.PagedKVPool if cache == "fp32" else nv.Mx4KVPool)(2, blocks, bs, kv, hd)


def cached_rows(pool, cache, layer, tabs, seqs, pos):
    """(k, v) held for the rows."""
    if cache == "mx4":
        return pool.read_rows(layer, tabs, pos, seqs)
    k = np.zeros((len(pos), pool.n_kv_heads, pool.head_dim), np.float32)
    v = np.zeros_like(k)
    blocks = {}
    for r, (s, p) in enumerate(zip(seqs, pos)):
        if p < 0:
            continue
        b = int(tabs[s, p // pool.block_size])
        if b not in blocks:
            blocks[b] = pool.download_block(layer, b)
        k[r], v[r] = blocks[b][0][p % pool.block_size], blocks[b][1][p % pool.block_size]
    return k, v


def check(got, want, amp, what):
    """fp32 results: rounded once (half a step of fp32 of the value).  Beside it 1e-10 of the row's size: the two sides' angles
    differ by at most pos * freq * 2^-51 < 1e-10 for positions below 2^17, their sums by 2^-50."""
    tol = oo.U * np.abs(want) + 1e-10 * amp + 1e-45
    assert (np.abs(got - want) <= tol).all(), f"{what}: {np.abs(got - want).max():.3e}"


SCALINGS = {"none": nv.ROPE_SCALE_NONE, "linear": nv.ROPE_SCALE_LINEAR, "ntk": nv.ROPE_SCALE_NTK, "yarn": nv.ROPE_SCALE_YARN}

# cache, heads, kv heads, head_dim, rotary_dim, block size, layout, scaling, norm
FORMS = [
    ("fp32", 32, 8, 128, 128, 16, "interleaved", "none", False),
    ("fp32", 32, 8, 128, 128, 16, "half", "yarn", True),
    ("fp32", 6, 6, 48, 48, 16, "half", "linear", True),
    ("fp32", 5, 1, 80, 32, 5, "half", "ntk", False),
    ("fp32", 7, 7, 12, 2, 3, "interleaved", "none", True),
    ("fp32", 2, 2, 256, 64, 16, "half", "none", True),
    ("fp32", 3, 3, 160, 160, 1, "interleaved", "linear", False),
    ("fp32", 12, 4, 32, 32, 8, "half", "none", True),
    ("mx4", 32, 8, 128, 128, 16, "half", "none", True),
    ("mx4", 32, 8, 128, 128, 32, "interleaved", "yarn", False),
    ("mx4", 6, 6, 48, 48, 16, "interleaved", "none", False),
    ("mx4", 6, 6, 48, 16, 48, "half", "linear", True),
    ("mx4", 8, 2, 120, 60, 16, "half", "none", True),
    ("mx4", 3, 3, 56, 56, 16, "half", "none", False),
    ("mx4", 9, 3, 80, 40, 16, "interleaved", "ntk", True),
    ("mx4", 5, 5, 8, 8, 16, "half", "none", True),
    ("mx4", 2, 1, 24, 24, 64, "interleaved", "none", False),
    ("mx4", 4, 2, 256, 128, 16, "half", "yarn", True),
    ("mx4", 3, 1, 200, 200, 16, "half", "none", True),
    ("mx4", 17, 17, 32, 32, 16, "half", "none", False),
]


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(str(x) for x in f))
@pytest.mark.parametrize("rows", [1, 3, 37, 600])
def test_against_definition(form, rows):
    cache, H, KV, hd, rd, bs, layout, scaling, norm = form
    rng = np.random.default_rng(rows * 1000 + hd)
    seqs_n = min(rows, 5)
    seqs = np.sort(np.arange(rows) % seqs_n).astype(np.int32)
    start = rng.integers(0, 4000, seqs_n)
    pos = np.array([start[s] + (i - np.searchsorted(seqs, s)) for i, s in enumerate(seqs)], np.int32)
    tabs, blocks = oo.tables_for([int(pos[seqs == s].max()) + 1 for s in range(seqs_n)], bs, seed=rows)
    q = rng.normal(size=(rows, H, hd)).astype(np.float32)
    k = (rng.normal(size=(rows, KV, hd)) * np.exp(rng.normal(size=(1, KV, hd)))).astype(np.float32)
    v = rng.normal(size=(rows, KV, hd)).astype(np.float32)
    wq, wk = (rng.normal(1, 0.3, hd).astype(np.float32) for _ in range(2)) if norm else (None, None)
    rope = nv.RotaryTable(hd, rd, nv.ROPE_HALF if layout == "half" else nv.ROPE_INTERLEAVED, 10000.0, SCALINGS[scaling], 4.0, 2048)
    freq, m = oo.frequencies(rd, 10000.0, scaling, 4.0, 2048)
    got_f, got_m = rope.frequencies()
    assert np.allclose(got_f, freq, rtol=1e-14, atol=0) and got_m == pytest.approx(m, rel=1e-15)
    with make_pool(cache, blocks, bs, KV, hd) as pool:
        before = cached_rows(pool, cache, 0, tabs, seqs, pos)
        qr = nv.norm_rope_append(pool, 1, rope, q, k, v, tabs, pos, seqs, wq, wk, EPS)
        kc, vc = cached_rows(pool, cache, 1, tabs, seqs, pos)
        after = cached_rows(pool, cache, 0, tabs, seqs, pos)
    assert all((a == 0).all() and (b == 0).all() for a, b in zip(before, after)), "another layer was written"
    qw = oo.norm_rope(q, wq, EPS, pos, freq, m, layout == "half")
    kw = oo.norm_rope(k, wk, EPS, pos, freq, m, layout == "half")
    check(qr, qw, np.abs(qw).max(-1, keepdims=True), "q")
    if cache == "fp32":
        check(kc, kw, np.abs(kw).max(-1, keepdims=True), "k")
        assert (vc == v).all()
    else:
        assert (kc == oo.round4(kw)).all(), "keys are not the nearest codes"
        assert (vc == oo.round4(v)).all(), "values are not the nearest codes"


@pytest.mark.parametrize("cache", ["fp32", "mx4"])
def test_padding_and_places(cache):
    """Rows of padding and rows without a place leave q_out, the cache and every other slot as they were (device form)."""
    H, KV, hd, bs, rows = 4, 2, 64, 16, 6
    rng = np.random.default_rng(5)
    q = rng.normal(size=(rows, H, hd)).astype(np.float32)
    k, v = (rng.normal(size=(rows, KV, hd)).astype(np.float32) for _ in range(2))
    tabs = np.array([[2, 0], [1, 99]], np.int32)
    #       fine, padding, beyond the table, sequence that is not there, block outside the pool, fine
    seqs = np.array([0, 0, 0, 2, 1, 1], np.int32)
    pos = np.array([17, -1, 32, 0, 16, 3], np.int32)
    with make_pool(cache, 3, bs, KV, hd) as pool:
        d = [DeviceArray(x) for x in (q, np.full_like(q, 7), k, v, seqs, pos, tabs)]
        nv.norm_rope_append_device(pool, 0, None, rows, H, d[0], d[1], d[2], d[3], None, None, EPS, d[4], d[5], d[6], 2, 2)
        pool.synchronize()
        out = d[1].numpy()
        assert (out[[0, 5]] == q[[0, 5]]).all() and (out[4] == q[4]).all(), "rows with a place (or only a bad block) pass"
        assert (out[[1, 2, 3]] == 7).all()
        ident = np.arange(3, dtype=np.int32)[:, None]
        s, p = np.repeat(np.arange(3), bs).astype(np.int32), np.tile(np.arange(bs), 3).astype(np.int32)
        kc, vc = cached_rows(pool, cache, 0, ident, s, p)
        f = (lambda x: x) if cache == "fp32" else oo.round4
        want_k, want_v = np.zeros_like(kc), np.zeros_like(vc)
        want_k[0 * bs + 1], want_v[0 * bs + 1] = f(k[0]), f(v[0])
        want_k[1 * bs + 3], want_v[1 * bs + 3] = f(k[5]), f(v[5])
        assert (kc == want_k).all() and (vc == want_v).all()


@pytest.mark.parametrize("cache", ["fp32", "mx4"])
def test_parts_of_the_call(cache):
    """q alone, keys and values alone, in place; no table is needed to rotate queries."""
    H, KV, hd, bs, rows = 6, 3, 48, 16, 40
    rng = np.random.default_rng(6)
    q = rng.normal(size=(rows, H, hd)).astype(np.float32)
    k, v = (rng.normal(size=(rows, KV, hd)).astype(np.float32) for _ in range(2))
    pos = np.arange(rows, dtype=np.int32)
    seqs = np.zeros(rows, np.int32)
    tabs, blocks = oo.tables_for([rows], bs)
    rope = nv.RotaryTable(hd, layout=nv.ROPE_HALF)
    with make_pool(cache, blocks, bs, KV, hd) as pool:
        both = nv.norm_rope_append(pool, 0, rope, q, k, v, tabs, pos, seqs)
        rows0 = cached_rows(pool, cache, 0, tabs, seqs, pos)
        assert nv.norm_rope_append(pool, 1, rope, None, k, v, tabs, pos, seqs) is None
        rows1 = cached_rows(pool, cache, 1, tabs, seqs, pos)
        assert (rows0[0] == rows1[0]).all() and (rows0[1] == rows1[1]).all()
        d, dp = DeviceArray(q), DeviceArray(pos)
        nv.norm_rope_append_device(pool, 0, rope, rows, H, d, d, None, None, None, None, EPS, None, dp, None, 0, 0)
        pool.synchronize()
        assert (d.numpy() == both).all(), "in place, without tables"


def test_matches_the_reference_form():
    """Interleaved, whole head, unscaled: what rope_append_batch does, whose angles are products of fp32 numbers: an angle of up to
    2048 is off by up to 2048 * 2^-23 there, which bounds the difference."""
    H, KV, hd, bs, n = 8, 4, 64, 16, 24
    rng = np.random.default_rng(7)
    q = rng.normal(size=(n, H, hd)).astype(np.float32)
    k, v = (rng.normal(size=(n, KV, hd)).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, 2048, n).astype(np.int32)
    tabs, blocks = oo.tables_for(pos + 1, bs)
    with nv.PagedKVPool(2, blocks, bs, KV, hd) as pool:
        old = pool.rope_append_batch(0, q, k, v, tabs, pos)
        new = nv.norm_rope_append(pool, 1, nv.RotaryTable(hd), q, k, v, tabs, pos)
        assert np.abs(old - new).max() <= 2048 * 2.0 ** -22 * np.abs(q).max() * 2
        a, b = (cached_rows(pool, "fp32", l, tabs, np.arange(n), pos) for l in (0, 1))
        assert np.abs(a[0] - b[0]).max() <= 2048 * 2.0 ** -22 * np.abs(k).max() * 2 and (a[1] == b[1]).all()


def test_codes_of_odd_values():
    """Ties, the largest magnitudes, zeros, tiny and huge rows, infinities and NaN."""
    hd, bs = 64, 16
    rows = [np.zeros(hd), np.full(hd, 1e-44), np.full(hd, 3e38), np.linspace(-7, 7, hd), np.linspace(-6, 6, hd),
            np.tile([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7], 8), -np.tile([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7.0001], 8),
            np.concatenate([np.full(32, 1e-20), np.full(32, 1e20)])]
    bad = np.linspace(-1, 1, hd)
    for i, x in ((3, np.inf), (40, -np.inf), (31, np.nan), (32, np.nan)):
        r = bad.copy()
        r[i] = x
        rows.append(r)
    v = np.array(rows, np.float32)[:, None, :]
    pos = np.arange(len(rows), dtype=np.int32)
    with nv.Mx4KVPool(1, 1, bs, 1, hd) as pool:
        nv.norm_rope_append(pool, 0, None, None, v, v, np.zeros((1, 1), np.int32), pos, np.zeros(len(rows), np.int32))
        k, w = pool.read_rows(0, np.zeros((1, 1), np.int32), pos, np.zeros(len(rows), np.int32))
        want = oo.round4(v.astype(np.float64)).astype(np.float32)
        assert np.array_equal(k, want, equal_nan=True) and np.array_equal(w, want, equal_nan=True)
        # what came out goes in again unchanged; a slot written twice holds the second row
        fine = np.isfinite(want).all((1, 2))
        nv.norm_rope_append(pool, 0, None, None, want[fine], want[fine], np.zeros((1, 1), np.int32), pos[fine], np.zeros(fine.sum(), np.int32))
        k2, w2 = pool.read_rows(0, np.zeros((1, 1), np.int32), pos[fine], np.zeros(fine.sum(), np.int32))
        assert (k2 == want[fine]).all() and (w2 == want[fine]).all()


@pytest.mark.parametrize("cache", ["fp32", "mx4"])
def test_refusals(cache):
    H, KV, hd, bs = 4, 2, 64, 16
    z = lambda *s: np.zeros(s, np.float32)  # noqa: E731
    with make_pool(cache, 4, bs, KV, hd) as pool:
        def call(pos=(0, 1), seqs=(0, 0), tabs=((0, 1),), layer=0, rope=None, q=z(2, H, hd), k=z(2, KV, hd), v=z(2, KV, hd), eps=EPS):
            return nv.norm_rope_append(pool, layer, rope, q, k, v, np.array(tabs, np.int32), np.array(pos, np.int32),
                                       None if seqs is None else np.array(seqs, np.int32), None, None, eps)

        call()
        for kw in (dict(pos=(0, 32)), dict(seqs=(0, 1)), dict(seqs=(0, -1)), dict(tabs=((4, 1),)), dict(tabs=((-1, 1),)), dict(pos=(3, 3)),
                   dict(layer=2), dict(layer=-1), dict(rope=nv.RotaryTable(32)), dict(eps=-1.0), dict(eps=float("nan")),
                   dict(seqs=(0, 1), tabs=((0, 1), (0, 1)), pos=(5, 5))):
            with pytest.raises(nv.NvkError):
                call(**kw)
        for kw in (dict(q=z(3, H, hd)), dict(k=z(2, KV, 32)), dict(k=None), dict(seqs=None), dict(tabs=(0, 1))):
            with pytest.raises(ValueError):
                call(**kw)
        call(pos=(-1, -5))  # padding only
        call(pos=(), seqs=(), q=z(0, H, hd), k=z(0, KV, hd), v=z(0, KV, hd))
        with pytest.raises(nv.NvkError):  # neither queries nor keys
            nv.norm_rope_append(pool, 0, None, None, None, None, np.zeros((1, 1), np.int32), np.zeros(1, np.int32))
    with pytest.raises(RuntimeError):
        call()


@pytest.mark.parametrize("cache", ["fp32", "mx4"])
def test_captured_and_on_another_stream(cache):
    """Replays of a captured call take the positions and rows of the moment, every time the eager result."""
    H, KV, hd, bs, n = 8, 2, 128, 16, 5
    rng = np.random.default_rng(8)
    tabs, blocks = oo.tables_for([200] * n, bs)
    rope = nv.RotaryTable(hd, layout=nv.ROPE_HALF)
    freq, m = oo.frequencies(hd, 10000.0)
    st = Stream()
    from hipmem import _hip, H2D
    import ctypes as C
    with make_pool(cache, blocks, bs, KV, hd) as pool:
        d = {x: DeviceArray(np.zeros((n, h, hd), np.float32)) for x, h in (("q", H), ("o", H), ("k", KV), ("v", KV))}
        dp, dt = DeviceArray(np.zeros(n, np.int32)), DeviceArray(tabs)
        run = lambda: nv.norm_rope_append_device(pool, 0, rope, n, H, d["q"], d["o"], d["k"], d["v"], None, None, EPS, None, dp, dt, n,  # noqa: E731
                                                 tabs.shape[1], st)
        exe = st.capture(run)
        for step in range(3):
            host = {x: rng.normal(size=d[x].shape).astype(np.float32) for x in ("q", "k", "v")}
            pos = rng.integers(0, 200, n).astype(np.int32)
            for a, b in [(d[x], host[x]) for x in host] + [(dp, pos)]:
                assert _hip.hipMemcpy(a.ptr, C.c_void_p(b.ctypes.data), b.nbytes, H2D) == 0
            st.launch(exe)
            st.synchronize()
            want = oo.norm_rope(host["q"], None, EPS, pos, freq, m, True)
            check(d["o"].numpy(), want, np.abs(want).max(-1, keepdims=True), "q")
            k, v = cached_rows(pool, cache, 0, tabs, np.arange(n), pos)
            kw = oo.norm_rope(host["k"], None, EPS, pos, freq, m, True)
            if cache == "mx4":
                assert (k == oo.round4(kw)).all() and (v == oo.round4(host["v"])).all()
            else:
                check(k, kw, np.abs(kw).max(-1, keepdims=True), "k")
                assert (v == host["v"]).all()
    st.close()


@pytest.mark.parametrize("layout", [nv.ROPE_HALF, nv.ROPE_INTERLEAVED])
@pytest.mark.parametrize("turned", [0, 32])
def test_channels_that_do_not_turn_keep_their_values(layout, turned):
    """Infinities, NaN and signed zeros beside each other: nothing of a channel reaches its neighbour."""
    H, KV, hd, bs, n = 3, 2, 64, 16, 20
    rng = np.random.default_rng(12)
    q, k, v = (rng.normal(size=(n, h, hd)).astype(np.float32) for h in (H, KV, KV))
    for x in (q, k):
        x[:, :, 33], x[:, :, 36], x[:, :, 38], x[:, :, 41] = np.inf, -np.inf, np.nan, -0.0
        x[:, :, 40] = -1.0
    tabs, blocks = oo.tables_for([n], bs)
    rope = nv.RotaryTable(hd, turned, layout) if turned else None
    pos, seqs = np.arange(n, dtype=np.int32), np.zeros(n, np.int32)
    with make_pool("fp32", blocks, bs, KV, hd) as pool:
        got = nv.norm_rope_append(pool, 0, rope, q, k, v, tabs, pos, seqs)
        kc, vc = cached_rows(pool, "fp32", 0, tabs, seqs, pos)
    for a, b in ((got, q), (kc, k), (vc, v)):
        a, b = a[..., turned:], b[..., turned:]
        assert np.array_equal(a, b, equal_nan=True) and np.array_equal(np.signbit(a[~np.isnan(a)]), np.signbit(b[~np.isnan(b)]))
        assert np.isfinite(got[..., :turned]).all()


@pytest.mark.parametrize("cache", ["fp32", "mx4"])
def test_rows_at_any_float(cache):
    """Rows, weights and results that start 4 bytes behind a line, device form; sizes and addresses that are refused."""
    H, KV, hd, bs, n = 5, 2, 128, 16, 37
    rng = np.random.default_rng(13)
    q, k, v = (rng.normal(size=(n, h, hd)).astype(np.float32) for h in (H, KV, KV))
    wq, wk = (rng.normal(1, 0.2, hd).astype(np.float32) for _ in range(2))
    tabs, blocks = oo.tables_for([n], bs)
    pos, seqs = np.arange(n, dtype=np.int32), np.zeros(n, np.int32)
    rope = nv.RotaryTable(hd, layout=nv.ROPE_HALF)
    shifted = lambda x: DeviceArray(np.concatenate([np.zeros(1, x.dtype), x.reshape(-1)]))  # noqa: E731
    d = {name: shifted(x) for name, x in (("q", q), ("o", np.zeros_like(q)), ("k", k), ("v", v), ("wq", wq), ("wk", wk))}
    at = {name: x.data_ptr() + 4 for name, x in d.items()}
    i = [DeviceArray(x) for x in (seqs, pos, tabs)]
    with make_pool(cache, blocks, bs, KV, hd) as pool:
        want = nv.norm_rope_append(pool, 0, rope, q, k, v, tabs, pos, seqs, wq, wk, EPS)

        def call(rows=n, heads=H, **kw):
            a = {**at, **kw}
            nv.norm_rope_append_device(pool, 1, rope, rows, heads, a["q"], a["o"], a["k"], a["v"], a["wq"], a["wk"], EPS, *i, 1, tabs.shape[1])

        call()
        pool.synchronize()
        assert (d["o"].numpy()[1:].reshape(q.shape) == want).all()
        rows0, rows1 = (cached_rows(pool, cache, layer, tabs, seqs, pos) for layer in (0, 1))
        assert (rows0[0] == rows1[0]).all() and (rows0[1] == rows1[1]).all()
        for kw in (dict(q=at["q"] + 1), dict(o=at["o"] + 2), dict(k=at["k"] + 3), dict(v=at["v"] + 1), dict(rows=2 ** 31 - 1), dict(rows=-1),
                   dict(heads=2 ** 31 - 1)):
            with pytest.raises(nv.NvkError):
                call(**kw)


def test_far_positions():
    """Positions of a million: the angle's fraction is kept (the two sides' products differ by 2^20 * 2^-52 * pi < 1e-9 of a turn)."""
    H, hd, n = 2, 64, 50
    rng = np.random.default_rng(14)
    q = rng.normal(size=(n, H, hd)).astype(np.float32)
    pos = (2 ** 20 - rng.integers(0, 5000, n)).astype(np.int32)
    freq, m = oo.frequencies(hd, 10000.0)
    want = oo.norm_rope(q, None, EPS, pos, freq, m, True)
    d, dp = DeviceArray(q), DeviceArray(pos)
    with make_pool("fp32", 1, 16, 1, hd) as pool:
        nv.norm_rope_append_device(pool, 0, nv.RotaryTable(hd, layout=nv.ROPE_HALF), n, H, d, d, None, None, None, None, EPS, None, dp, None, 0, 0)
        pool.synchronize()
    assert (np.abs(d.numpy() - want) <= oo.U * np.abs(want) + 2e-9 * np.abs(want).max(-1, keepdims=True)).all()
