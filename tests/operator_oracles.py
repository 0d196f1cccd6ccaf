"""Plain 64-bit definitions of the paged-cache operators (numpy), for the tests of norm_rope_append, the 4-bit cache and the
block-sparse decode."""
import math

import numpy as np

U = 2.0 ** -24  # half a step of fp32, relative
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def frequencies(rotary_dim, theta, scaling="none", factor=1.0, original_len=0):
    i = np.arange(0, rotary_dim, 2, dtype=np.float64)
    if scaling == "ntk":
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    f = theta ** (-i / rotary_dim)
    m = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        keep = np.clip((original_len * f / (2 * math.pi) - 1) / 31, 0, 1)
        f = (1 - keep) * f / factor + keep * f
        m = 0.1 * math.log(factor) + 1
    return f, m


def norm_rope(x, weight, eps, pos, freq, m, half):
    """x [rows, heads, hd] -> float64; freq None: no rotation."""
    y = np.asarray(x, np.float64).copy()
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + float(np.float32(eps))) * np.asarray(weight, np.float64)
    if freq is None:
        return y
    r = 2 * len(freq)
    ang = np.asarray(pos, np.float64)[:, None] * freq[None, :]
    c, s = (m * np.cos(ang))[:, None, :], (m * np.sin(ang))[:, None, :]
    ia, ib = (np.arange(r // 2), np.arange(r // 2) + r // 2) if half else (np.arange(0, r, 2), np.arange(1, r, 2))
    a, b = y[..., ia].copy(), y[..., ib].copy()
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    return y


def round4(x):
    """The values a 4-bit cache holds for rows x [..., hd]."""
    x = np.asarray(x, np.float64)
    out = np.zeros_like(x)
    for lo in range(0, x.shape[-1], 32):
        p = x[..., lo:lo + 32]
        finite = (np.abs(p) < 2.0 ** 128).all(-1, keepdims=True)  # (False for a NaN)
        a = np.abs(np.where(finite, p, 0.0))
        top = a.max(-1, keepdims=True)
        man, ex = np.frexp(top)  # top = man * 2^ex, man in [0.5, 1)
        e = np.where(man <= 0.875, ex - 3, ex - 2)
        e = np.where(top == 0, -126, np.clip(e, -126, 125))
        z = np.ldexp(a, -e)
        code = ((z > 0.25).astype(int) + (z >= 0.75) + (z > 1.25) + (z >= 1.75) + (z > 2.5) + (z >= 3.5) + (z > 5.0))
        val = np.ldexp(LEVELS[code], np.broadcast_to(e, code.shape)) * np.where(p < 0, -1.0, 1.0)
        out[..., lo:lo + 32] = np.where(finite, val, np.nan)
    return out


def attention(q, k, v, limits):
    """q [rows, H, hd], k / v [T, KV, hd]; row r sees tokens below limits[r].  Returns (out, bound on |error|) where the bound is that
    of fp32 sums of exact products: see attention_bound."""
    rows, H, hd = q.shape
    KV = k.shape[1]
    g = H // KV
    out, bound = np.zeros((rows, H, hd)), np.zeros((rows, H, hd))
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    for r in range(rows):
        n = int(limits[r])
        if n <= 0:
            continue
        for h in range(H):
            kk, vv = k[:n, h // g], v[:n, h // g]
            x = kk @ q[r, h] / math.sqrt(hd)
            p = np.exp(x - x.max())
            p /= p.sum()
            out[r, h] = p @ vv
            # a score: 3 hd exact products summed in fp32, then one rounding of scale, one of the product and one of the
            # difference from the maximum; twice, since numerator and denominator both carry it
            ds = (3 * hd + 4) * U * (np.abs(kk) @ np.abs(q[r, h]) / math.sqrt(hd)).max() + 4 * U * np.abs(x).max()
            # exp2 (2 steps of fp32), rescaling and joins (8), and a sum over n tokens, for numerator and denominator
            bound[r, h] = (2 * ds + (2 * n + 16) * U) * (p @ np.abs(vv)) + 1e-38
    return out, bound


def block_scores(q, k, ctx, bs, n_kv):
    """[kv, blocks] fp32 scores of one sequence: q [H, hd], k [ctx, KV, hd]."""
    nb = (ctx + bs - 1) // bs
    g = q.shape[0] // n_kv
    q64 = np.asarray(q, np.float64)
    s = np.zeros((n_kv, nb))
    for b in range(nb):
        blk = np.asarray(k[b * bs:min(ctx, (b + 1) * bs)], np.float64)
        lo, hi = blk.min(0), blk.max(0)
        for j in range(n_kv):
            qq = q64[j * g:(j + 1) * g]
            s[j, b] = (np.maximum(qq, 0) @ hi[j] + np.minimum(qq, 0) @ lo[j]).max()
    return s.astype(np.float32)


def choose(scores, nb, top, first, last):
    """Blocks read for one kv-head: first and last ones, then the best, equal scores lowest first; ascending."""
    if nb <= top:
        return list(range(nb))
    must = sorted(set(range(first)) | set(range(nb - last, nb)))
    rest = [b for b in range(nb) if b not in set(must)]
    rest.sort(key=lambda b: (-float(scores[b]), b))
    return sorted(must + rest[:top - len(must)])


def tables_for(ctx_lens, bs, seed=0, spare=3, width=None):
    """Fragmented block tables and the pool size they need; unused entries hold -1."""
    need = [(int(c) + bs - 1) // bs for c in ctx_lens]
    total = sum(need) + spare
    perm = np.random.default_rng(seed).permutation(total).astype(np.int32)
    w = max(max(need), 1) if width is None else width
    tabs = np.full((len(need), w), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        tabs[s, :n] = perm[at:at + n]
        at += n
    return tabs, total
