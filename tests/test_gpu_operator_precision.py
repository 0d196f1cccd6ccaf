"""What the worst-case bounds of test_gpu_mx4.py and test_gpu_sparse.py cannot notice: that both products of the 4-bit attention take
all three bf16 pieces of a query and of a probability, and that a list cut into many pieces is joined right.

BAR, relative to a call's output by the norm over its rows.  A score is a sum of 3 head_dim products that are exact, in fp32: roundings of
at most half a step U of the partial sum.  Taken as independent they come to sqrt(3 head_dim) U / sqrt(3) of a partial sum (the mean
square of a rounding of up to U is U^2 / 3), 16 U for 256 channels, and scores are two to three units of log2 wide: about 40 U on a
token's share, less where tokens and channels average it; the sums of the second product add less.  32 U = 1.9e-6 is the bar.  A piece that is
lost costs a cut at 16 bits, 2^-16 at most and half of it on average, for a query times the score and for a probability (always
downwards) as it is: 5e-6 and more.  test_the_bar_tells_two_pieces_from_three holds both against a plain emulation."""
import numpy as np
import pytest

import nano_vllm_amd as nv
import operator_oracles as oo
from test_gpu_mx4 import GEOMS
from test_gpu_mx4 import filled as filled_mx4
from test_gpu_sparse import filled as filled_index

BAR = 32 * oo.U


def off(got, want):
    """distance relative to the expected output's size"""
    size = np.linalg.norm(want)
    return np.linalg.norm(np.asarray(got, np.float64) - want) / size if size else float(np.abs(got).max(initial=0.0))


def limits_of(rows, ctx):
    return [[c - n + i + 1 for i in range(n)] for n, c in zip(rows, ctx)]


# ---- on the CPU: what two pieces would come to --------------------------------------------------------------------------
def pieces(x, n):
    """the first n bf16 pieces of x, cut and not rounded"""
    out, rest = [], np.asarray(x, np.float32)
    for _ in range(n):
        cut = (rest.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
        out.append(cut)
        rest = rest - cut
    return out


def emulate(q, k, v, limits, of_q, of_p):
    """attention with of_q and of_p pieces, sums in fp32 eight products at a time"""
    rows, H, hd = q.shape
    g = H // k.shape[1]
    out = np.zeros((rows, H, hd))
    for h in range(H):
        kk, vv = k[:, h // g].astype(np.float64), v[:, h // g].astype(np.float64)
        s = np.zeros((rows, len(kk)), np.float32)
        for piece in pieces(q[:, h] * np.float32(np.log2(np.e) / np.sqrt(hd)), of_q):
            for c in range(0, hd, 8):
                s = (s + piece[:, c:c + 8].astype(np.float64) @ kk[:, c:c + 8].T).astype(np.float32)
        s = np.where(np.arange(len(kk)) < np.asarray(limits)[:, None], s, np.float32(-np.inf))
        p = np.exp2((s - s.max(1, keepdims=True)).astype(np.float64)).astype(np.float32)
        o, total = np.zeros((rows, hd), np.float32), np.zeros((rows, 1), np.float32)
        for t in range(0, len(kk), 8):
            total += p[:, t:t + 8].sum(1, keepdims=True)
            for piece in reversed(pieces(p[:, t:t + 8], of_p)):
                o = (o + piece.astype(np.float64) @ vv[t:t + 8]).astype(np.float32)
        out[:, h] = o / total
    return out


@pytest.mark.parametrize("geom", [(8, 2, 128), (6, 6, 48), (32, 2, 64), (2, 2, 8), (4, 1, 256)], ids=lambda g: "x".join(map(str, g)))
def test_the_bar_tells_two_pieces_from_three(geom):
    H, KV, hd = geom
    rows, ctx = [40, 33], [40, 133]
    rng = np.random.default_rng(hd)
    got = {}
    for n, lim, c in zip(rows, limits_of(rows, ctx), ctx):
        k, v = (oo.round4(rng.normal(size=(c, KV, hd)) * s) for s in (np.exp(0.7 * rng.normal(size=(1, KV, hd))), 1.0))
        q = rng.normal(size=(n, H, hd)).astype(np.float32)
        want, _ = oo.attention(q, k, v, lim)
        for of in ((3, 3), (2, 3), (3, 2)):
            got.setdefault(of, []).append(off(emulate(q, k, v, lim, *of), want))
    assert max(got[3, 3]) <= BAR < min(got[2, 3] + got[3, 2]), got


# ---- the kernels --------------------------------------------------------------------------------------------------------
def check_prefill(geom, rows, ctx, seed):
    H, KV, hd, bs = geom
    pool, tabs, held = filled_mx4(ctx, bs, KV, hd, seed=seed)
    q = np.random.default_rng(seed + 1).normal(size=(sum(rows), H, hd)).astype(np.float32)
    with pool:
        got = nv.mx4_prefill(pool, 1, q, tabs, rows, ctx)
    want, at = [], 0
    for s, (n, lim) in enumerate(zip(rows, limits_of(rows, ctx))):
        want.append(oo.attention(q[at:at + n], *held[s], lim)[0])
        assert n == 0 or off(got[at:at + n], want[-1]) <= BAR, f"sequence {s}: {off(got[at:at + n], want[-1]):.2e}"
        at += n


@pytest.mark.gpu
@pytest.mark.parametrize("geom", GEOMS, ids=lambda g: "x".join(map(str, g)))
def test_prefill_takes_all_pieces(geom):
    check_prefill(geom, [40, 129, 0, 64], [40, 229, 50, 77], seed=81)


@pytest.mark.gpu
@pytest.mark.parametrize("geom", [(2, 2, 128, 16), (4, 2, 64, 32), (6, 2, 48, 16), (1, 1, 256, 16), (8, 2, 128, 16)], ids=lambda g: "x".join(map(str, g)))
def test_prefill_of_a_few_rows_takes_all_pieces(geom):
    """the decode kernel with several rows a sequence, packed and not, whole contexts and pieces of them"""
    check_prefill(geom, [4, 2, 0, 2, 4], [9, 40, 9, 700, 2001], seed=82)


@pytest.mark.gpu
def test_prefill_behind_long_contexts_takes_all_pieces():
    check_prefill((4, 1, 128, 16), [9, 33], [3000, 5001], seed=83)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(4, 2, 32, 4, [9001, 37, 0], 2000), (8, 2, 128, 16, [5000, 3, 900], 100), (12, 2, 64, 8, [4000, 4000], 64),
                                  (4, 2, 256, 16, [3001, 40], 90)], ids=lambda c: "x".join(map(str, c[:4])) + f"-top{c[5]}")
def test_chosen_blocks_against_the_definition(case):
    """Lists in up to 167 pieces, which a kernel of their own joins, beside lines that are written directly, and lists that the attention
    kernel joins; sums of head_dim products where the 4-bit cache has three times as many, so the same bar."""
    H, KV, hd, bs, ctx, top = case
    g = H // KV
    pool, tabs, held = filled_index(ctx, bs, KV, hd, seed=84)
    q = np.random.default_rng(85).normal(size=(len(ctx), H, hd)).astype(np.float32)
    with pool, nv.BlockIndex(pool) as index:
        index.update(1, tabs, [0] * len(ctx), ctx)
        got, sel = nv.sparse_decode(index, 1, q, tabs, ctx, top, 1, 2)
    for s, n in enumerate(ctx):
        score, want = oo.block_scores(q[s], held[s][0], n, bs, KV), np.zeros((H, hd))
        for j in range(KV):
            blocks = oo.choose(score[j], (n + bs - 1) // bs, top, 1, 2)
            assert sel[s, j].tolist() == blocks + [-1] * (top - len(blocks)), f"sequence {s}, kv-head {j}"
            tok = np.array([t for b in blocks for t in range(b * bs, min(n, (b + 1) * bs))], int)
            want[j * g:(j + 1) * g] = oo.attention(q[s:s + 1, j * g:(j + 1) * g], held[s][0][tok, j:j + 1], held[s][1][tok, j:j + 1], [len(tok)])[0][0]
        assert off(got[s], want) <= BAR, f"sequence {s} of {n} tokens: {off(got[s], want):.2e}"
