"""Edges of the paged-cache operators that their own files leave out."""
import numpy as np
import pytest

import nano_vllm_amd as nv
import operator_oracles as oo
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
