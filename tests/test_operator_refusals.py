"""Arguments that norm_rope_append, the 4-bit pool and the block index refuse before any device work (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest

import nano_vllm_amd as nv
from nano_vllm_amd import _capi

lib = _capi.lib
BAD = _capi.ERR_INVALID_ARG


def rope(head_dim=128, rotary=128, layout=0, theta=1e4, scaling=0, factor=1.0, original=0, device=0, out=True):
    h = C.c_void_p()
    rc = lib.nvk_rope_create(head_dim, rotary, layout, theta, scaling, factor, original, device, C.byref(h) if out else None)
    if rc == 0:
        lib.nvk_rope_destroy(h)
    return rc


@pytest.mark.parametrize("kw", [dict(head_dim=0), dict(head_dim=-8), dict(head_dim=258, rotary=258), dict(head_dim=127, rotary=126),
                                dict(rotary=0), dict(rotary=130), dict(rotary=63), dict(layout=2), dict(layout=-1), dict(theta=0.0),
                                dict(theta=-1.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(scaling=4), dict(scaling=-1),
                                dict(scaling=1, factor=0.5), dict(scaling=1, factor=float("nan")), dict(scaling=2, factor=float("inf")),
                                dict(scaling=2, factor=2.0, rotary=2), dict(scaling=3, factor=2.0, original=0), dict(device=-1), dict(out=False)])
def test_rope_create_refuses(kw):
    assert rope(**kw) in (BAD, _capi.ERR_NO_DEVICE if "device" in kw else BAD)
    assert "nvk_rope_create" in _capi.last_error()


@pytest.mark.parametrize("args", [(0, 4, 16, 1, 64), (1, 0, 16, 1, 64), (1, 4, 0, 1, 64), (1, 4, 8, 1, 64), (1, 4, 24, 1, 64),
                                  (1, 4, -16, 1, 64), (1, 4, 16, 0, 64), (1, 4, 16, 1, 0), (1, 4, 16, 1, 12), (1, 4, 16, 1, 264),
                                  (1, 2 ** 31 - 1, 32, 1, 64)])
def test_mx4_pool_create_refuses(args):
    h = C.c_void_p(1)
    assert lib.nvk_mx4_pool_create(*args, 0, C.byref(h)) == BAD
    assert h.value is None and "nvk_mx4_pool_create" in _capi.last_error()
    assert lib.nvk_mx4_pool_create(1, 4, 16, 1, 64, 0, None) == BAD


def test_null_handles():
    x = C.c_void_p()
    one = (C.c_int * 6)()
    assert lib.nvk_mx4_pool_geometry(None, one) == BAD
    assert lib.nvk_mx4_pool_layer_bytes(None) == -1 and lib.nvk_mx4_pool_workspace_generation(None) == -1
    assert lib.nvk_mx4_pool_layer_ptr(None, 0, C.byref(x)) == BAD
    assert lib.nvk_mx4_pool_stream(None, C.byref(x)) == BAD and lib.nvk_mx4_pool_synchronize(None) == BAD
    assert lib.nvk_mx4_pool_reserve_workspace(None, 1, 1, 1, 1, 1) == BAD
    assert lib.nvk_mx4_pool_read_rows(None, 0, 1, None, None, None, 1, 1, None, None, 1, None) == BAD
    for f in (lib.nvk_pool_norm_rope_append, lib.nvk_mx4_pool_norm_rope_append):
        assert f(None, 0, None, 1, 1, *[None] * 6, 1e-5, None, None, None, 1, 1, 1, None) == BAD
    assert lib.nvk_mx4_decode(None, 0, 1, 1, None, None, 1, None, None) == BAD
    assert lib.nvk_mx4_decode_device(None, 0, 1, 1, None, None, 1, None, 1, None, None) == BAD
    assert lib.nvk_mx4_prefill(None, 0, 1, 1, None, None, 1, None, None, None) == BAD
    assert lib.nvk_mx4_prefill_device(None, 0, 1, 1, 1, None, None, 1, None, 1, None, 1, None, None) == BAD
    assert lib.nvk_block_index_create(None, C.byref(x)) == BAD and lib.nvk_block_index_create(None, None) == BAD
    assert lib.nvk_block_index_layer_ptr(None, 0, C.byref(x)) == BAD and lib.nvk_block_index_workspace_generation(None) == -1
    assert lib.nvk_block_index_reserve_workspace(None, 1, 1, 1, 1) == BAD
    assert lib.nvk_block_index_update(None, 0, 1, None, 1, None, None, 1, 1, None) == BAD
    assert lib.nvk_sparse_decode(None, 0, 1, 1, None, None, 1, None, 1, 0, 1, None, None) == BAD
    assert lib.nvk_sparse_decode_device(None, 0, 1, 1, None, None, 1, None, 1, 1, 0, 1, None, None, None) == BAD
    assert lib.nvk_rope_frequencies(None, None, 0, None) == BAD
    # destroying nothing is allowed, as for the other handles
    assert lib.nvk_rope_destroy(None) == 0 and lib.nvk_mx4_pool_destroy(None) == 0 and lib.nvk_block_index_destroy(None) == 0


def test_without_a_device_creation_says_so():
    if nv.device_count() > 0:
        pytest.skip("a device is visible")
    with pytest.raises(nv.NvkError) as e:
        nv.RotaryTable(128)
    assert e.value.code == _capi.ERR_NO_DEVICE
    with pytest.raises(nv.NvkError) as e:
        nv.Mx4KVPool(1, 4, 16, 1, 64)
    assert e.value.code == _capi.ERR_NO_DEVICE


def test_oracle_of_the_format():
    """The 4-bit rounding the GPU tests hold the cache to: every level comes back, ties go to even codes, 7 is not clipped twice."""
    import operator_oracles as oo

    row = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -.5, -6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, .26, .74, 1.26, 1.74, 2.6, 3.4, 5.1, 7, 6.9,
                    -1.25, -2.5, -5, 0, 0, 0])
    want = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -.5, -6, 0, 1, 1, 2, 2, 4, 4, .5, .5, 1.5, 1.5, 3, 3, 6, 6, 6, -1, -2, -4, 0, 0, 0])
    assert (oo.round4(row) == want).all()
    assert (oo.round4(row * 2.0 ** -40) == want * 2.0 ** -40).all()
    row[0] = 7.01  # one step up: the unit is 2 now
    assert oo.round4(row)[0] == 8 and oo.round4(row)[5] == 3 and oo.round4(row)[1] == 0
    x = np.random.default_rng(0).normal(size=(50, 48))
    assert (oo.round4(oo.round4(x)) == oo.round4(x)).all()
