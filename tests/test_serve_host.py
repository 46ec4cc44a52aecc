"""Host side of head norms with rotation, shared prefixes, summed weights and eviction (no
GPU): the rotation's tables, the refusals that come before any device work, and handles
that touch no device until they are built."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kvcache_ffi as ffi
import paged
from test_spec_host import _pool


def test_rotation_tables():
    r = paged.Rotation(8, 100.0)
    assert (r.rotary_dim, r.pairs, r.axes, r.neox) == (8, 4, 1, True)
    np.testing.assert_allclose(r.inv_freq, 100.0 ** -(np.arange(4) / 4), rtol=1e-15)
    assert r.axis.tolist() == [0] * 4 and r.axis.dtype == np.uint8

    r = paged.Rotation(12, 100.0, [1, 2, 3])
    np.testing.assert_allclose(r.inv_freq, 100.0 ** -(np.arange(6) / 6), rtol=1e-15)
    assert r.axis.tolist() == [0, 1, 1, 2, 2, 2] and r.axes == 3

    # in turns while an axis has pairs left, the first one behind that
    r = paged.Rotation(16, 100.0, [4, 2, 2], order="cyclic", neox=False)
    assert r.axis.tolist() == [0, 1, 2, 0, 1, 2, 0, 0] and not r.neox
    np.testing.assert_allclose(r.inv_freq, 100.0 ** -(np.arange(8) / 8), rtol=1e-15)

    # every axis on a ladder of its own
    r = paged.Rotation(12, 100.0, [3, 0, 3], order="ladders")
    assert r.axis.tolist() == [0, 0, 0, 2, 2, 2]
    np.testing.assert_allclose(r.inv_freq, np.tile(100.0 ** -(np.arange(3) / 3), 2), rtol=1e-15)

    own = [1.0, 0.5, -0.25]
    r = paged.Rotation(6, inv_freq=own)
    own[0] = 7.0
    assert r.inv_freq.tolist() == [1.0, 0.5, -0.25]
    with pytest.raises(ValueError):       # the calls hold its address
        r.inv_freq[0] = 2.0


@pytest.mark.parametrize("bad", [
    dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=-2), dict(rotary_dim=8, freq_base=0.0),
    dict(rotary_dim=8, freq_base=float("inf")), dict(rotary_dim=8, sections=[1, 2]),
    dict(rotary_dim=8, sections=[5, -1]), dict(rotary_dim=8, sections=[]),
    dict(rotary_dim=10, sections=[1] * 5), dict(rotary_dim=8, order="other"),
    dict(rotary_dim=12, sections=[1, 2, 3], order="cyclic"), dict(rotary_dim=8, inv_freq=[1.0] * 3),
    dict(rotary_dim=4, inv_freq=[1.0, float("nan")])])
def test_rotations_that_are_refused(bad):
    with pytest.raises(ValueError):
        paged.Rotation(**bad)


def test_unbuilt_handles_and_null_pools():
    p = paged.SharedPlan()
    assert p.info().n_queries == 0 and p.info().scratch_bytes == 0
    p.close()
    p.close()
    none = ffi.KVC_ERR_INVALID_ARG
    assert ffi.lib.kvc_shared_plan_destroy(None) == ffi.KVC_OK
    assert ffi.lib.kvc_shared_plan_create(None) == none
    assert ffi.lib.kvc_shared_plan_info(None, None, None, None) == none
    assert ffi.lib.kvc_tree_plan_set_weights(None, 1) == none
    assert ffi.lib.kvc_plan_shared(None, None, None, None, 0, None, None, 0, 1, None) == none
    assert ffi.lib.kvc_decode_shared(None, None, 0, None, None, None, 1, 1.0, None) == none
    assert ffi.lib.kvc_decode_tree_weights(None, None, 0, None, None, 0, None, 1, 1, None, None, 1,
                                           1.0, None) == none
    args = ffi.NORM_ROPE_ARGS.pack(*[0] * 12, *[0] * 11, 1e-6)
    assert len(args) == 12 * 8 + 11 * 4 + 4
    assert ffi.lib.kvc_append_norm_rope(None, args, None) == none
    assert ffi.lib.kvc_evict(None, None, 1, 1, None, None, 1, None, None, 1, 1, 1, 0, None,
                             None) == none
    h = ctypes.c_void_p()
    assert ffi.lib.kvc_shared_plan_create(ctypes.byref(h)) == ffi.KVC_OK
    assert ffi.lib.kvc_shared_plan_destroy(h) == ffi.KVC_OK


def test_host_tensors_and_shapes_are_refused_before_any_call():
    pool = _pool()       # 2 layers, 2 KV heads of 64, fp16
    z = lambda *s, t=torch.float16: torch.zeros(s, dtype=t)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    f = lambda *s: torch.zeros(s)  # noqa: E731
    rot = paged.Rotation(64, sections=[16, 16])
    with pytest.raises(ValueError):
        pool.append_norm_rope(0, None, z(3, 2, 64), z(3, 2, 64), i(1, 4), i(3), rot)
    for sizes, prefix, lens in (([2], [0, 16], [20, 20]), ([[2]], [[0]], [20, 20]),
                                ([1 << 40], [0], [20]), ([1], [0], [[20]])):
        with pytest.raises(ValueError):
            pool.plan_shared(lens, sizes, prefix, 4)
    with pytest.raises(ValueError):
        pool.plan_shared([20, 20], [2], [16], 4, rows=[0])
    plan = paged.SharedPlan()
    plan.n_tokens, plan.num_heads = 3, 4
    with pytest.raises(ValueError):
        pool.decode_shared(plan, 0, z(3, 4, 64), z(3, 4, 64), i(3, 4), 0.1)
    plan.close()
    tree = paged.TreePlan()
    tree.n_tokens, tree.num_heads = 3, 4
    with pytest.raises(ValueError):
        pool.decode_tree_weights(tree, 0, z(3, 4, 64), None, f(1, 2, 64), z(3, 4, 64), i(1, 4), 0.1)
    tree.close()
    for kw in (dict(ctx_lens=i(2), weights=f(2, 1, 2, 64), budget=8),                   # rows
               dict(ctx_lens=i(1), weights=f(1, 1, 2, 64), budget=8),                   # layers
               dict(ctx_lens=i(1), weights=f(2, 1, 3, 64), budget=8),                   # KV heads
               dict(ctx_lens=i(1), weights=f(2, 2, 64), budget=8),
               dict(ctx_lens=i(1), weights=f(2, 1, 2, 64), budget=8, weights_out=f(2, 1, 2, 63)),
               dict(ctx_lens=i(1), weights=f(2, 1, 2, 64), budget=8, kept=i(2, 1, 2, 9)),
               dict(ctx_lens=i(1), weights=f(2, 1, 2, 64), budget=8, kept=i(2, 1, 2, 8))):   # host
        with pytest.raises((ValueError, IndexError)):
            pool.evict(i(1, 4), **kw)
