"""Host side of the drafted-token and beam operators (no GPU): mask rows of drafted
trees, the argument errors that come before any device work, and the handles that
touch no device until they are built."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import beam
import kvcache_ffi as ffi
import paged


def test_tree_masks_and_depths():
    par = [-1, 0, 0, 1, -1, 4, 3]
    m = paged.tree_masks(par)
    assert m.dtype == np.int32 and m.shape == (7, 1)
    see = [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {4}, {4, 5}, {0, 1, 3, 6}]
    assert [{j for j in range(7) if int(m[i, 0]) >> j & 1} for i in range(7)] == see
    assert paged.tree_depths(par).tolist() == [0, 1, 1, 2, 0, 1, 3]
    chain = paged.tree_masks(range(-1, 255)).view(np.uint32)     # 256 nodes, bit 31 among them
    assert chain.shape == (256, 8) and np.all(chain[255] == 0xFFFFFFFF)
    assert int(chain[31, 0]) == 0xFFFFFFFF and not chain[31, 1:].any()
    assert paged.tree_masks([], 2).shape == (0, 2)
    assert paged.tree_masks([-1], 3).shape == (1, 3)
    for bad in ([0], [-1, 1], [-2], list(range(-1, 256))):
        with pytest.raises(ValueError):
            paged.tree_masks(bad)
    with pytest.raises(ValueError):
        paged.tree_masks([-1] * 33, words=1)


def test_unbuilt_handles():
    p = paged.TreePlan()
    info = p.info()
    assert (info.n_queries, info.scratch_bytes) == (0, 0)
    p.close()
    p.close()
    assert ffi.lib.kvc_tree_plan_destroy(None) == ffi.KVC_OK
    assert ffi.lib.kvc_beam_destroy(None) == ffi.KVC_OK
    assert ffi.lib.kvc_tree_plan_create(None) == ffi.KVC_ERR_INVALID_ARG
    assert ffi.lib.kvc_tree_plan_info(None, None, None, None) == ffi.KVC_ERR_INVALID_ARG


def test_null_pools_and_bad_beam_sizes():
    h = ctypes.c_void_p()
    none = ffi.KVC_ERR_INVALID_ARG
    assert ffi.lib.kvc_append_rope(None, 0, None, 0, None, 0, None, 0, None, 0, None, 1, 1, None,
                                   None, None, 0, 1e4, 0, None) == none
    assert ffi.lib.kvc_plan_tree(None, None, None, None, None, 0, 1, None) == none
    assert ffi.lib.kvc_decode_tree(None, None, 0, None, None, 0, None, None, 1, 1.0, None) == none
    assert ffi.lib.kvc_commit_tree(None, None, 1, 1, None, None, None, 1, None, 1, None) == none
    assert ffi.lib.kvc_reorder_beams(None, None, 1, None, None, 1, 1, None) == none
    assert ffi.lib.kvc_beam_select(None, None, 0, 0, None, 1, 1, 1, 1, None, None, None,
                                   None) == none
    assert ffi.lib.kvc_beam_create(1, 1, 1, 1, 0, None) == none
    for bad in ((0, 1, 9, 1), (1, 0, 9, 1), (1, 17, 9, 1), (1, 1, 0, 1), (1, 1, 9, 0),
                (1, 1, 9, 33), (5000, 16, 9, 1), (1, 1, 1 << 27, 1)):
        assert ffi.lib.kvc_beam_create(*bad, 0, ctypes.byref(h)) == none
        assert not h.value


def _pool():
    p = paged.PagedKVCache.__new__(paged.PagedKVCache)      # geometry only, nothing native
    p.handle, p.num_layers, p.num_pages, p.page_size = None, 2, 8, 16
    p.num_kv_heads, p.head_dim, p.dtype, p.device = 2, 64, torch.float16, 0
    return p


def test_host_tensors_are_refused_before_any_call():
    pool = _pool()
    z = lambda *s, t=torch.float16: torch.zeros(s, dtype=t)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        pool.append_rope(0, None, z(3, 2, 64), z(3, 2, 64), i(1, 4), i(3))
    plan = paged.TreePlan()
    plan.n_tokens, plan.num_heads = 3, 4
    with pytest.raises(ValueError):
        pool.decode_tree(plan, 0, z(3, 4, 64), None, z(3, 4, 64), i(1, 4), 0.1)
    with pytest.raises(ValueError):
        pool.decode_tree(plan, 0, z(3, 4, 64), i(3), z(3, 4, 64), i(1, 4), 0.1)   # a flat mask
    with pytest.raises(ValueError):
        pool.commit_tree(i(1, 4), i(1), i(1, 2), i(1))
    with pytest.raises(ValueError):
        pool.commit_tree(i(1, 4), i(1), i(2), i(1))
    with pytest.raises(ValueError):
        pool.reorder_beams(i(4, 4), i(1, 4), i(1))
    with pytest.raises(ValueError):
        pool.reorder_beams(i(3, 4), i(1, 4), i(1))                                # rows and beams
    with pytest.raises(ValueError):
        pool.plan_tree([1, 2], [3], 4)
    sel = beam.BeamSelector.__new__(beam.BeamSelector)
    sel.handle, sel.device = None, 0
    for logits, scores in ((z(4, 9), z(2, 2, t=torch.float32)), (z(4, 9, t=torch.int32), z(2, 2)),
                           (z(3, 9), z(2, 2)), (z(9), z(2, 2)), (z(4, 9), z(4))):
        with pytest.raises(ValueError):
            sel.select(logits, scores, 2)
    plan.close()


class _Geometry:
    num_layers = 2
    page_size = 16


def test_decoder_checks_trees_paths_and_parents_first():
    bt = torch.zeros((3, 4), dtype=torch.int32)
    dec = paged.BatchDecoder(_Geometry(), [object(), object()], bt, 8, [10, 62, 62])
    x = lambda n: torch.zeros((n, 16), dtype=torch.float16)  # noqa: E731
    with pytest.raises(ValueError):
        dec.verify(x(1), [[-1]])                          # one tree per sequence
    with pytest.raises(ValueError):
        dec.verify(x(2), [[-1], [], []])                  # one row per token
    with pytest.raises(ValueError):
        dec.verify(x(1), [[0], [], []])                   # its own parent
    with pytest.raises(IndexError):
        dec.verify(x(3), [[], [-1, 0, 1], []])            # 62 + 3 > 64
    with pytest.raises(RuntimeError):
        dec.commit([[], [], []])
    assert dec.verify(x(0), [[], [], []]).shape[0] == 0
    with pytest.raises(ValueError):
        dec.commit([[0], [], []])                         # nothing was drafted
    dec.commit([[], [], []])
    assert list(dec.ctx) == [10, 62, 62]
    for bad in ([[0, 1]], [0, 1, 2], [[0, 1, 3]], [[0, -1, 1]], [[0, 1, 2]]):
        with pytest.raises(ValueError):
            dec.reorder(bad)                              # (the last: lengths differ)
    dec.close()
