"""Drafted-token and beam operators where they can go wrong: flat tails far below a peak,
the kernels' variants for large batches, side streams, plans of other pools, scores that
nearly tie.  Bounds are derived from the arithmetic as in tests/test_gpu_spec_ops.py."""

from __future__ import annotations

import math

import numpy as np
import pytest

from conftest import HAS_GPU

pytestmark = pytest.mark.gpu

if HAS_GPU:
    import torch

    import batch_generate as BG
    import paged
    from test_gpu_batch_generate import _model
    from test_gpu_spec_ops import BF16, F16, dev, no_error, raw


# -- tree attention: a flat tail far below one peak ------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("at", [0, 200, 20000])
def test_tree_keeps_a_flat_tail_below_a_peak(dtype, at):
    """One key stands x nats above 39,999 equal ones, whose values do not cancel, in more
    runs than the GPU has SMs, so that one piece of work goes through all of a run.

    Each probability is rounded by h relative; fp16 ones below 2^-14, where the peak's is
    2^7, by 2^-25, which is 2^-32 of the peak's weight each.  Scores are exact up to the
    roundings of the scale, the product and the max (2^-24 of x and the factor's 5 nats, three of
    them and the exponential's own).  The sums of V take 16 positions at a time, 2,501 times
    with one rounding, perhaps towards zero; those of the weights 32 of a tile and 313 tiles."""
    dt = getattr(torch, dtype)
    seqs, hkv, d, ctx, ps = 20, 8, 32, 40000, 16
    cols = ctx // ps + 1
    pool = paged.PagedKVCache(1, seqs * cols, ps, hkv, d, dtype=dt)
    bt = dev(np.random.default_rng(at).permutation(seqs * cols).reshape(seqs, cols))
    g = torch.Generator(device="cuda")
    g.manual_seed(at + 1)
    v = (1.0 + 0.25 * torch.randn(ctx + 1, 1, d, generator=g, device="cuda")).to(dt)
    v[at] = 0.0
    v = v.expand(ctx + 1, hkv, d).contiguous()
    q = torch.zeros(seqs, hkv, d, dtype=dt, device="cuda")
    q[..., 0] = 8.0
    pos = torch.arange(ctx + 1, dtype=torch.int32, device="cuda")
    half = torch.finfo(dt).eps / 2
    plan = pool.plan_tree([ctx] * seqs, [1] * seqs, hkv)
    vals = v[:, 0].double()
    for x in (5.5, 13.0, 15.0, 17.5):
        k = torch.zeros(ctx + 1, hkv, d, dtype=dt, device="cuda")
        k[at, :, 0] = x                                 # 8 x / 8 = x, exactly
        for i in range(seqs):
            pool.append(0, k, v, bt, pos, torch.full_like(pos, i))
        out = torch.zeros_like(q)
        pool.decode_tree(plan, 0, q, None, out, bt, 0.125)
        no_error()
        w = torch.full((ctx + 1,), math.exp(-x), dtype=torch.float64, device="cuda")
        w[at] = 1.0
        w /= w.sum()
        ref, mag = w @ vals, w @ vals.abs()
        rel = 2.0 ** -24 * (4 * (x + 5) + 2 * 2501 + 345) + 2.0 ** -21
        tol = half * ref.abs() + (half + rel) * mag
        if dtype == F16:
            tol += 2.0 ** -32 * w[at] * vals.abs().sum(0) + 2.0 ** -25
        err = (out.double() - ref).abs() - tol
        assert float(err.max()) <= 0, f"{x} nats: over by {float(err.max()):.3g}"
    plan.close()
    pool.close()


# -- the whole layer: a refused call leaves the cache alone ---------------------------------------
def test_refused_layer_calls_launch_nothing():
    cfg, tensors = _model()
    model = BG.BatchModel.from_tensors(cfg, tensors)
    pool = paged.PagedKVCache(cfg.layers, 8, 16, cfg.kv_heads, cfg.head_dim)
    bt, n = dev(np.arange(8).reshape(2, 4)), 3
    x = model.embedding[:n].contiguous()
    out = torch.full_like(x, 7.0)
    for m in raw(pool):
        m.fill_(3.0)
    plan = pool.plan_tree([20], [n], cfg.heads)
    good = dict(plan=plan, layer=0, weights=model.layers[0], mask=None, block_tables=bt)
    others = []
    for layers, ps, hkv, d in ((cfg.layers, 32, cfg.kv_heads, cfg.head_dim),
                               (cfg.layers, 16, 2 * cfg.kv_heads, cfg.head_dim),
                               (cfg.layers, 16, cfg.kv_heads, 2 * cfg.head_dim)):
        o = paged.PagedKVCache(layers, 8, ps, hkv, d)
        others.append((o, o.plan_tree([20], [n], cfg.heads if hkv == cfg.kv_heads else 2 * cfg.heads)))
    off = torch.zeros(model.layers[0].w[6].numel() + 2, dtype=torch.uint8, device="cuda")[2:]
    lw = model.layers[0]
    crooked = paged.DeviceLayerWeights(lw.attn_norm, lw.ffn_norm, list(lw.w[:6]) + [off], lw.types,
                                       lw.hidden, lw.intermediate)
    bad = [dict(plan=p) for _, p in others]
    bad += [dict(layer=cfg.layers), dict(layer=-1), dict(block_tables=bt[:, :1].contiguous()),
            dict(mask=torch.zeros(n, 0, dtype=torch.int32, device="cuda")),
            dict(scale=math.nan), dict(freq_base=0.0), dict(freq_base=math.inf),
            dict(weights=crooked), dict(plan=paged.TreePlan())]
    for change in bad:
        with pytest.raises((ValueError, IndexError)):
            pool.forward_layer_tree(**{**dict(x=x, out=out), **good, **change})
        no_error()
        assert torch.all(out == 7.0), change
        for m in raw(pool):
            assert torch.all(m == 3.0), change
    pool.forward_layer_tree(x=x, out=out, **good)
    no_error()
    assert not torch.any(out == 7.0) and int((raw(pool)[1] != 3.0).sum()) == n * cfg.kv_heads * cfg.head_dim
