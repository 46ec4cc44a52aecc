"""Summed attention weights where something went wrong on the way: pages out of range and
waits that gave up.  The sums are kept over many steps, so nothing may come into them that the
call did not compute.  References and tolerances as in test_gpu_serve_ops."""

from __future__ import annotations

import math

import numpy as np
import pytest

from conftest import HAS_GPU

pytestmark = pytest.mark.gpu

if HAS_GPU:
    import torch

    import kvcache_ffi as ffi

from test_gpu_serve_ops import BAD_PAGE, attend64, check
from test_gpu_spec_ops import BF16, F16, F32, dev, make_pool, no_error

WAIT_LIMIT = 2           # KVC_DEVERR_*
BAD = 1 << 20            # no pool here has as many pages


def weighed(dtype, d, h, hkv, ps, ctx, seed):
    """(pool, table, weights, lengths with the token): one token of each sequence."""
    n = [c + 1 for c in ctx]
    width = max(-(-x // ps) for x in n)
    pool = make_pool(1, len(ctx) * width, ps, hkv, d, dtype, fill=0.0)
    pool.fill_normal(seed=seed)
    table = np.random.default_rng(seed).permutation(len(ctx) * width).reshape(len(ctx), width)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    weights = torch.rand(len(ctx), hkv, max(n), generator=g, device="cuda")
    return pool, table, weights, n


# D, H, Hkv, page, contexts, bad (sequence, column) entries
PAGES = [
    (128, 8, 2, 16, [300, 200, 40], [(0, 3), (0, 18)]),         # the last page has the token itself
    (64, 24, 2, 32, [700, 90], [(0, 0), (1, 1)]),               # two chunks of q-heads
    (256, 8, 2, 16, [500, 77], [(0, 7), (0, 8), (0, 31)]),
    (128, 32, 8, 16, [5000, 9000, 64], [(1, 0), (1, 100), (1, 562), (0, 311)]),      # several splits
    (96, 6, 2, 48, [100, 30], [(0, 0), (0, 1), (0, 2)]),        # nothing is left of the first one
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", PAGES, ids=[f"{c[0]}-{c[1]}" for c in PAGES])
def test_single_tokens_beside_pages_out_of_range(case, dtype):
    """Positions of such a page take no part: they get no weight, whatever an earlier call of the
    plan, of other scores, has left behind, and the others get theirs without them."""
    d, h, hkv, ps, ctx, bad = case
    dt = getattr(torch, dtype)
    pool, table, weights, n = weighed(dtype, d, h, hkv, ps, ctx, seed=d)
    plan = pool.plan_tree(ctx, [1] * len(ctx), h, weights=True)
    scale = 1.0 / math.sqrt(d)
    good = dev(table)
    hurt = table.copy()
    for s, c in bad:
        hurt[s, c] = BAD if (s + c) % 2 else -1
    for step in range(3):
        q = torch.randn(len(ctx), h, d, device="cuda").to(dt)
        out = torch.full_like(q, 9.0)
        # what an earlier call keeps: scores that are far above the next one's
        junk = weights.clone()
        pool.decode_tree_weights(plan, 0, (8 * q).contiguous(), None, junk, out, good, scale)
        no_error()
        before = weights.clone()
        pool.decode_tree_weights(plan, 0, q, None, weights, out, dev(hurt), scale)
        torch.cuda.synchronize()
        assert ffi.device_error(0)[0] == BAD_PAGE
        for s in range(len(ctx)):
            seen = np.repeat((hurt[s] >= 0) & (hurt[s] < BAD), ps)[:n[s]]
            vis = torch.from_numpy(seen)[None].cuda()
            k, v = pool.gather(0, good, s, 0, n[s])
            ref, tol, wt, rel = attend64(q[s:s + 1], k, v, scale, dtype, vis)
            want = before[s, :, :n[s]].double()
            want[:, n[s] - 1] = 0.0
            add = wt.view(hkv, -1, n[s]).sum(1)
            err = (wt * rel).view(hkv, -1, n[s]).sum(1) if seen.any() else 0.0
            want += add
            check(weights[s, :, :n[s]], want, err + (h // hkv + 2) * 2.0 ** -24 * add + 2.0 ** -23 * want + 1e-30)
            # (bit by bit: what was there, or the zero that a token's own slot starts from)
            gone = torch.from_numpy(~seen).cuda()
            base = before[s, :, :n[s]].clone()
            base[:, n[s] - 1] = 0.0
            assert torch.equal(weights[s, :, :n[s]][:, gone], base[:, gone])
            assert torch.equal(weights[s, :, n[s]:], before[s, :, n[s]:])
            check(out[s:s + 1], ref, tol)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("nodes", [1, 3, 40])
def test_pages_out_of_range_stay_with_their_sequence(dtype, nodes):
    """Every form of the call: the other sequences' sums and rows are what they are without, and
    those of the sequence are finite."""
    ctx, d, h, hkv, ps = [900, 333], 64, 8, 2, 16
    dt = getattr(torch, dtype)
    pool = make_pool(1, 2 * 64, ps, hkv, d, dtype, fill=0.0)
    pool.fill_normal(seed=3)
    table = np.random.default_rng(1).permutation(128).reshape(2, 64)
    hurt = table.copy()
    hurt[0, 5], hurt[0, 56] = BAD, -3
    q = torch.randn(2 * nodes, h, d, device="cuda").to(dt)
    plan = pool.plan_tree(ctx, [nodes] * 2, h, weights=True)
    got = []
    for t in (table, hurt):
        weights, out = torch.zeros(2, hkv, 1000, device="cuda"), torch.zeros_like(q)
        pool.decode_tree_weights(plan, 0, q, None, weights, out, dev(t), 0.125)
        torch.cuda.synchronize()
        assert ffi.device_error(0)[0] == (0 if t is table else BAD_PAGE)
        assert torch.all(torch.isfinite(weights)) and torch.all(torch.isfinite(out))
        got.append((weights[1], out[nodes:]))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("nodes,mask", [(1, None), (1, "any"), (3, None), (60, None)])
def test_an_attention_that_gave_up_adds_nothing(dtype, nodes, mask):
    """A wait that gives up leaves scores and statistics of an older call behind.  The plan carries
    the mark that such a wait sets: its calls leave the sums alone, bit by bit, and say so, until it
    is built again; another plan's calls are not concerned."""
    ctx, d, h, hkv, ps = [900, 333], 64, 8, 2, 16
    dt = getattr(torch, dtype)
    pool = make_pool(1, 2 * 64, ps, hkv, d, dtype, fill=0.0)
    pool.fill_normal(seed=4)
    table = dev(np.random.default_rng(2).permutation(128).reshape(2, 64))
    q = torch.randn(2 * nodes, h, d, device="cuda").to(dt)
    bits = None if mask is None else dev(np.full((2 * nodes, 2), -1, np.int32))
    weights, out = torch.rand(2, hkv, 1000, device="cuda"), torch.zeros_like(q)
    want, start = weights.clone(), weights.clone()
    args = (0, q, bits)
    fresh = pool.plan_tree(ctx, [nodes] * 2, h, weights=True)
    pool.decode_tree_weights(fresh, *args, want, out, table, 0.125)
    no_error()
    ffi.inject_failure(ffi.FAULT_KERNEL_WAIT)
    try:
        plan = pool.plan_tree(ctx, [nodes] * 2, h, weights=True)
    finally:
        ffi.inject_failure(ffi.FAULT_KERNEL_WAIT, 0)
    for _ in range(2):
        pool.decode_tree_weights(plan, *args, weights, out, table, 0.125)
        torch.cuda.synchronize()
        assert ffi.device_error(0)[0] == WAIT_LIMIT
        assert torch.equal(weights, start)
    pool.decode_tree(plan, *args, out, table, 0.125)      # (adds nothing anyway)
    no_error()
    pool.decode_tree_weights(fresh, *args, start, out, table, 0.125)
    no_error()
    assert torch.equal(start, want)
    pool.plan_tree(ctx, [nodes] * 2, h, plan=plan, weights=True)
    pool.decode_tree_weights(plan, *args, weights, out, table, 0.125)
    no_error()
    assert torch.equal(weights, want)
