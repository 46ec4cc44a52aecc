"""Forms of the serving operators that the documentation allows or rules out: rows of every head
dim through both variants of the norm kernel, the rotated K rows against append_rope's, outputs over
their own queries, groups of one.  References and tolerances as in test_gpu_serve_ops."""

from __future__ import annotations

import math

import numpy as np
import pytest

from conftest import HAS_GPU

pytestmark = pytest.mark.gpu

if HAS_GPU:
    import torch

    import kvcache_ffi as ffi
    import paged

from test_gpu_serve_ops import TYPES, attend64, check, norm_case
from test_gpu_spec_ops import BF16, F16, F32, dev, make_pool, no_error

SMS = torch.cuda.get_device_properties(0).multi_processor_count if HAS_GPU else 148


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("more", [-1, 0])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
def test_norm_rope_on_both_sides_of_many_tokens(dtype, more, d):
    """One token below the variant for many tokens, and the first of it: lane groups of every width,
    some partly filled (96), in place, without weights, without q."""
    n = 4 * SMS + more
    counts, ctx = [n - 200, 1, 199], [0, 31, 700]
    a = d // 2
    r = paged.Rotation(d, 1e6, [a - 2 * (a // 4), a // 4, a // 4], "cyclic", neox=d != 64)
    norm_case(dtype, d, 5, 2, 16, r, counts, ctx, seed=d, padding=True)
    norm_case(dtype, d, 5, 2, 16, r, counts, ctx, seed=d + 1, fused=False, in_place=True)
    norm_case(dtype, d, 3, 1, 32, r, counts, ctx, seed=d + 2, weights=(False, True))
    norm_case(dtype, d, 3, 1, 32, r, counts, ctx, seed=d + 3, weights=(False, False), turn="slots")
    norm_case(dtype, d, 3, 2, 16, paged.Rotation(d // 2), counts, ctx, seed=d + 4, with_q=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("n", [50, 4 * SMS])
def test_norm_rope_without_norms_against_append_rope(dtype, neox, n):
    """One axis, the whole head and no weights: append_rope's K rows and q, each within a rounding
    of the storage type of the exact rotation, so within two of one another (and, in 32 bits, within
    2 (2^-22 + 3 * 2^-24) (|y0| + |y1|)); V bit by bit."""
    dt = getattr(torch, dtype)
    a, b = (make_pool(1, 48, 16, 2, 128, dtype, fill=0.0) for _ in range(2))
    bt = dev(np.random.default_rng(0).permutation(48)[None])
    q, k, v = (torch.randn(n, x, 128, device="cuda").to(dt) for x in (8, 2, 2))
    pos = dev(np.arange(n) + 60)
    qa = a.append_rope(0, q, k, v, bt, pos, freq_base=500000.0, neox=neox)
    qb = b.append_norm_rope(0, q, k, v, bt, pos, paged.Rotation(128, 500000.0, neox=neox))
    no_error()
    (ka, va), (kb, vb) = (p.gather(0, bt, 0, 60, n) for p in (a, b))
    assert torch.equal(va, vb) and torch.equal(va, v)
    half = torch.finfo(dt).eps / 2
    for x, ya, yb in ((q, qa, qb), (k, ka, kb)):
        # |a cos - b sin| and |a sin + b cos| are at most |a| + |b|
        pair = x.double().abs()
        both = pair[..., :64] + pair[..., 64:] if neox else pair[..., ::2] + pair[..., 1::2]
        both = torch.cat([both, both], -1) if neox else both.repeat_interleave(2, -1)
        exact = 2 * (2.0 ** -22 + 3 * 2.0 ** -24) * both
        assert torch.all((ya.double() - yb.double()).abs() <=
                         exact + half * (ya.double().abs() + yb.double().abs()) * (1 + 2.0 ** -9) + 2.0 ** -24)
        assert not torch.equal(x, yb)


# -- groups of one -------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("large", [False, True])
def test_the_prefix_of_a_group_of_one_does_not_matter(dtype, large):
    """Not a whole number of pages, longer than the member, longer than the table: the bits of a
    plan that names none; beside groups that do share."""
    dt = getattr(torch, dtype)
    n, pre, h, hkv, d, ps = (30, 2048, 16, 4, 128, 16) if large else (3, 64, 4, 2, 64, 32)
    lens = [pre + 5 * i + 1 for i in range(n)] + [0, 7, pre + 9]
    sizes = [n, 1, 1, 1]
    width = -(-max(lens) // ps)
    pool = make_pool(1, len(lens) * width, ps, hkv, d, dtype, fill=0.0)
    pool.fill_normal(seed=2)
    table = np.random.default_rng(0).permutation(len(lens) * width).reshape(-1, width)
    table[1:n, :pre // ps] = table[0, :pre // ps]
    bt = dev(table)
    q = torch.randn(len(lens), h, d, device="cuda").to(dt)
    outs = []
    for alone in ([0, 0, 0], [pre, 8, 1 << 20], [ps + 1, (1 << 31) - 1, pre]):
        out = torch.full_like(q, 9.0)
        pool.decode_shared(pool.plan_shared(lens, sizes, [pre] + alone, h), 0, q, out, bt, 0.09)
        no_error()
        outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    for i in (0, n - 1, n + 1, n + 2):
        ref, tol, _, _ = attend64(q[i:i + 1], *pool.gather(0, bt, i, 0, lens[i]), 0.09, dtype)
        check(outs[0][i:i + 1], ref, tol)
    assert torch.all(outs[0][n] == 0)
    for bad in ([-1, 0, 0], [0, 0, -ps]):
        with pytest.raises(ValueError):
            pool.plan_shared(lens, sizes, [pre] + bad, h)


# -- outputs over their own queries --------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nodes", [1, 4, 50])
def test_weights_with_the_output_over_its_queries(dtype, nodes):
    """Rows that are counted again are read again behind the attention: there the call is refused,
    with nothing written; elsewhere an output in place of q is what it is in a tensor of its own."""
    ctx, d, h, hkv, ps = [500, 90], 64, 8, 2, 16
    dt = getattr(torch, dtype)
    pool = make_pool(1, 80, ps, hkv, d, dtype, fill=0.0)
    pool.fill_normal(seed=6)
    bt = dev(np.random.default_rng(3).permutation(80).reshape(2, 40))
    tokens = 2 * nodes
    buf = torch.randn(2 * tokens, h, d, device="cuda").to(dt)
    was, q = buf.clone(), buf[:tokens]
    plan = pool.plan_tree(ctx, [nodes] * 2, h, weights=True)
    want, out = torch.zeros(2, hkv, 640, device="cuda"), torch.zeros_like(q)
    pool.decode_tree_weights(plan, 0, q, None, want, out, bt, 0.125)
    no_error()
    weights = torch.zeros_like(want)
    if dtype != F32 and nodes == 50:
        for over in (q, buf[tokens - 1:2 * tokens - 1], buf[1:tokens + 1]):
            with pytest.raises(ValueError, match="overlap"):
                pool.decode_tree_weights(plan, 0, q, None, weights, over, bt, 0.125)
        assert torch.equal(buf, was) and torch.all(weights == 0)
        pool.decode_tree_weights(plan, 0, q, None, weights, buf[tokens:], bt, 0.125)
        assert torch.equal(buf[tokens:], out)
    else:
        pool.decode_tree_weights(plan, 0, q, None, weights, q, bt, 0.125)
        assert torch.equal(q, out)
    no_error()
    assert torch.equal(weights, want)
