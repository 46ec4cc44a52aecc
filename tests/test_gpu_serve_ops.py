"""Head norms with rotation, shared prefixes, summed weights and eviction on the paged
pool, against 64-bit references.

Tolerances are derived from the arithmetic, not fitted.  With h = finfo(t).eps / 2 the
half step of a storage type t:

* norm + rotation: the sum of D squares in 32 bits is off by at most D 2^-24 relative,
  its root by half of that, rsqrt by 2^-22 and the products with it and the weight by
  2^-23; cos and sin are within 2^-22 and the two products and their sum add 3 * 2^-24, all
  relative to |y0| + |y1| of the pair; then one rounding to t (2^-25 below fp16's normal range).
* attention: as in the tree attention's tests: one rounding of the output, one of each
  probability of a 16-bit pool, D + 2 roundings in a score, 2^-19 for exp2, sums and joins.
* summed weights: a weight is a probability in 32 bits, so a score's error and the 2^-19,
  relative; R rows are added in order (R 2^-24) and then to what was there (2^-23).
* moved rows, kept slots, appended V rows and moved weights are bit-exact.
"""

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

from test_gpu_spec_ops import BF16, F16, F32, dev, make_pool, no_error, raw, tables

TYPES = [F32, F16, BF16]
BAD_PAGE, BAD_POSITION = 1, 3   # KVC_DEVERR_*


def check(got, ref, tol):
    assert torch.all(torch.isfinite(got)), "not finite"
    over = float(((got.double() - ref).abs() - tol).max()) if got.numel() else 0.0
    assert over <= 0, f"over the bound by {over:.3g}"


# -- norm + rotation + append ---------------------------------------------------------------
def normed_rotated(x, w, eps, rotation, turn):
    """(reference, tolerance without the rounding to the storage type), fp64."""
    d = x.shape[-1]
    y, rel = x.double(), 0.0
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        rel = d * 2.0 ** -25 + 2.0 ** -22 + 2.0 ** -23
    if rotation is None:
        return y, rel * y.abs()
    half, rot = rotation.pairs, rotation.rotary_dim
    ang = turn[:, rotation.axis.astype(np.int64)].astype(np.float64) * rotation.inv_freq
    ang = torch.from_numpy(ang).cuda()[:, None]
    if rotation.neox:
        i0, i1 = torch.arange(half), torch.arange(half) + half
    else:
        i0, i1 = 2 * torch.arange(half), 2 * torch.arange(half) + 1
    a, b = y[..., i0], y[..., i1]
    out, tol = y.clone(), rel * y.abs()
    out[..., i0] = a * ang.cos() - b * ang.sin()
    out[..., i1] = a * ang.sin() + b * ang.cos()
    both = (rel + 2.0 ** -22 + 3 * 2.0 ** -24) * (a.abs() + b.abs())
    tol[..., i0], tol[..., i1] = both, both
    assert rot <= d
    return out, tol


def norm_case(dtype, d, h, hkv, ps, rotation, counts, ctx, seed, fused=True, weights=(True, True),
              turn="own", in_place=False, with_q=True, scale=1.0, padding=False, eps=1e-6):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = getattr(torch, dtype)
    n = sum(counts)
    bt, total = tables([max(1, -(-(c + k) // ps)) for c, k in zip(ctx, counts)], seed)
    pool = make_pool(2, total, ps, hkv, d, dtype, fill=3.0)
    before = [x.clone() for x in raw(pool)]
    rows = np.repeat(np.arange(len(counts)), counts)
    pos = np.concatenate([c + np.arange(k) for c, k in zip(ctx, counts)]).astype(np.int64)
    slots = pos.copy()
    if padding:
        slots[rng.random(n) < 0.3] = -1
    qkv = (scale * torch.randn(n, h + 2 * hkv, d, generator=g, device="cuda")).to(dt)
    q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    wq, wk = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt) if w else None
              for w in weights)
    axes = 1 if rotation is None else rotation.axes
    angles = np.repeat(pos[:, None], axes, 1)
    rope = None
    if turn == "own":
        angles = rng.integers(-5, 100000, (n, axes))
        rope = dev(angles)
    ref_q, tol_q = normed_rotated(q, wq, eps, rotation, angles)
    ref_k, tol_k = normed_rotated(k, wk, eps, rotation, angles)
    q_out = q if in_place else torch.full((n, h, d), 9.0, dtype=dt, device="cuda")
    v0 = v.clone()
    pool.append_norm_rope(1, q if with_q else None, k, v, bt, dev(slots), rotation, rows=dev(rows),
                          rope_positions=rope, q_weight=wq, k_weight=wk, eps=eps,
                          q_out=q_out if with_q else None)
    no_error()
    half = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dtype == F16 else 1e-38
    live = torch.from_numpy(slots >= 0).cuda()
    if with_q:
        check(q_out[live], ref_q[live], (tol_q + half * ref_q.abs() * (1 + 2 ** -10) + tiny)[live])
        assert in_place or torch.all(q_out[~live] == 9.0)
    for s in range(len(counts)):
        if counts[s] == 0:
            continue
        gk, gv = pool.gather(1, bt, s, int(ctx[s]), int(counts[s]))
        at = torch.from_numpy(rows == s).cuda()
        ok = live[at]
        check(gk[ok], ref_k[at][ok], (tol_k + half * ref_k.abs() * (1 + 2 ** -10) + tiny)[at][ok])
        assert torch.equal(gv[ok], v0[at][ok])
        assert torch.all(gk[~ok] == 3.0) and torch.all(gv[~ok] == 3.0)
    # nothing else was written
    for x, y in zip(raw(pool), before):
        assert torch.equal(x[0], y[0])
        assert int((x[1] != 3.0).sum()) <= int(live.sum()) * hkv * d


NORM = [
    # D, H, Hkv, page, rotary (0: none), sections, order, neox, counts, ctx
    (128, 32, 8, 16, 128, None, "blocks", True, [1], [511]),
    (128, 8, 2, 32, 128, [24, 20, 20], "cyclic", True, [5, 0, 40], [0, 7, 1000]),
    (128, 8, 2, 16, 128, [16, 24, 24], "blocks", False, [33, 1], [15, 31]),
    (64, 7, 1, 48, 64, [12, 10, 10], "ladders", True, [9], [40]),
    (64, 4, 4, 16, 32, [4, 12], "blocks", True, [3, 3], [0, 100]),     # a part of the head
    (96, 6, 2, 16, 96, [16, 16, 16], "cyclic", False, [17], [3]),
    (256, 4, 2, 16, 256, None, "blocks", True, [2, 6], [1, 2]),
    (256, 4, 1, 16, 64, [32], "blocks", False, [6], [0]),
    (128, 4, 2, 16, 20, [3, 3, 4], "ladders", True, [11], [9]),        # pairs that fill no unit
    (128, 4, 2, 16, 6, None, "blocks", False, [11], [9]),
    (80, 5, 1, 16, 80, None, "blocks", True, [7], [0]),
    (24, 3, 3, 16, 24, [4, 4, 4], "blocks", True, [7], [12]),          # odd units a row
    (8, 2, 2, 16, 8, [1, 1, 1, 1], "cyclic", False, [5], [12]),
    (128, 16, 4, 16, 0, None, "blocks", True, [13], [77]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", NORM, ids=[f"{c[0]}-{c[4]}-{i}" for i, c in enumerate(NORM)])
def test_norm_rope(case, dtype):
    d, h, hkv, ps, rot, sec, order, neox, counts, ctx = case
    r = paged.Rotation(rot, 500000.0, sec, order, neox) if rot else None
    norm_case(dtype, d, h, hkv, ps, r, counts, ctx, seed=d + rot)
    norm_case(dtype, d, h, hkv, ps, r, counts, ctx, seed=d + rot + 1, fused=False, turn="slots",
              padding=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_rope_many_tokens(dtype):
    """Four tokens a CTA, ragged at the end; several rounds of heads."""
    r = paged.Rotation(128, 1e6, [24, 20, 20], "cyclic")
    norm_case(dtype, 128, 12, 3, 16, r, [500, 1, 202], [0, 40, 3000], seed=1, padding=True)
    norm_case(dtype, 64, 32, 8, 16, paged.Rotation(64, neox=False), [594], [3], seed=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 20)])
def test_norm_rope_without_parts(dtype, d, rot):
    r = paged.Rotation(rot, inv_freq=np.linspace(1.0, -0.25, rot // 2))   # frequencies of one's own
    for kw in (dict(weights=(False, True)), dict(weights=(True, False)), dict(weights=(False, False)),
               dict(with_q=False), dict(in_place=True, fused=False), dict(scale=0.0),
               dict(scale=1e-3, eps=1e-2)):
        norm_case(dtype, d, 8, 2, 16, r, [9, 4], [20, 0], seed=3, **kw)


def test_norm_rope_is_append_rope_without_norms():
    """One axis, the whole head and no weights: the bits of append_rope."""
    for dtype in TYPES:
        dt = getattr(torch, dtype)
        for neox in (False, True):
            a, b = (make_pool(1, 8, 16, 2, 128, dtype, fill=0.0) for _ in range(2))
            bt = dev(np.arange(8)[None])
            q, k, v = (torch.randn(50, x, 128, device="cuda").to(dt) for x in (8, 2, 2))
            pos = dev(np.arange(50) + 60)
            qa = a.append_rope(0, q, k, v, bt, pos, freq_base=500000.0, neox=neox)
            qb = b.append_norm_rope(0, q, k, v, bt, pos, paged.Rotation(128, 500000.0, neox=neox))
            no_error()
            half = torch.finfo(dt).eps / 2
            assert float((qa.double() - qb.double()).abs().max()) <= 2 ** -20 + 16 * half
            assert torch.equal(raw(a)[1], raw(b)[1])


def test_norm_rope_bad_pages_and_rows():
    pool = make_pool(1, 4, 16, 2, 64, F16, fill=3.0)
    bt = dev([[0, 99], [1, 2]])
    x = torch.ones(4, 2, 64, dtype=torch.float16, device="cuda")
    r = paged.Rotation(64)
    for pos, rows, code in (([16, 3, 4, 5], [0, 0, 0, 1], BAD_PAGE),
                            ([32, 3, 4, 5], [1, 0, 0, 1], BAD_POSITION),
                            ([0, 3, 4, 5], [2, 0, 0, 1], BAD_POSITION),
                            ([0, 3, 4, 5], [-1, 0, 0, 1], BAD_POSITION)):
        for d_r in (r, paged.Rotation(6)):          # both kernels
            out = torch.full((4, 2, 64), 9.0, dtype=torch.float16, device="cuda")
            pool.append_norm_rope(0, x, x, x, bt, dev(pos), d_r, rows=dev(rows), q_out=out)
            torch.cuda.synchronize()
            assert ffi.device_error(0)[0] == code
            assert torch.all(out[0] == 9.0) and not torch.any(out[1:] == 9.0)


# -- attention over shared prefixes ------------------------------------------------------------
def attend64(q, k, v, scale, dtype, vis=None):
    """Reference and tolerance of q (n, H, D) over k, v (L, Hkv, D), and the weights (n, H, L)."""
    g, d = q.shape[1] // k.shape[1], q.shape[2]
    kk, vv = k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    sc = torch.einsum("nhd,lhd->nhl", q.double(), kk) * scale
    mag = torch.einsum("nhd,lhd->nhl", q.double().abs(), kk.abs()) * abs(scale)
    vis = torch.ones_like(sc, dtype=torch.bool) if vis is None else vis[:, None].expand_as(sc)
    sc, mag = torch.where(vis, sc, -math.inf), torch.where(vis, mag, 0.0)
    wt = torch.nan_to_num(torch.softmax(sc, -1), 0.0)
    ref = torch.einsum("nhl,lhd->nhd", wt, vv)
    spread = torch.einsum("nhl,lhd->nhd", wt, vv.abs())
    half = torch.finfo(getattr(torch, dtype)).eps / 2
    score = 2 * (d + 2) * 2.0 ** -24 * mag.amax(-1, keepdim=True) + 2.0 ** -19
    tol = half * ref.abs() + (score + (0 if dtype == F32 else 2 * half)) * spread + 1e-30
    return ref, tol + (2.0 ** -25 if dtype == F16 else 0), wt, score


def shared_case(dtype, d, h, hkv, ps, sizes, prefix, own, seed, scale=None, rows=None, tweak=None):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = getattr(torch, dtype)
    lens = np.repeat(prefix, sizes) + np.asarray(own, dtype=np.int64)
    n = len(lens)
    group = np.repeat(np.arange(len(sizes)), sizes)
    need = [max(1, -(-int(x) // ps) - prefix[k] // ps) for x, k in zip(lens, group)]
    bt, total = tables(need + [max(1, p // ps) for p in prefix], seed)
    flat = bt.cpu().numpy()
    table = np.full((n if rows is None else max(rows) + 1,
                     max(1, max(-(-int(x) // ps) for x in lens))), flat[-1, -1], np.int32)
    for i in range(n):
        r, a, b = i if rows is None else rows[i], prefix[group[i]] // ps, -(-int(lens[i]) // ps)
        table[r, :a] = flat[n + group[i], :a]
        table[r, a:b] = flat[i, :b - a]
    bt = dev(table)
    pool = make_pool(2, total, ps, hkv, d, dtype)

    def fill(row, a, b):
        k = torch.randn(b - a, hkv, d, generator=g, device="cuda").to(dt)
        v = torch.randn(b - a, hkv, d, generator=g, device="cuda").to(dt)
        if tweak:
            tweak(k, v, a)
        if b > a:
            pool.append(1, k, v, bt, torch.arange(a, b, dtype=torch.int32, device="cuda"),
                        torch.full((b - a,), row, dtype=torch.int32, device="cuda"))
        return k, v

    row_of = list(range(n)) if rows is None else rows
    firsts = np.concatenate([[0], np.cumsum(sizes)[:-1]])
    common = [fill(row_of[firsts[k]], 0, prefix[k]) for k in range(len(sizes))]
    q = torch.randn(n, h, d, generator=g, device="cuda").to(dt)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    ref = torch.zeros(n, h, d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(ref)
    for i in range(n):
        ko, vo = fill(row_of[i], prefix[group[i]], int(lens[i]))
        k = torch.cat([common[group[i]][0], ko])
        v = torch.cat([common[group[i]][1], vo])
        if len(k):
            r, t, _, _ = attend64(q[i:i + 1], k, v, scale, dtype)
            ref[i], tol[i] = r[0], t[0]
    out = torch.full((n + 2, h, d), 7.0, dtype=dt, device="cuda")
    plan = pool.plan_shared(lens, sizes, prefix, h, rows=rows)
    pool.decode_shared(plan, 1, q, out, bt, scale)
    no_error()
    assert torch.all(out[n:] == 7.0)
    check(out[:n], ref, tol)
    first = out[:n].clone()
    pool.decode_shared(plan, 1, q, out, bt, scale)        # the same bits again
    no_error()
    assert torch.equal(first, out[:n])
    return first


SHARED = [
    # D, H, Hkv, page, group sizes, prefixes, own lengths
    (64, 8, 2, 16, [1], [0], [1]),
    (128, 8, 2, 16, [3], [128], [1, 0, 40]),                   # one tile; nothing of one's own
    (128, 8, 2, 16, [2, 1, 3], [160, 48, 0], [5, 100, 3, 0, 1, 300]),   # a zero length
    (128, 32, 8, 32, [20, 4], [608, 2016], list(range(1, 25))),
    (64, 7, 1, 48, [40], [480], [7 * i % 130 for i in range(40)]),     # 280 rows: two blocks
    (96, 12, 2, 16, [5, 6], [1040, 32], [130] * 11),
    (256, 4, 2, 16, [9, 2], [400, 800], list(range(60, 71))),
    (192, 20, 1, 16, [15], [272], list(range(15))),            # 300 rows in blocks of 128
    (32, 4, 4, 16, [70], [1600], [3] * 70),
    (128, 64, 8, 64, [48], [1024], [i * 11 % 90 for i in range(48)]),
    (80, 6, 2, 16, [4, 1], [96, 0], [6, 20, 1, 0, 45]),        # no tensor tiles
    (16, 36, 1, 16, [4], [320], [3, 50, 0, 33]),               # more q-heads than a small block
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", SHARED, ids=[f"{c[0]}-{c[1]}-{i}" for i, c in enumerate(SHARED)])
def test_shared_prefix(case, dtype):
    d, h, hkv, ps, sizes, prefix, own = case
    shared_case(dtype, d, h, hkv, ps, sizes, prefix, own, seed=d + h)


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_prefix_long(dtype):
    """More tiles than the GPU takes at once; q-heads of one KV head in two blocks of a prefix."""
    shared_case(dtype, 128, 16, 2, 16, [50, 1, 9], [6000 // 16 * 16, 0, 3040],
                [i * 37 % 700 for i in range(60)], seed=5)
    shared_case(dtype, 64, 12, 1, 16, [33], [4096], [i * 5 for i in range(33)], seed=6, scale=-0.1)


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_prefix_rows_scales_and_large_scores(dtype):
    shared_case(dtype, 64, 8, 4, 16, [2, 2], [256, 128], [9, 8, 7, 130], seed=7, rows=[5, 0, 2, 3])
    for s in (0.0, 1.0):
        shared_case(dtype, 128, 8, 4, 16, [3], [256], [9, 8, 0], seed=8, scale=s)

    def grow(k, v, a):   # the largest scores stand last
        ramp = (a + torch.arange(k.shape[0], device="cuda")) / 200.0
        k.copy_((k.float() * ramp[:, None, None]).to(k.dtype))
    shared_case(dtype, 128, 8, 2, 16, [4], [640], [90, 0, 33, 700], seed=9, tweak=grow)


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_prefix_beside_decode(dtype):
    """The plain decode over the same tables, and a graph of the step on another stream."""
    dt = getattr(torch, dtype)
    n, ps, pre, hkv, d = 12, 16, 512, 2, 128
    lens = [pre + 5 * i for i in range(n)]
    pool = make_pool(1, 32 + 5 * n, ps, hkv, d, dtype, fill=0.0)
    pool.fill_normal(seed=4)
    t = np.zeros((n, 36), np.int32)
    t[:, :32] = np.random.default_rng(0).permutation(32)
    for i in range(n):
        t[i, 32:] = 32 + 5 * i + np.arange(4)
    bt = dev(t)
    q = torch.randn(n, 8, d, device="cuda").to(dt)
    a, b, c = (torch.zeros_like(q) for _ in range(3))
    pool.decode(pool.plan(lens, 8), 0, q, a, bt, 0.09)
    plan = pool.plan_shared(lens, [n], [pre], 8)
    pool.decode_shared(plan, 0, q, b, bt, 0.09)
    no_error()
    step = 2.0 ** -18 if dtype == F32 else 6 * torch.finfo(dt).eps
    assert float((a.float() - b.float()).abs().max()) <= step * 4.0
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        pool.decode_shared(plan, 0, q, c, bt, 0.09)
        with pytest.raises(ValueError, match="captured"):
            pool.plan_shared(lens, [n], [pre], 8, plan=plan)
    for _ in range(2):
        c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b, c)
    no_error()


def test_shared_prefix_bad_pages():
    pool = make_pool(1, 20, 16, 2, 128, F16, fill=0.0)
    t = np.tile(np.arange(20), (3, 1))
    t[1, 18] = 99          # a page of its own
    q = torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda")
    out = torch.ones_like(q)
    plan = pool.plan_shared([300, 300, 300], [3], [256], 4)
    pool.decode_shared(plan, 0, q, out, dev(t), 1.0)
    torch.cuda.synchronize()
    assert ffi.device_error(0) == (BAD_PAGE, 99)
    t[1, 18], t[0, 3] = 0, -7
    pool.decode_shared(plan, 0, q, out, dev(t), 1.0)
    torch.cuda.synchronize()
    assert ffi.device_error(0)[0] == BAD_PAGE


# -- attention that adds its weights up -----------------------------------------------------------
def weigh_case(dtype, d, h, hkv, ps, ctx, nodes, seed, mask=None, scale=None, rows=None, tweak=None):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = getattr(torch, dtype)
    n_rows = len(ctx) if rows is None else max(rows) + 1
    row_of = list(range(len(ctx))) if rows is None else rows
    need = [1] * n_rows
    for r, c, n in zip(row_of, ctx, nodes):
        need[r] = max(1, -(-(c + n) // ps))
    bt, total = tables(need, seed)
    pool = make_pool(2, total, ps, hkv, d, dtype)
    slots = max(c + n for c, n in zip(ctx, nodes)) + 5
    start = torch.rand(n_rows + 1, hkv, slots, generator=g, device="cuda") * 3
    for r, c, n in zip(row_of, ctx, nodes):
        start[r, :, c:c + n] = math.nan                     # slots of new tokens hold anything
    weights = start.clone()
    words = max(1, (max(nodes) + 31) // 32)
    tokens, q0 = sum(nodes), 0
    q = torch.randn(tokens, h, d, generator=g, device="cuda").to(dt)
    out = torch.full((tokens + 1, h, d), 7.0, dtype=dt, device="cuda")
    ref, tol = (torch.zeros(tokens, h, d, dtype=torch.float64, device="cuda") for _ in range(2))
    want, wtol, packed = start.double(), torch.zeros_like(start, dtype=torch.float64), []
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    for r, c, n in zip(row_of, ctx, nodes):
        k = torch.randn(c + n, hkv, d, generator=g, device="cuda").to(dt)
        v = torch.randn(c + n, hkv, d, generator=g, device="cuda").to(dt)
        if tweak:
            tweak(k, v, c)
        bits = rng.integers(0, 1 << 32, (n, words), dtype=np.uint64).astype(np.uint32)
        bits[rng.random(n) < 0.3] = 0
        packed.append(bits)
        if n == 0:
            continue
        pool.append(1, k, v, bt, torch.arange(c + n, dtype=torch.int32, device="cuda"),
                    torch.full((c + n,), r, dtype=torch.int32, device="cuda"))
        vis = np.ones((n, c + n), dtype=bool)
        for t in range(n):
            for j in range(n):
                vis[t, c + j] = j <= t if mask is None else (int(bits[t, j // 32]) >> (j % 32)) & 1
        vis = torch.from_numpy(vis).cuda()
        ks = torch.where(vis.any(0)[:, None, None], k, 0.0) if tweak else k
        vs = torch.where(vis.any(0)[:, None, None], v, 0.0) if tweak else v
        ref[q0:q0 + n], tol[q0:q0 + n], wt, rel = attend64(q[q0:q0 + n], ks, vs, scale, dtype, vis)
        add = wt.view(n, hkv, -1, c + n).sum((0, 2))
        err = (wt * rel).view(n, hkv, -1, c + n).sum((0, 2))
        want[r, :, c:c + n] = 0.0
        want[r, :, :c + n] += add
        wtol[r, :, :c + n] = err + (n * h // hkv + 2) * 2.0 ** -24 * add + \
            2.0 ** -23 * want[r, :, :c + n] + 1e-30
        q0 += n
    plan = pool.plan_tree(ctx, nodes, h, rows=rows, weights=True)
    m = None if mask is None else dev(np.concatenate(packed).view(np.int32))
    pool.decode_tree_weights(plan, 1, q, m, weights, out, bt, scale)
    no_error()
    assert torch.all(out[tokens:] == 7.0)
    check(out[:tokens], ref, tol)
    touched = torch.zeros_like(start, dtype=torch.bool)
    for r, c, n in zip(row_of, ctx, nodes):
        if n:
            touched[r, :, :c + n] = True
    assert torch.equal(weights[~touched], start[~touched]) or torch.equal(
        weights[~touched].nan_to_num(-1.0), start[~touched].nan_to_num(-1.0))
    check(weights[touched], want[touched], wtol[touched])
    # the attention is decode_tree's
    plain = torch.zeros_like(out)
    pool.decode_tree(plan, 1, q, m, plain, bt, scale)
    no_error()
    check(plain[:tokens], ref, tol)


WEIGH = [
    # D, H, Hkv, page, ctx, nodes
    (64, 8, 2, 16, [0], [1]),
    (64, 32, 4, 16, [511], [1]),
    (128, 8, 2, 16, [0, 5, 127, 128, 129, 3000], [3, 0, 1, 2, 7, 1]),
    (128, 32, 8, 32, [1000, 17, 2333], [1, 1, 1]),
    (128, 16, 2, 16, [700, 40], [100, 70]),               # two blocks of rows
    (96, 6, 2, 48, [250, 90], [13, 64]),
    (256, 4, 2, 16, [300, 64, 0], [20, 1, 100]),
    (32, 4, 4, 16, [600, 31], [256, 200]),
    (64, 7, 1, 16, [100, 383, 384], [64, 1, 40]),
    (80, 4, 2, 16, [77, 200], [6, 20]),
    (160, 4, 2, 16, [130, 0], [40, 129]),
    (192, 6, 2, 32, [700, 130], [33, 200]),
    (128, 32, 4, 16, [2000, 300, 64], [40, 4, 5]),         # 320, 32 and 40 rows
    (128, 32, 4, 16, [2500, 300, 0, 15, 16, 9000], [1, 1, 1, 0, 1, 1]),     # single tokens
    (64, 24, 2, 48, [700, 0, 4000], [1, 1, 1]),            # 12 q-heads: two chunks of a warp
    (128, 40, 1, 16, [900, 30], [1, 1]),                   # 40 q-heads
    (256, 8, 2, 16, [1300], [1]),
    (32, 4, 4, 16, [70000], [1]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", WEIGH, ids=[f"{c[0]}-{c[1]}-{i}" for i, c in enumerate(WEIGH)])
def test_weights(case, dtype):
    d, h, hkv, ps, ctx, nodes = case
    weigh_case(dtype, d, h, hkv, ps, ctx, nodes, seed=d + h)


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_masks_rows_scales(dtype):
    weigh_case(dtype, 128, 8, 2, 16, [0, 40, 0], [40, 33, 9], seed=3, mask="any")   # rows that see nothing
    weigh_case(dtype, 64, 8, 4, 16, [50, 400], [7, 9], seed=4, rows=[3, 1])
    for s in (0.0, -0.1, 1.0):
        weigh_case(dtype, 128, 4, 2, 16, [130, 9], [7, 9], seed=5, scale=s)
        weigh_case(dtype, 128, 4, 2, 16, [900, 9], [1, 1], seed=5, scale=s)
        weigh_case(dtype, 128, 4, 2, 16, [900, 9], [1, 1], seed=5, scale=s, mask="any")
        weigh_case(dtype, 128, 8, 2, 16, [130, 9], [40, 70], seed=5, scale=s, mask="any")

    def grow(k, v, c):
        ramp = torch.linspace(0.1, 5.0, k.shape[0], device="cuda")[:, None, None]
        k.copy_((k.float() * ramp).to(k.dtype))
    weigh_case(dtype, 128, 8, 2, 16, [2500, 700], [1, 20], seed=6, tweak=grow)
    weigh_case(dtype, 64, 8, 2, 16, [1500], [90], seed=6, tweak=grow)


@pytest.mark.parametrize("dtype", TYPES)
def test_weights_of_unseen_values(dtype):
    """What no token sees may be anything in K and V, and gets no weight."""
    def poison(k, v, c):
        k[c + 2], v[c + 2] = math.nan, math.inf
    import test_gpu_serve_ops as me

    class Rng:      # masks without node 2
        def __init__(self, seed):
            self.r = np.random.Generator(np.random.PCG64(seed))

        def __getattr__(self, name):
            return getattr(self.r, name)

        def integers(self, lo, hi, shape=None, dtype=np.int64):
            x = self.r.integers(lo, hi, shape, dtype=dtype)
            return x & ~np.uint64(4) if dtype is np.uint64 else x
    orig = np.random.default_rng
    np.random.default_rng = Rng
    try:
        me.weigh_case(dtype, 128, 8, 2, 16, [300, 60], [9, 6], seed=7, mask="any", tweak=poison)
        me.weigh_case(dtype, 128, 8, 2, 16, [300, 60], [40, 29], seed=8, mask="any", tweak=poison)
    finally:
        np.random.default_rng = orig


# -- eviction -------------------------------------------------------------------------------------
def keep64(w, n, budget, recent):
    """The slots that stay of one head's weights w, by definition."""
    if n <= budget:
        return np.arange(n)
    key = np.where(np.isnan(w[:n]), -np.inf, w[:n].astype(np.float64))
    nan_last = np.isnan(w[:n - recent])
    order = sorted(range(n - recent), key=lambda i: (bool(nan_last[i]), -key[i], i))
    return np.sort(np.concatenate([order[:budget - recent], np.arange(n - recent, n)])).astype(np.int64)


def evict_case(dtype, layers, d, hkv, ps, ctx, budget, recent, seed, make=None, rows=None,
               in_place=False):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n_rows = len(ctx) if rows is None else max(rows) + 1
    row_of = list(range(len(ctx))) if rows is None else rows
    need = [1] * n_rows
    for r, c in zip(row_of, ctx):
        need[r] = max(1, -(-c // ps))
    bt, total = tables(need, seed)
    pool = make_pool(layers, total, ps, hkv, d, dtype)
    for x in raw(pool):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda").to(x.dtype))
    slots = bt.shape[1] * ps + 3
    w = torch.randn(layers, n_rows, hkv, slots, generator=g, device="cuda").exp()
    if make:
        make(w)
    w0 = w.cpu().numpy().copy()
    out = w if in_place else torch.full_like(w, -9.0)
    full = [[pool.gather(lay, bt, r, 0, bt.shape[1] * ps) for r in range(n_rows)]
            for lay in range(layers)]
    kept = pool.evict(bt, dev(ctx), w, budget, recent=recent,
                      rows=None if rows is None else dev(rows),
                      weights_out=None if in_place else out)
    no_error()
    kept = kept.cpu().numpy()
    assert kept.shape == (layers, len(ctx), hkv, budget)
    want_w = w0.copy() if in_place else np.full_like(w0, -9.0)
    for lay in range(layers):
        now = [pool.gather(lay, bt, r, 0, bt.shape[1] * ps) for r in range(n_rows)]
        for i, c in enumerate(ctx):
            r, m = row_of[i], min(c, budget)
            for h in range(hkv):
                stay = keep64(w0[lay, r, h], c, budget, recent)
                assert kept[lay, i, h, :m].tolist() == stay.tolist()
                assert np.all(kept[lay, i, h, m:] == -1)
                want_w[lay, r, h, :m] = w0[lay, r, h, stay]
                s = torch.from_numpy(stay).cuda()
                for a, b in zip(now[r], full[lay][r]):
                    assert torch.equal(a[:m, h], b[s, h])
                    assert torch.equal(a[m:, h], b[m:, h])     # behind them: as it was
        for r in range(n_rows):
            if r not in row_of:
                assert all(torch.equal(a, b) for a, b in zip(now[r], full[lay][r]))
    assert np.array_equal(out.cpu().numpy(), want_w, equal_nan=True)


EVICT = [
    # layers, D, Hkv, page, ctx, budget, recent
    (1, 64, 1, 16, [1], 1, 0),
    (2, 64, 2, 16, [40, 5, 0, 17], 16, 4),
    (1, 128, 2, 16, [600], 512, 64),
    (2, 128, 8, 32, [700, 100, 300], 257, 257),      # only the newest
    (1, 96, 3, 48, [999, 1000], 999, 0),
    (3, 256, 1, 16, [300, 90], 33, 1),
    (1, 8, 2, 16, [3000], 700, 10),                  # 2048 units are more than 256 rows
    (1, 24, 2, 16, [1500], 900, 900),
    (1, 32, 1, 64, [9000, 20000], 5000, 100),        # keys that shared memory does not hold
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", EVICT, ids=[f"{c[1]}-{c[5]}-{i}" for i, c in enumerate(EVICT)])
def test_evict(case, dtype):
    evict_case(dtype, *case, seed=case[1] + case[5])


def test_evict_in_place_rows_ties_and_odd_weights():
    evict_case(F16, 2, 64, 2, 16, [300, 90, 500], 100, 10, seed=1, in_place=True)
    evict_case(BF16, 1, 64, 2, 16, [300, 90], 100, 0, seed=2, rows=[4, 2])
    evict_case(F32, 1, 64, 2, 16, [9500], 3000, 500, seed=2, in_place=True)
    evict_case(F32, 1, 64, 1, 16, [500, 300], 100, 7, seed=3, make=lambda w: w.fill_(0.25))
    evict_case(F16, 1, 64, 2, 16, [700], 333, 50, seed=4, make=lambda w: w.copy_((w * 3).floor()))

    def odd(w):
        x = w.view(-1)
        x[::3], x[1::7], x[2::5], x[3::11] = 0.0, -0.0, math.nan, math.inf
        x[4::13], x[5::17] = -math.inf, -w.view(-1)[5::17].abs() - 1
    for budget in (20, 200, 450):
        evict_case(F16, 1, 64, 2, 16, [500, 480], budget, 9, seed=5, make=odd)


def test_evict_bad_rows_lengths_and_pages():
    pool = make_pool(1, 8, 16, 1, 64, F16, fill=0.0)
    pool.fill_normal(seed=1)
    t = np.arange(8).reshape(2, 4)
    w = torch.rand(1, 2, 1, 64, device="cuda")
    before = [x.clone() for x in raw(pool)]
    for ctx, rows, slots in (([65], [0], 64), ([-1], [0], 64), ([60], [2], 64), ([60], [-1], 64),
                             ([60], [0], 50)):
        kept = pool.evict(dev(t), dev(ctx), w[..., :slots].contiguous(), 10, rows=dev(rows))
        torch.cuda.synchronize()
        assert ffi.device_error(0)[0] == BAD_POSITION
        assert torch.all(kept == -1)
        assert all(torch.equal(a, b) for a, b in zip(raw(pool), before))
    t[0, 2] = 8
    pool.evict(dev(t), dev([64]), w, 40)
    torch.cuda.synchronize()
    assert ffi.device_error(0) == (BAD_PAGE, 8)
    # rows of other pages moved, page 3 (the last of row 0) is only read
    assert all(torch.equal(a[:, 3:], b[:, 3:]) for a, b in zip(raw(pool), before))


# -- together ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_a_generation_with_shared_prefix_weights_and_eviction(dtype):
    """A prompt goes in (norm + rotation with positions on three axes), its tokens' weights are
    counted, the cache is cut back and decoding goes on behind it, against a dense model."""
    dt = getattr(torch, dtype)
    d, h, hkv, ps, layers, n = 64, 8, 2, 16, 2, 3
    rot = paged.Rotation(d, sections=[12, 10, 10], order="cyclic")
    pool = make_pool(layers, 40, ps, hkv, d, dtype, fill=0.0)
    bt = dev(np.random.default_rng(1).permutation(39).reshape(3, 13))
    weights = torch.full((layers, n, hkv, 13 * ps), math.nan, device="cuda")
    wq, wk = ((1 + 0.2 * torch.randn(d, device="cuda")).to(dt) for _ in range(2))
    ctx, cached = [0] * n, [[[[] for _ in range(hkv)] for _ in range(n)] for _ in range(layers)]
    turn = 0
    sums = [[[[] for _ in range(hkv)] for _ in range(n)] for _ in range(layers)]
    half = torch.finfo(dt).eps / 2
    scale = 1 / math.sqrt(d)
    for step, new in enumerate(([70, 33, 100], [1, 1, 1], [1, 1, 1], [5, 1, 0], [1, 1, 1])):
        tokens = sum(new)
        rows = np.repeat(np.arange(n), new)
        slot = np.concatenate([c + np.arange(k) for c, k in zip(ctx, new)])
        pos = np.stack([turn + np.concatenate([np.arange(k) // a for k in new]) for a in (1, 3, 5)], 1)
        plan = pool.plan_tree(ctx, new, h, weights=True)
        for lay in range(layers):
            qkv = torch.randn(tokens, h + 2 * hkv, d, device="cuda").to(dt)
            q = pool.append_norm_rope(lay, qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:], bt,
                                      dev(slot), rot, rows=dev(rows), rope_positions=dev(pos),
                                      q_weight=wq, k_weight=wk)
            ref, tol = normed_rotated(qkv[:, :h], wq, 1e-6, rot, pos)
            check(q, ref, tol + half * ref.abs() * (1 + 2 ** -10) + 2.0 ** -25)
            out = torch.zeros_like(q)
            pool.decode_tree_weights(plan, lay, q, None, weights[lay], out, bt, scale)
            no_error()
            at = 0
            for i in range(n):
                k, v = pool.gather(lay, bt, i, 0, ctx[i] + new[i])
                if new[i] == 0:
                    continue
                vis = torch.ones(new[i], ctx[i] + new[i], dtype=torch.bool, device="cuda").tril(ctx[i])
                r, t, wt, rel = attend64(q[at:at + new[i]], k, v, scale, dtype, vis)
                check(out[at:at + new[i]], r, t)
                for x in range(hkv):
                    # what is cached is what went in and was not evicted
                    got = v[:, x]
                    was = cached[lay][i][x] + [qkv[at + j, h + hkv + x] for j in range(new[i])]
                    assert torch.equal(got, torch.stack(was))
                    cached[lay][i][x] = was
                    add = wt.view(new[i], hkv, -1, ctx[i] + new[i])[:, x].sum((0, 1)).cpu().numpy()
                    add[:ctx[i]] += np.array(sums[lay][i][x])
                    sums[lay][i][x] = add.tolist()
                    np.testing.assert_allclose(weights[lay, i, x, :ctx[i] + new[i]].cpu().numpy(), add,
                                               rtol=2e-4, atol=1e-7)
                at += new[i]
        turn += max(new)
        ctx = [c + k for c, k in zip(ctx, new)]
        if step in (0, 3):
            w = weights.cpu().numpy()
            kept = pool.evict(bt, dev(ctx), weights, 40, recent=8).cpu().numpy()
            no_error()
            for lay in range(layers):
                for i in range(n):
                    for x in range(hkv):
                        stay = keep64(w[lay, i, x], ctx[i], 40, 8)
                        assert kept[lay, i, x, :len(stay)].tolist() == stay.tolist()
                        cached[lay][i][x] = [cached[lay][i][x][j] for j in stay]
                        sums[lay][i][x] = [sums[lay][i][x][j] for j in stay]
            ctx = [min(c, 40) for c in ctx]
    # the same prompt for everyone: the first sequence's pages, shared
    shared = bt.clone()
    shared[:, :2] = shared[0, :2]
    lens = [c for c in ctx]
    q = torch.randn(n, h, d, device="cuda").to(dt)
    out = torch.zeros_like(q)
    pool.decode_shared(pool.plan_shared(lens, [n], [2 * ps], h), 1, q, out, shared, scale)
    no_error()
    for i in range(n):
        k, v = pool.gather(1, shared, i, 0, lens[i])
        r, t, _, _ = attend64(q[i:i + 1], k, v, scale, dtype)
        check(out[i:i + 1], r, t)
