"""Drafted-token and beam operators of the paged pool against 64-bit references.

Tolerances are derived from the arithmetic, not fitted.  With h = finfo(t).eps / 2 the
half step of a storage type t:

* tree attention: the output is rounded once (h relative to its value); 16-bit pools
  round each probability (h relative, so h * sum_j w_j |v_j| on the sum).  A score is
  a 32-bit sum of D products, off by at most (D + 2) 2^-24 sum |q k| scale, which
  moves its weight by that much relatively, numerator and denominator both; 2^-19
  covers exp2, the running sums and the joins.
* rotation: cos and sin are within 2^-22, the two products and their sum add
  3 * 2^-24, all relative to |x0| + |x1|; then one rounding to t.
* moved rows and appended V rows are bit-exact; so are tokens, parents and tables.
* beam scores: log sums in 32-bit pieces (2^-20 relative covers exp2 and 16-term
  sums), and one rounding to fp32.
"""

from __future__ import annotations

import math

import numpy as np
import pytest

from conftest import HAS_GPU

pytestmark = pytest.mark.gpu

if HAS_GPU:
    import torch

    import beam
    import kvcache_ffi as ffi
    import paged

F16, BF16, F32 = "float16", "bfloat16", "float32"


class _Memory:
    def __init__(self, ptr, nbytes, keep):
        self.keep = keep
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1",
                                         "data": (ptr, False), "version": 2}


def raw(pool):
    """The pool's memory: (2, layers, pages, heads, page_size * D) in its type."""
    info = pool.info()
    n = info["bytes_per_layer"] * pool.num_layers
    shape = (pool.num_layers, pool.num_pages, pool.num_kv_heads, pool.page_size * pool.head_dim)
    return [torch.as_tensor(_Memory(info[x], n, pool), device="cuda").view(pool.dtype).view(shape)
            for x in ("k", "v")]


def make_pool(layers, pages, ps, hkv, d, dtype, fill=math.nan):
    pool = paged.PagedKVCache(layers, pages, ps, hkv, d, dtype=getattr(torch, dtype))
    for x in raw(pool):
        x.fill_(fill)
    return pool


def tables(need, seed, spare=3):
    """Distinct shuffled pages; unused entries name a page that holds NaN."""
    rng = np.random.default_rng(seed)
    total = int(sum(need)) + spare
    perm = rng.permutation(total).astype(np.int32)
    t = np.full((len(need), max(1, max(need))), perm[-1], dtype=np.int32)
    o = 0
    for i, n in enumerate(need):
        t[i, :n] = perm[o:o + n]
        o += n
    return torch.from_numpy(t).cuda(), total


def dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=dtype))).cuda()


def no_error():
    torch.cuda.synchronize()
    assert ffi.device_error(0) == (0, 0)


# -- tree attention ---------------------------------------------------------------------
def tree_case(dtype, d, h, hkv, ps, ctx, nodes, seed, mask="tree", scale=None, layer=1, words=None,
              rows=None, tweak=None):
    """Runs decode_tree on fresh inputs: (got, reference, tolerance)."""
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = getattr(torch, dtype)
    n_rows = len(ctx) if rows is None else max(rows) + 1
    need = [1] * n_rows
    for i, (c, n) in enumerate(zip(ctx, nodes)):
        need[i if rows is None else rows[i]] = max(1, -(-(c + n) // ps))
    bt, total = tables(need, seed)
    pool = make_pool(2, total, ps, hkv, d, dtype)
    ks, vs = [], []
    for i, (c, n) in enumerate(zip(ctx, nodes)):
        k = torch.randn(c + n, hkv, d, generator=g, device="cuda").to(dt)
        v = torch.randn(c + n, hkv, d, generator=g, device="cuda").to(dt)
        if tweak:
            tweak(i, k, v, c)
        ks.append(k)
        vs.append(v)
        if c + n:
            pool.append(layer, k, v, bt, torch.arange(c + n, dtype=torch.int32, device="cuda"),
                        torch.full((c + n,), i if rows is None else rows[i], dtype=torch.int32,
                                   device="cuda"))
    w = words or max(1, (max(nodes, default=0) + 31) // 32)
    sees, packed = [], []
    for n in nodes:
        if mask == "tree":
            par = [int(rng.integers(-1, j)) if j else -1 for j in range(n)]
            bits = paged.tree_masks(par, w).view(np.uint32) if n else np.zeros((0, w), np.uint32)
        else:  # any bits at all, some rows without one; bits past the nodes are noise
            bits = rng.integers(0, 1 << 32, (n, w), dtype=np.uint64).astype(np.uint32)
            bits[rng.random(n) < 0.3] = 0
        packed.append(bits)
        full = np.zeros((n, n), dtype=bool)
        for t in range(n):
            for j in range(n):
                full[t, j] = j <= t if mask is None else (
                    j // 32 < w and (int(bits[t, j // 32]) >> (j % 32)) & 1)
        sees.append(full)
    tokens = sum(nodes)
    q = torch.randn(tokens, h, d, generator=g, device="cuda").to(dt)
    out = torch.full((tokens + 2, h, d), 7.0, dtype=dt, device="cuda")
    m = None if mask is None else dev(np.concatenate(packed).view(np.int32))
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    plan = pool.plan_tree(ctx, nodes, h, rows=rows)
    pool.decode_tree(plan, layer, q, m, out, bt, scale)
    no_error()
    assert torch.all(out[tokens:] == 7.0)  # rows behind the last sequence
    half = torch.finfo(dt).eps / 2
    ref = torch.zeros(tokens, h, d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(ref)
    o = 0
    for i, (c, n) in enumerate(zip(ctx, nodes)):
        if n == 0:
            continue
        vis = np.ones((n, c + n), dtype=bool)
        vis[:, c:] = sees[i]
        vis = torch.from_numpy(vis).cuda()[:, None, :]
        kk = ks[i].double().repeat_interleave(h // hkv, 1)
        vv = vs[i].double().repeat_interleave(h // hkv, 1)
        qq = q[o:o + n].double()
        sc = torch.einsum("nhd,lhd->nhl", qq, kk) * scale
        mag = torch.einsum("nhd,lhd->nhl", qq.abs(), kk.abs()) * abs(scale)
        sc = torch.where(vis, sc, -math.inf)
        top = sc.amax(-1, keepdim=True)
        e = torch.where(vis, (sc - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
        tot = e.sum(-1, keepdim=True)
        wt = torch.where(tot > 0, e / tot, 0.0)
        vz = torch.nan_to_num(vv, 0.0, 0.0, 0.0) if tweak else vv
        ref[o:o + n] = torch.einsum("nhl,lhd->nhd", wt, vz)
        spread = torch.einsum("nhl,lhd->nhd", wt, vz.abs())
        ds = torch.where(vis, mag, 0.0).nan_to_num(0.0, 0.0, 0.0).amax(-1, keepdim=True)
        rel = 2 * (d + 2) * 2.0 ** -24 * ds + 2.0 ** -19 + (0 if dtype == F32 else 2 * half)
        tol[o:o + n] = half * ref[o:o + n].abs() + rel * spread + 1e-30
        if dtype == F16:
            tol[o:o + n] += 2.0 ** -25  # fp16 results below the normal range
        o += n
    plan.close()
    return out[:tokens], ref, tol


def check(got, ref, tol):
    bad = (got.double() - ref).abs() - tol
    assert torch.all(torch.isfinite(got)), "not finite"
    assert float(bad.max()) <= 0, f"over the bound by {float(bad.max()):.3g}"


TREE = [
    # D, H, Hkv, page, ctx, nodes
    (64, 8, 2, 16, [0], [1]),
    (64, 8, 2, 16, [1], [1]),
    (128, 8, 2, 16, [0, 5, 127, 128, 129, 0], [3, 0, 1, 2, 7, 31]),
    (128, 32, 8, 16, [1000, 17, 333], [16, 5, 33]),
    (128, 16, 2, 32, [700, 4000], [12, 9]),
    (64, 7, 1, 48, [100, 383, 384], [64, 1, 40]),
    (96, 6, 2, 16, [250, 90], [13, 64]),
    (128, 8, 2, 64, [2000, 100], [63, 64]),        # rows fill two tiles
    (128, 8, 1, 16, [515, 1], [40, 70]),           # more rows than one block holds
    (32, 4, 4, 16, [600, 31], [256, 200]),         # no head groups, the widest trees
    (256, 4, 2, 16, [300, 64, 0], [20, 65, 100]),
    (160, 4, 2, 16, [130], [9]),
    (192, 6, 2, 16, [130, 700], [9, 33]),
    (80, 4, 2, 16, [77, 200], [6, 20]),            # a head dim without tensor tiles
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", TREE, ids=[f"{c[0]}-{c[1]}-{c[2]}-{i}" for i, c in enumerate(TREE)])
def test_tree_attention(case, dtype):
    d, h, hkv, ps, ctx, nodes = case
    check(*tree_case(dtype, d, h, hkv, ps, ctx, nodes, seed=11 + d + len(ctx)))


LONG = [
    (64, 32, 4, 16, [3000, 17, 700], [30, 64, 5]),
    (128, 16, 2, 48, [2000, 0, 1, 3333], [33, 64, 7, 1]),
    (256, 12, 2, 32, [1500, 900], [64, 21]),
    (96, 8, 8, 16, [5000, 63, 64, 65], [9, 250, 3, 17]),
    (12, 6, 2, 16, [4000, 1000], [64, 100]),          # fp32 only: 24-byte rows of 16-bit types
]


@pytest.mark.parametrize("case,dtype", [(c, t) for c in LONG for t in (F32, F16, BF16)
                                        if c[0] != 12 or t == F32])
def test_tree_long_batches(case, dtype):
    """Batches with more tiles than the GPU takes at once: pieces are cut and joined."""
    d, h, hkv, ps, ctx, nodes = case
    check(*tree_case(dtype, d, h, hkv, ps, ctx, nodes, seed=100 + d))
    check(*tree_case(dtype, d, h, hkv, ps, ctx, nodes, seed=200 + d, mask="any", scale=-0.05))

    def poison(i, k, v, c):      # node 2 holds anything, and nobody sees it
        if k.shape[0] > c + 2:
            k[c + 2], v[c + 2] = math.nan, math.inf
    orig = paged.tree_masks

    def without_2(parents, words=None):
        m = orig([-1] * len(parents), words)
        if len(m) > 2:
            m[2] = 0
        return m
    paged.tree_masks = without_2
    try:
        check(*tree_case(dtype, d, h, hkv, ps, ctx, nodes, seed=300 + d, tweak=poison))
    finally:
        paged.tree_masks = orig


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_tree_values_that_are_seen_come_through(dtype):
    """A drafted V that is not finite reaches the rows that see it, and only there."""
    dt = getattr(torch, dtype)
    ctx, n, d = 200, 40, 128
    pool = make_pool(1, 16, 16, 2, d, dtype, fill=0.0)
    pool.fill_normal(seed=3)
    bt = dev(np.arange(16).reshape(1, 16))
    k = torch.randn(n, 2, d, device="cuda").to(dt)
    v = torch.randn(n, 2, d, device="cuda").to(dt)
    v[3, 1, 5], v[7, 0, 9], v[9, 0, 9] = math.inf, math.nan, -math.inf
    pool.append(0, k, v, bt, torch.arange(ctx, ctx + n, dtype=torch.int32, device="cuda"))
    par = [-1, 0, 1, 2, 3, 2, 5, 6, 2, 8] + [4] * 30      # 3 and 9 lie on different branches
    q = torch.randn(n, 8, d, device="cuda").to(dt)
    out = torch.zeros_like(q)
    pool.decode_tree(pool.plan_tree([ctx], [n], 8), 0, q, dev(paged.tree_masks(par)), out, bt, 0.09)
    no_error()
    seen = [{j for j in range(n) if int(paged.tree_masks(par, 2)[i, j // 32]) >> (j % 32) & 1}
            for i in range(n)]
    o = out.float().cpu().numpy()
    for i in range(n):
        for h in range(8):
            for x in (5, 9):
                val = o[i, h, x]
                if x == 5 and h >= 4 and 3 in seen[i]:
                    assert val == np.inf
                elif x == 9 and h < 4 and 7 in seen[i]:
                    assert np.isnan(val)
                elif x == 9 and h < 4 and 9 in seen[i]:
                    assert val == -np.inf
                else:
                    assert np.isfinite(val)
            assert np.all(np.isfinite(np.delete(o[i, h], [5, 9])))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_tree_any_mask_and_empty_rows(dtype):
    got, ref, tol = tree_case(dtype, 128, 8, 2, 16, [0, 40, 0], [40, 33, 9], seed=3, mask="any")
    check(got, ref, tol)
    empty = (ref == 0).all(-1)
    assert bool(empty.any())  # rows that see nothing are there, and are zero
    assert torch.all(got[empty] == 0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_tree_chain_short_masks_rows_and_scales(dtype):
    check(*tree_case(dtype, 64, 8, 4, 16, [200, 3], [20, 5], seed=5, mask=None))
    # mask rows shorter than the tree: the nodes past them are not seen
    check(*tree_case(dtype, 64, 8, 4, 16, [50], [70], seed=6, mask="any", words=1))
    check(*tree_case(dtype, 64, 8, 4, 16, [50, 400], [7, 9], seed=7, rows=[3, 1]))
    for s in (0.0, -0.1, 1.0):
        check(*tree_case(dtype, 64, 4, 2, 16, [130, 9], [7, 9], seed=8, scale=s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_tree_large_scores(dtype):
    """Scores that grow along the context: the running max moves at every tile."""
    def grow(i, k, v, c):
        ramp = torch.linspace(0.1, 6.0, k.shape[0], device="cuda")[:, None, None]
        k.copy_((k.float() * ramp).to(k.dtype))
    check(*tree_case(dtype, 128, 8, 2, 16, [1500, 700], [9, 20], seed=9, tweak=grow))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_tree_masked_values_do_not_spread(dtype, value):
    """A drafted node that nobody sees may hold anything in K and V."""
    def poison(i, k, v, c):
        k[c + 2], v[c + 2] = value, value

    d, h, hkv, ctx, nodes = 128, 8, 2, [300, 60], [9, 6]
    orig = paged.tree_masks

    def without_2(parents, words=None):
        m = orig([-1] * len(parents), words)
        m[2] = 0
        return m
    paged.tree_masks = without_2
    try:
        got, ref, tol = tree_case(dtype, d, h, hkv, 16, ctx, nodes, seed=10, tweak=poison)
    finally:
        paged.tree_masks = orig
    check(got, ref, tol)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_tree_graph_streams_and_repeats(dtype):
    """Captured and replayed, on another stream, and twice: the same bits."""
    dt = getattr(torch, dtype)
    pool = make_pool(1, 64, 16, 2, 128, dtype, fill=0.0)
    pool.fill_normal(seed=5)
    bt = dev(np.random.default_rng(0).permutation(64).reshape(2, 32))
    q = torch.randn(30, 8, 128, device="cuda").to(dt)
    mask = dev(np.concatenate([paged.tree_masks([-1] * 13), paged.tree_masks(range(-1, 16))]))
    plan = pool.plan_tree([400, 90], [13, 17], 8)
    a, b, c = (torch.zeros_like(q) for _ in range(3))
    pool.decode_tree(plan, 0, q, mask, a, bt, 0.09)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool.decode_tree(plan, 0, q, mask, b, bt, 0.09)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.decode_tree(plan, 0, q, mask, c, bt, 0.09)
        pool.decode_tree(plan, 0, c, mask, b, bt, 0.09)
        pool.decode_tree(plan, 0, q, mask, b, bt, 0.09)
    c.zero_()
    graph.replay()
    graph.replay()
    no_error()
    assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("d", [32, 128])
def test_tree_on_two_streams_at_once(d):
    """Two plans on two streams share the SMs and their tensor memory."""
    pool = make_pool(1, 512, 16, 4, d, F16, fill=0.0)
    pool.fill_normal(seed=9)
    bt = dev(np.random.default_rng(1).permutation(512).reshape(4, 128))
    qs = [torch.randn(n, 16, d, device="cuda").half() for n in (4 * 20, 4 * 63)]
    plans = [pool.plan_tree([1900, 700, 33, 1200], [n] * 4, 16) for n in (20, 63)]
    want = [torch.zeros_like(q) for q in qs]
    for p, q, o in zip(plans, qs, want):
        pool.decode_tree(p, 0, q, None, o, bt, 0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [torch.zeros_like(q) for q in qs]
    for _ in range(30):
        for st, p, q, o in zip(streams, plans, qs, got):
            pool.decode_tree(p, 0, q, None, o, bt, 0.1, stream=st)
    no_error()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_pages_past_four_gigabytes():
    """Every operator on pages whose byte offsets need more than 32 bits."""
    pages, ps, hkv, d = 140000, 16, 8, 128                  # 4.6 GB of K, and of V
    pool = paged.PagedKVCache(1, pages, ps, hkv, d)
    ctx, n, h = 100, 20, 32
    table = np.arange(pages - 8, pages, dtype=np.int32)[::-1].copy().reshape(1, 8)
    bt = dev(table)
    k = torch.randn(ctx + n, hkv, d, device="cuda").half()
    v = torch.randn(ctx + n, hkv, d, device="cuda").half()
    q = torch.randn(n, h, d, device="cuda").half()
    pos = torch.arange(ctx + n, dtype=torch.int32, device="cuda")
    zero = torch.zeros_like(pos)
    # angle 0 leaves the rows as they are
    pool.append_rope(0, None, k, v, bt, pos, rope_positions=zero)
    gk, gv = pool.gather(0, bt, 0, 0, ctx + n)
    assert torch.equal(gk, k) and torch.equal(gv, v)
    out = torch.zeros_like(q)
    pool.decode_tree(pool.plan_tree([ctx], [n], h), 0, q, None, out, bt, 0.09)
    low = paged.PagedKVCache(1, 8, ps, hkv, d)
    bt2, want = dev(np.arange(8).reshape(1, 8)), torch.zeros_like(q)
    low.append_rope(0, None, k, v, bt2, pos, rope_positions=zero)
    low.decode_tree(low.plan_tree([ctx], [n], h), 0, q, None, want, bt2, 0.09)
    no_error()
    assert torch.equal(out, want)
    pool.commit_tree(bt, dev([ctx]), dev([[3, 7, 19]]), dev([3]))
    gk, _ = pool.gather(0, bt, 0, ctx, 3)
    assert torch.equal(gk, k[[ctx + 3, ctx + 7, ctx + 19]])
    beams = dev(np.arange(pages - 8, pages).reshape(2, 4))   # rows of 4 pages, 37 positions
    old = [pool.gather(0, beams, r, 0, 37) for r in range(2)]
    pool.reorder_beams(beams, dev([[1, 0]]), dev([37]))
    for r in range(2):
        for x, y in zip(old[1 - r], pool.gather(0, beams, r, 0, 37)):
            assert torch.equal(x, y)
    no_error()


def test_tree_bad_page_is_reported():
    pool = make_pool(1, 8, 16, 2, 64, F16, fill=0.0)
    bt = dev([[0, 99, 2, 3]])
    q = torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda")
    plan = pool.plan_tree([40], [3], 4)
    pool.decode_tree(plan, 0, q, None, torch.empty_like(q), bt, 0.1)
    torch.cuda.synchronize()
    assert ffi.device_error(0) == (1, 99)
    no_error()


# -- rotate + append ----------------------------------------------------------------------
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("dtype,d,hkv,h,ps", [
    (F32, 64, 4, 32, 16), (F16, 128, 8, 32, 16), (BF16, 128, 2, 14, 48), (F16, 8, 3, 5, 16),
    (F16, 40, 2, 4, 16), (BF16, 256, 1, 3, 32), (F32, 12, 2, 2, 16)])
def test_append_rope(dtype, d, hkv, h, ps, neox):
    rng = np.random.default_rng(d + h)
    dt = getattr(torch, dtype)
    counts, ctx = [5, 1, 40, 2], [0, ps - 1, 1003, 131072]
    need = [-(-(c + n) // ps) for c, n in zip(ctx, counts)]
    cols = max(need)
    bt = np.zeros((4, cols), dtype=np.int32)   # only the pages the new rows touch are in the pool
    perm = iter(rng.permutation(40))
    for i, (c, n) in enumerate(zip(ctx, counts)):
        for p in range(c // ps, need[i]):
            bt[i, p] = next(perm)
    n = sum(counts)
    pool = make_pool(2, 40, ps, hkv, d, dtype, fill=3.0)
    before = [x.clone() for x in raw(pool)]
    rows = np.repeat(np.arange(4), counts)
    pos = np.concatenate([c + np.arange(k) for c, k in zip(ctx, counts)])
    ang = pos + rng.integers(-3, 4, n)
    pad = [3, 20]
    slots = pos.copy()
    slots[pad] = -1
    g = torch.Generator(device="cuda")
    g.manual_seed(d)
    qkv = torch.randn(n, h + 2 * hkv, d, generator=g, device="cuda").to(dt)
    q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
    q_out = torch.full((n, h, d), 5.0, dtype=dt, device="cuda")
    got = pool.append_rope(1, q, k, v, dev(bt), dev(slots), rows=dev(rows), rope_positions=dev(ang),
                           q_out=q_out, freq_base=500000.0, neox=neox)
    assert got is q_out
    no_error()
    freq = 500000.0 ** (-2.0 * np.arange(d // 2) / d)
    th = torch.from_numpy(ang[:, None].astype(np.float64) * freq).cuda()[:, None]

    def rot(x):
        x = x.double()
        a, b = (x[..., :d // 2], x[..., d // 2:]) if neox else (x[..., 0::2], x[..., 1::2])
        y0, y1 = a * th.cos() - b * th.sin(), a * th.sin() + b * th.cos()
        t = a.abs() + b.abs()
        cat = (lambda u, w: torch.cat([u, w], -1)) if neox else (
            lambda u, w: torch.stack([u, w], -1).flatten(-2))
        return cat(y0, y1), cat(t, t)

    half = torch.finfo(dt).eps / 2
    slack = 2.0 ** -22 + 3 * 2.0 ** -24 + 2.0 ** -23   # and the angle's rounding to fp32
    live = [i for i in range(n) if i not in pad]
    ref, mag = rot(q)
    tol = half * ref.abs() + slack * mag + (2.0 ** -25 if dtype == F16 else 0)
    assert torch.all((q_out.double() - ref).abs()[live] <= tol[live])
    assert torch.all(q_out[pad] == 5.0)
    kref, kmag = rot(k)
    ktol = half * kref.abs() + slack * kmag + (2.0 ** -25 if dtype == F16 else 0)
    pool_bt = dev(bt)
    for i in live:
        kk, vv = pool.gather(1, pool_bt, int(rows[i]), int(pos[i]), 1)
        assert torch.all((kk[0].double() - kref[i]).abs() <= ktol[i])
        assert torch.equal(vv[0], v[i])
    # nothing else changed: the other layer, and as many elements as there are new rows
    after = raw(pool)
    for x, y in zip(before, after):
        assert torch.equal(x[0], y[0])
        assert int((x[1] != y[1]).sum()) <= len(live) * hkv * d
    # without q, packed rows, default rows and angles
    pool2 = make_pool(1, 40, ps, hkv, d, dtype, fill=3.0)
    assert pool2.append_rope(0, None, k[:5].contiguous(), v[:5].contiguous(), pool_bt,
                             dev(np.arange(5)), neox=neox) is None
    no_error()
    # q rotated in place gives the same bits
    packed = q.contiguous()
    pool.append_rope(1, packed, k, v, pool_bt, dev(slots), rows=dev(rows),
                     rope_positions=dev(ang), q_out=packed, freq_base=500000.0, neox=neox)
    no_error()
    assert torch.equal(packed[live], q_out[live])


def test_append_rope_reports_bad_places():
    pool = make_pool(1, 4, 16, 1, 64, F16, fill=0.0)
    k = torch.ones(1, 1, 64, dtype=torch.float16, device="cuda")
    bt = dev([[0, 9]])
    for pos, row, code in ((32, 0, 3), (0, 1, 3), (0, -1, 3), (16, 0, 1)):
        pool.append_rope(0, None, k, k, bt, dev([pos]), rows=dev([row]))
        torch.cuda.synchronize()
        assert ffi.device_error(0)[0] == code
    assert all(bool((x == 0).all()) for x in raw(pool))


# -- commit --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,d,hkv,ps,layers", [(F32, 64, 2, 16, 3), (F16, 128, 4, 16, 2),
                                                   (BF16, 40, 1, 48, 1)])
def test_commit_tree(dtype, d, hkv, ps, layers):
    rng = np.random.default_rng(7)
    ctx = [0, ps - 1, 100, 5, 31]
    nodes = [1, 30, 60, 256, 4]
    paths = [[0], [0, 1, 2, 29], [2, 5, 6, 40, 41, 42, 43, 50, 51, 52, 59], list(range(1, 250, 7)),
             []]
    need = [-(-(c + n) // ps) for c, n in zip(ctx, nodes)]
    bt, total = tables(need, 1)
    pool = make_pool(layers, total, ps, hkv, d, dtype)
    for x in raw(pool):
        x.copy_(torch.randn(x.shape, device="cuda").to(x.dtype))
    longest = max(len(p) for p in paths)
    mat = rng.integers(-9, 999, (5, longest + 1))   # entries past a path are never read
    for i, p in enumerate(paths):
        mat[i, :len(p)] = p
    old = [[pool.gather(l, bt, i, 0, c + n) for i, (c, n) in enumerate(zip(ctx, nodes))]
           for l in range(layers)]
    pool.commit_tree(bt, dev(ctx), dev(mat), dev([len(p) for p in paths]))
    no_error()
    for l in range(layers):
        for i, (c, n) in enumerate(zip(ctx, nodes)):
            for x, y in zip(old[l][i], pool.gather(l, bt, i, 0, c + n)):
                want = x.clone()
                for j, a in enumerate(paths[i]):
                    want[c + j] = x[c + a]
                assert torch.equal(y, want)


def test_commit_tree_rejects_paths():
    pool = make_pool(1, 8, 16, 1, 64, F16, fill=0.0)
    for x in raw(pool):
        x.copy_(torch.randn(x.shape, device="cuda").to(x.dtype))
    before = [x.clone() for x in raw(pool)]
    bt = dev([[0, 1], [2, 3]])
    for path, ln, ctx in (([1, 1], 2, 0), ([3, 2], 2, 0), ([-1, 5], 2, 0), ([1, 300], 2, 0),
                          ([1, 5], 3, 0), ([1, 5], 2, 30), ([0, 1], 2, -4)):
        pool.commit_tree(bt, dev([ctx, 0]), dev([path, [0, 0]]), dev([ln, 0]))
        torch.cuda.synchronize()
        assert ffi.device_error(0)[0] == 3
    assert all(torch.equal(x, y) for x, y in zip(before, raw(pool)))


# -- beam selection ----------------------------------------------------------------------------
def select_ref(logits, scores, n_out):
    x = logits.double().cpu().numpy()
    n, b = scores.shape
    x = x.reshape(n, b, -1)
    cum = scores.double().cpu().numpy()
    out = []
    for i in range(n):
        cand = []
        for j in range(b):
            r = x[i, j]
            ok = np.isfinite(r)
            lse = r[ok].max() + np.log(np.exp(r[ok] - r[ok].max()).sum()) if ok.any() else 0.0
            s = np.where(ok & np.isfinite(cum[i, j]), cum[i, j] + (np.where(ok, r, 0.0) - lse), -np.inf)
            cand.append(s)
        s = np.concatenate(cand)
        order = np.argsort(-s, kind="stable")[:n_out]
        out.append((order % x.shape[2], order // x.shape[2], s[order]))
    return [np.stack([o[k] for o in out]) for k in range(3)]


def check_select(logits, scores, n_out, sel=None):
    n, b = scores.shape
    sel = sel or beam.BeamSelector(n, b, logits.shape[1], n_out)
    tok, par, best = sel.select(logits, scores, n_out)
    no_error()
    rt, rp, rs = select_ref(logits, scores, n_out)
    assert np.array_equal(par.cpu().numpy(), rp)
    assert np.array_equal(tok.cpu().numpy(), rt)
    got = best.double().cpu().numpy()
    fin = np.isfinite(rs)
    assert np.array_equal(fin, np.isfinite(got)) and np.all(got[~fin] == -np.inf)
    assert np.all(np.abs(got[fin] - rs[fin]) <= 2.0 ** -20 + 2.0 ** -24 * np.abs(rs[fin]))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,b,v,k", [(1, 1, 1, 1), (1, 1, 40, 32), (2, 3, 2, 6), (3, 4, 33, 8),
                                     (2, 16, 5000, 32), (1, 4, 32000, 8), (5, 3, 8193, 6),
                                     (2, 8, 50257, 16), (1, 2, 128256, 4)])
def test_beam_select(n, b, v, k, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(v + b)
    logits = (3 * torch.randn(n * b, v, generator=g, device="cuda")).to(getattr(torch, dtype))
    scores = -5 * torch.rand(n, b, generator=g, device="cuda")
    check_select(logits, scores, k)
    scores[:, 1:] = -math.inf      # the first step: one beam
    if v >= k:
        check_select(logits, scores, k)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_beam_select_ties_and_masks(dtype):
    dt = getattr(torch, dtype)
    sel = beam.BeamSelector(4, 8, 20000, 32)
    same = torch.zeros(6, 9001, dtype=dt, device="cuda")
    check_select(same, torch.zeros(2, 3, device="cuda"), 32, sel)       # every candidate ties
    same[:, 1::2] = -0.0
    check_select(same, torch.zeros(2, 3, device="cuda"), 32, sel)
    x = torch.randn(6, 9001, device="cuda").to(dt)
    x[0] = -math.inf                     # a row whose mask leaves nothing
    x[1, 5:] = -math.inf                 # five tokens are left
    x[2, 17] = math.inf
    x[2, 18] = math.nan
    x[3] = math.nan
    x[4] = torch.finfo(dt).min           # a mask of the type's lowest value
    x[4, 7000] = 1.0
    check_select(x, torch.zeros(2, 3, device="cuda"), 20, sel)
    check_select(x, torch.tensor([[math.nan, 0, -1], [math.inf, -2, -1.]], device="cuda"), 20, sel)
    check_select(x, torch.full((2, 3), -math.inf, device="cuda"), 20, sel)
    twice = x[5:].repeat(4, 1)           # equal beams: the lower beam, then the lower token
    check_select(twice, torch.zeros(1, 4, device="cuda"), 32, sel)
    peak = torch.zeros(1, 9001, dtype=dt, device="cuda")
    peak[0, 64:96] = 5.0                 # all winners next to each other
    check_select(peak, torch.zeros(1, 1, device="cuda"), 32, sel)
    up = torch.arange(9001, device="cuda").float().div(1000).to(dt)[None]
    check_select(up.contiguous(), torch.zeros(1, 1, device="cuda"), 32, sel)
    check_select(up.flip(1).contiguous(), torch.zeros(1, 1, device="cuda"), 32, sel)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_beam_select_strided_rows_and_graph(dtype):
    dt = getattr(torch, dtype)
    buf = torch.randn(6, 7003, device="cuda").to(dt)
    buf[:, :3], buf[:, 7000:] = math.inf, math.inf
    logits = buf[:, 3:7000]              # rows start on every alignment
    scores = torch.zeros(2, 3, device="cuda")
    check_select(logits, scores, 9)
    sel = beam.BeamSelector(2, 3, 6997, 9)
    want = sel.select(logits, scores, 9)
    out = tuple(torch.zeros_like(x) for x in want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sel.select(logits, scores, 9, out=out)
        sel.select(logits, scores, 9, out=out)
    g.replay()
    g.replay()
    no_error()
    assert all(torch.equal(x, y) for x, y in zip(want, out))


# -- beam reorder ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,d,hkv,ps,layers,beams", [
    (F32, 64, 2, 16, 2, 4), (F16, 128, 4, 16, 3, 16), (BF16, 64, 1, 48, 1, 3), (F16, 40, 2, 32, 2, 5),
    (F16, 64, 1, 16, 1, 1)])
def test_reorder_beams(dtype, d, hkv, ps, layers, beams):
    rng = np.random.default_rng(beams)
    ctx = [0, 1, ps, 5 * ps - 1, 3 * ps + 5, 6 * ps]
    n, w = len(ctx), 6
    pages = n * beams * w
    bt = rng.permutation(pages).reshape(n * beams, w).astype(np.int32)
    pool = make_pool(layers, pages, ps, hkv, d, dtype)
    for x in raw(pool):
        x.copy_(torch.randn(x.shape, device="cuda").to(x.dtype))
    parents = rng.integers(0, beams, (n, beams))
    parents[1] = (np.arange(beams) + 1) % beams          # every beam moves, in a ring
    table = dev(bt)
    old = [[pool.gather(l, table, r, 0, c) for r, c in enumerate(np.repeat(ctx, beams))]
           for l in range(layers)]
    before = [x.clone() for x in raw(pool)]
    pool.reorder_beams(table, dev(parents), dev(ctx))
    no_error()
    new = table.cpu().numpy()
    for i, c in enumerate(ctx):
        full = c // ps
        for b in range(beams):
            r, p = i * beams + b, i * beams + int(parents[i, b])
            assert np.array_equal(new[r, :full], bt[p, :full])
            assert np.array_equal(new[r, full:], bt[r, full:])
            if c == 0:
                continue
            for l in range(layers):
                for x, y in zip(old[l][p], pool.gather(l, table, r, 0, c)):
                    assert torch.equal(x, y)
    # full pages and the rows behind the context are as they were
    for x, y in zip(before, raw(pool)):
        for i, c in enumerate(ctx):
            for r in range(i * beams, (i + 1) * beams):
                cols = [j for j in range(w) if j != c // ps or c % ps == 0]
                assert torch.equal(x[:, bt[r, cols]], y[:, bt[r, cols]])


def test_reorder_rejects_what_it_cannot_do():
    pool = make_pool(1, 8, 16, 1, 64, F16, fill=0.0)
    for x in raw(pool):
        x.copy_(torch.randn(x.shape, device="cuda").to(x.dtype))
    before = [x.clone() for x in raw(pool)]
    for table, par, ctx, code in (([[0, 1], [2, 3]], [1, 2], 20, 3), ([[0, 1], [2, 3]], [1, -1], 20, 3),
                                  ([[0, 1], [2, 3]], [1, 0], 33, 3), ([[0, 1], [2, 3]], [1, 0], -1, 3),
                                  ([[0, 1], [2, 1]], [1, 0], 20, 1), ([[0, 1], [2, 8]], [1, 0], 20, 1)):
        t = dev(table)
        pool.reorder_beams(t, dev([par]), dev([ctx]))
        torch.cuda.synchronize()
        assert ffi.device_error(0)[0] == code
        assert np.array_equal(t.cpu().numpy(), np.array(table))
    assert all(torch.equal(x, y) for x, y in zip(before, raw(pool)))


# -- refusals ----------------------------------------------------------------------------------
def test_refusals():
    pool = make_pool(2, 8, 16, 2, 64, F16, fill=0.0)
    z = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    k, bt, pos = z(3, 2, 64), dev([[0, 1], [2, 3]]), dev([0, 1, 2])
    q = z(3, 4, 64)
    with pytest.raises(IndexError):
        pool.append_rope(2, None, k, k, bt, pos)
    with pytest.raises(ValueError):
        pool.append_rope(0, None, k.float(), k, bt, pos)
    with pytest.raises(ValueError):
        pool.append_rope(0, None, k, k[:, :1], bt, pos)
    with pytest.raises(ValueError):
        pool.append_rope(0, None, k, k, bt, pos, freq_base=0.0)
    with pytest.raises(ValueError, match="packed"):
        pool.append_rope(0, None, k[:1].expand(3, 2, 64), k, bt, pos)
    with pytest.raises(ValueError, match="aligned"):
        pool.append_rope(0, None, z(3 * 128 + 1)[1:].view(3, 2, 64), k, bt, pos)
    with pytest.raises(ValueError, match="16 bytes"):
        pool.append_rope(0, None, z(3, 129)[:, :128].unflatten(1, (2, 64)), k, bt, pos)
    with pytest.raises(ValueError, match="in place"):
        wide = z(3, 6, 64)
        pool.append_rope(0, wide[:, :4], k, k, bt, pos, q_out=wide.view(-1)[:3 * 4 * 64])
    for bad in (([-1], [1], 4), ([1], [257], 4), ([1], [-1], 4), ([1], [1], 3), ([1], [1], 0)):
        with pytest.raises(ValueError):
            pool.plan_tree(*bad)
    with pytest.raises(ValueError):
        pool.plan_tree([1, 2], [1], 4)
    with pytest.raises(ValueError):
        pool.plan_tree([1], [1], 4, rows=[-1])
    plan = pool.plan_tree([20], [3], 4)
    out = torch.empty_like(q)
    with pytest.raises(IndexError):
        pool.decode_tree(plan, 2, q, None, out, bt, 0.1)
    with pytest.raises(IndexError, match="width"):
        pool.decode_tree(plan, 0, q, None, out, bt[:, :1].contiguous(), 0.1)
    with pytest.raises(IndexError, match="row"):
        pool.decode_tree(pool.plan_tree([20], [3], 4, rows=[2]), 0, q, None, out, bt, 0.1)
    with pytest.raises(ValueError):
        pool.decode_tree(plan, 0, q, None, out, bt, math.nan)
    with pytest.raises(ValueError):
        pool.decode_tree(plan, 0, q[:2], None, out, bt, 0.1)
    with pytest.raises(ValueError):
        pool.decode_tree(plan, 0, q, dev([[1], [1]]), out, bt, 0.1)
    other = make_pool(1, 8, 16, 1, 64, F16, fill=0.0)
    with pytest.raises(ValueError, match="geometry"):
        other.decode_tree(plan, 0, q, None, out, bt, 0.1)
    with pytest.raises(ValueError, match="built"):
        fresh = paged.TreePlan()
        ffi.check(ffi.lib.kvc_decode_tree(pool.handle, fresh.handle, 0, q.data_ptr(), None, 0,
                                          out.data_ptr(), bt.data_ptr(), 2, 0.1, None))
    with pytest.raises(ValueError):
        pool.commit_tree(bt, dev([1, 2]), dev([[0], [0], [0]]), dev([1, 1]))
    with pytest.raises(IndexError):
        pool.commit_tree(bt, dev([1, 2, 3]), dev([[0], [0], [0]]), dev([1, 1, 1]))
    with pytest.raises(ValueError):
        pool.reorder_beams(bt, dev([[0, 1, 2]]), dev([5]))
    with pytest.raises(ValueError):
        pool.reorder_beams(dev(np.zeros((17, 2))), dev([list(range(17))]), dev([5]))
    for bad in ((0, 1, 1, 1), (1, 17, 9, 1), (1, 1, 9, 33), (1, 1, 0, 1), (9999, 16, 9, 1)):
        with pytest.raises(ValueError):
            beam.BeamSelector(*bad)
    sel = beam.BeamSelector(2, 2, 100, 8)
    lg, sc = z(4, 100), z(2, 2, t=torch.float32)
    for bad in ((lg, sc, 9), (z(4, 101), sc, 8), (z(4, 3), sc, 7), (z(6, 100), z(3, 2, t=torch.float32), 2),
                (lg.int(), sc, 2), (lg, sc.half(), 2), (lg[:1].expand(4, 100), sc, 2), (lg, sc, 0),
                (lg.t().contiguous().t(), sc, 2)):
        with pytest.raises(ValueError):
            sel.select(*bad)
    no_error()
