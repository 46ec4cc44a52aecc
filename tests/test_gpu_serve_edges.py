"""Head norms with rotation, shared prefixes, summed weights and eviction where they can go
wrong: prefixes long enough to be shared, in every head dim of the tensor cores, beside own
positions of any length; captured and replayed calls, several streams, pools past four
gigabytes, and refusals.  References and tolerances as in test_gpu_serve_ops."""

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

from test_gpu_serve_ops import attend64, check, evict_case, keep64, norm_case, shared_case, weigh_case
from test_gpu_spec_ops import BF16, F16, F32, dev, make_pool, no_error, raw, tables

# -- prefixes that are shared (more than 32 MB a layer saved) -------------------------------------
LARGE = [
    # D, H, Hkv, page, group sizes, prefixes, own lengths
    (96, 12, 2, 16, [30, 6], [2048, 1040], lambda i: 7 * i % 300),
    (256, 4, 2, 16, [20, 3], [2048, 416], lambda i: 40 * i % 290),
    (192, 20, 1, 16, [60], [1600], lambda i: i % 4 * 33),             # 20 q-heads in blocks of 128 rows
    (160, 6, 3, 32, [25], [1280], lambda i: 31 * i),
    (64, 7, 1, 48, [150], [960], lambda i: i % 9),                    # 7 q-heads in blocks of 256
    (32, 8, 2, 16, [2] * 40, [2048] * 40, lambda i: 3 * i),
    (128, 8, 2, 64, [4, 1, 50, 2], [4096, 64, 2048, 0], lambda i: [0, 1, 700, 33, 2][i % 5]),
    (128, 80, 1, 16, [12], [8192], lambda i: 100 * i),                # ten chunks of 8 q-heads
    (128, 16, 4, 16, [70], [1024], lambda i: 0),                      # nothing but the prefix
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", LARGE, ids=[f"{c[0]}-{c[1]}-{i}" for i, c in enumerate(LARGE)])
def test_large_shared_prefixes(case, dtype):
    d, h, hkv, ps, sizes, prefix, own = case
    own = [own(i) for i in range(sum(sizes))]
    if 0 in prefix:      # (a member of a group without a prefix may be empty)
        own[-1] = 0
    shared_case(dtype, d, h, hkv, ps, sizes, prefix, own, seed=d + h)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_shared_prefix_scales_rows_and_growing_scores(dtype):
    def grow(k, v, a):
        ramp = (a + torch.arange(k.shape[0], device="cuda")) / 400.0
        k.copy_((k.float() * ramp[:, None, None]).to(k.dtype))
    own = [i * 17 % 400 for i in range(40)]
    shared_case(dtype, 128, 16, 4, 16, [40], [1024], own, seed=1, scale=-0.1)
    shared_case(dtype, 128, 16, 4, 16, [40], [1024], own, seed=2, scale=0.0)
    shared_case(dtype, 128, 16, 4, 16, [40], [1024], own, seed=3, tweak=grow,
                rows=[(7 * i) % 41 for i in range(40)])


def shared_state(dtype, n, prefix, own, hkv=4, d=128, h=16, ps=16, seed=0):
    """A pool, its table and a plan that shares `prefix` positions: (pool, table, lengths, plan)."""
    first = prefix // ps
    width = first + -(-max(own) // ps) + 1
    pool = make_pool(1, first + n * (width - first), ps, hkv, d, dtype, fill=0.0)
    pool.fill_normal(seed=seed + 1)
    t = np.zeros((n, width), np.int32)
    t[:, :first] = np.random.default_rng(seed).permutation(first)
    t[:, first:] = first + np.arange(n * (width - first)).reshape(n, -1)
    lens = [prefix + x for x in own]
    return pool, dev(t), lens, pool.plan_shared(lens, [n], [prefix], h)


def dense(pool, bt, row, length):
    return pool.gather(0, bt, row, 0, length)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_shared_decode_captured_and_on_two_streams(dtype):
    """The call's kernels run beside one another and beside those of another plan's call; a
    replayed one starts where the last replay ended."""
    dt = getattr(torch, dtype)
    made = [shared_state(dtype, 24, 2048, [7 * i + 1 for i in range(24)], seed=1),
            shared_state(dtype, 40, 1024, [i % 5 for i in range(40)], seed=2)]
    qs = [torch.randn(len(m[2]), 16, 128, device="cuda").to(dt) for m in made]
    want = []
    for (pool, bt, lens, plan), q in zip(made, qs):
        out = torch.zeros_like(q)
        pool.decode_shared(plan, 0, q, out, bt, 0.09)
        no_error()
        for i in (0, len(lens) // 2, len(lens) - 1):
            ref, tol, _, _ = attend64(q[i:i + 1], *dense(pool, bt, i, lens[i]), 0.09, dtype)
            check(out[i:i + 1], ref, tol)
        want.append(out)
    streams = [torch.cuda.Stream() for _ in made]
    outs = [torch.zeros_like(q) for q in qs]
    for _ in range(6):
        for (pool, bt, lens, plan), q, s, o in zip(made, qs, streams, outs):
            s.wait_stream(torch.cuda.current_stream())
            pool.decode_shared(plan, 0, q, o, bt, 0.09, stream=s)
    no_error()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    graphs = []
    for (pool, bt, lens, plan), q, s, o in zip(made, qs, streams, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for _ in range(3):
                pool.decode_shared(plan, 0, q, o, bt, 0.09)
        graphs.append(g)
    for o in outs:
        o.zero_()
    for k in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    no_error()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_shared_decode_sees_what_was_written_just_before(dtype):
    """Rows, q and the table change right in front of every call."""
    dt = getattr(torch, dtype)
    n, prefix, ps, hkv, d = 24, 2048, 16, 4, 128
    own = [1 + 3 * i for i in range(n)]
    pool, bt, lens, plan = shared_state(dtype, n, prefix, own)
    rot = paged.Rotation(d)
    outs, wants = [], []
    rows, pos = dev(np.arange(n)), dev([x - 1 for x in lens])
    base = bt.clone()
    for step in range(4):
        qkv = torch.randn(n, 16 + 2 * hkv, d, device="cuda").to(dt)
        bt.copy_(base)
        if step % 2:                    # own pages change places
            bt[:, prefix // ps:] = base[:, prefix // ps:].flip(0)
        q = pool.append_norm_rope(0, qkv[:, :16], qkv[:, 16:16 + hkv], qkv[:, 16 + hkv:], bt, pos, rot,
                                  rows=rows)
        out = torch.empty_like(q)
        pool.decode_shared(plan, 0, q, out, bt, 0.09)
        outs.append(out)
        some = (0, 11, n - 1)
        wants.append([(i, attend64(q[i:i + 1], *dense(pool, bt, i, lens[i]), 0.09, dtype)) for i in some])
    no_error()
    for out, want in zip(outs, wants):
        for i, (ref, tol, _, _) in want:
            check(out[i:i + 1], ref, tol)


# -- captured steps --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("new", [1, 9])
def test_a_captured_step_of_weights_and_eviction(dtype, new):
    dt = getattr(torch, dtype)
    n, ps, hkv, d, h, budget = 3, 16, 2, 128, 8, 200
    ctx = [300, 40, 210]
    start = torch.rand(1, n, hkv, 24 * ps, device="cuda")

    def step(pool, bt, plan, w, q, out, kept, pos, rows, kv):
        pool.append_norm_rope(0, None, kv[0], kv[1], bt, pos, rot, rows=rows, k_weight=kw)
        pool.decode_tree_weights(plan, 0, q, None, w[0], out, bt, 0.09)
        pool.evict(bt, dev_len, w, budget, recent=20, kept=kept)

    rot, kw = paged.Rotation(d), torch.ones(d, device="cuda").to(dt)
    dev_len = dev([c + new for c in ctx])
    pos = dev(np.concatenate([c + np.arange(new) for c in ctx]))
    rows = dev(np.repeat(np.arange(n), new))
    kv = torch.randn(2, n * new, hkv, d, device="cuda").to(dt)
    q = torch.randn(n * new, h, d, device="cuda").to(dt)
    results = []
    for captured in (False, True):
        pool = make_pool(1, n * 24, ps, hkv, d, dtype, fill=0.0)
        bt = dev(np.random.default_rng(3).permutation(n * 24).reshape(n, 24))
        plan = pool.plan_tree(ctx, [new] * n, h, weights=True)
        w, out = start.clone(), torch.zeros_like(q)
        kept = torch.zeros(1, n, hkv, budget, dtype=torch.int32, device="cuda")
        args = (pool, bt, plan, w, q, out, kept, pos, rows, kv)
        pool.fill_normal(seed=9)
        if captured:
            step(*args)
            g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=s):
                step(*args)
            for _ in range(2):
                pool.fill_normal(seed=9)
                w.copy_(start)
                g.replay()
        else:
            step(*args)
        no_error()
        results.append([x.clone() for x in (w, out, kept, *raw(pool))])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_weights_on_two_streams(dtype):
    """Counted-again and kept scores at once, on plans of their own: the same bits as alone."""
    dt = getattr(torch, dtype)
    pool = make_pool(1, 600, 16, 2, 128, dtype, fill=0.0)
    pool.fill_normal(seed=5)
    bt = dev(np.random.default_rng(0).permutation(600).reshape(3, 200))
    jobs = []
    for nodes in ([90, 40, 70], [1, 1, 1], [3, 1, 5]):
        q = torch.randn(sum(nodes), 8, 128, device="cuda").to(dt)
        plan = pool.plan_tree([3000, 77, 1500], nodes, 8, weights=True)
        w, out = torch.zeros(3, 2, 3200, device="cuda"), torch.zeros_like(q)
        pool.decode_tree_weights(plan, 0, q, None, w, out, bt, 0.09)
        no_error()
        jobs.append((plan, q, w, out, torch.zeros_like(w), torch.zeros_like(out), torch.cuda.Stream()))
    for _ in range(5):
        for plan, q, _, _, w, out, s in jobs:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                w.zero_()
            pool.decode_tree_weights(plan, 0, q, None, w, out, bt, 0.09, stream=s)
    no_error()
    for _, _, w0, out0, w, out, _ in jobs:
        assert torch.equal(w0, w) and torch.equal(out0, out)


# -- offsets that pass 32 bits ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, F32])
def test_pools_past_four_gigabytes(dtype):
    dt = getattr(torch, dtype)
    hkv, d, ps, h, n = 8, 128, 16, 16, 3
    per = hkv * ps * d * dt.itemsize
    pages = (5 << 30) // per
    pool = make_pool(1, pages, ps, hkv, d, dtype, fill=0.0)
    width = 40
    top = np.arange(pages - n * width, pages).reshape(n, width)
    bt = dev(top)
    rows = np.repeat(np.arange(n), 600)
    pos = np.tile(np.arange(600), n)
    kv = torch.randn(2, n * 600, hkv, d, device="cuda").to(dt)
    wk = torch.ones(d, device="cuda").to(dt)
    pool.append_norm_rope(0, None, kv[0], kv[1], bt, dev(pos), None, rows=dev(rows), k_weight=wk)
    no_error()
    for i in range(n):
        k, v = pool.gather(0, bt, i, 0, 600)
        assert torch.equal(v, kv[1][600 * i:600 * (i + 1)])
        x = kv[0][600 * i:600 * (i + 1)].double()
        y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        check(k, y, torch.finfo(dt).eps / 2 * y.abs() * (1 + 2 ** -10) + y.abs() * 2.0 ** -17 + 2.0 ** -25)
    q = torch.randn(n, h, d, device="cuda").to(dt)
    out, w = torch.zeros_like(q), torch.zeros(1, n, hkv, 640, device="cuda")
    pool.decode_tree_weights(pool.plan_tree([599] * n, [1] * n, h, weights=True), 0, q, None, w[0], out, bt, 0.09)
    no_error()
    for i in range(n):
        k, v = pool.gather(0, bt, i, 0, 600)
        ref, tol, _, _ = attend64(q[i:i + 1], k, v, 0.09, dtype)
        check(out[i:i + 1], ref, tol)
    table = bt.clone()
    table[:, :20] = table[0, :20]
    pool.decode_shared(pool.plan_shared([600] * n, [n], [320], h), 0, q, out, table, 0.09)
    no_error()
    for i in range(n):
        k, v = pool.gather(0, table, i, 0, 600)
        ref, tol, _, _ = attend64(q[i:i + 1], k, v, 0.09, dtype)
        check(out[i:i + 1], ref, tol)
    before = [pool.gather(0, bt, i, 0, 600) for i in range(n)]
    ww = w.cpu().numpy()
    kept = pool.evict(bt, dev([600] * n), w, 100, recent=10).cpu().numpy()
    no_error()
    for i in range(n):
        now = pool.gather(0, bt, i, 0, 100)
        for x in range(hkv):
            stay = keep64(ww[0, i, x], 600, 100, 10)
            assert kept[0, i, x].tolist() == stay.tolist()
            s = torch.from_numpy(stay).cuda()
            assert all(torch.equal(a[:, x], b[s, x]) for a, b in zip(now, before[i]))


# -- more of the ranges ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_more_draws(dtype):
    """Sizes as they come."""
    r = np.random.default_rng({F32: 1, F16: 2, BF16: 3}[dtype])
    for k in range(6):
        d = int(r.choice([64, 96, 128, 256]))
        hkv, g = [(1, 7), (2, 6), (4, 8), (8, 1), (5, 3)][int(r.integers(5))]
        ps = int(r.choice([16, 32, 48]))
        n = int(r.integers(1, 6))
        sizes = [int(x) for x in r.integers(1, 9, n)]
        prefix = [int(x) // ps * ps for x in r.integers(0, 900, n)]
        own = [int(x) for x in r.integers(0, 200, sum(sizes))]
        shared_case(dtype, d, hkv * g, hkv, ps, sizes, prefix, own, seed=k)
        ctx, nodes = [int(x) for x in r.integers(0, 900, n)], [int(x) for x in r.integers(0, 20, n)]
        nodes[0] = max(1, nodes[0])
        weigh_case(dtype, d, hkv * g, hkv, ps, ctx, nodes, seed=k, mask=[None, "any"][k % 2])
        weigh_case(dtype, d, hkv * g, hkv, ps, ctx, [min(1, x) for x in nodes], seed=k)
        budget = int(r.integers(1, 500))
        evict_case(dtype, 2, min(d, 128), hkv, ps, [max(1, c) for c in ctx], budget,
                   int(r.integers(0, budget + 1)), seed=k)
        rot = paged.Rotation(d, sections=[d // 2 - 2 * (d // 6), d // 6, d // 6],
                             order=["cyclic", "blocks", "ladders"][k % 3], neox=k % 2 == 0)
        norm_case(dtype, d, hkv * g, hkv, ps, rot, [int(x) for x in r.integers(1, 40, n)], ctx, seed=k)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_odd_slots_and_layer_slices_of_weights(dtype):
    """Weights of one layer need no alignment: (layers, rows, kv_heads, odd slots)."""
    dt = getattr(torch, dtype)
    pool = make_pool(3, 40, 16, 3, 64, dtype, fill=0.0)
    pool.fill_normal(seed=5)
    bt = dev(np.arange(40)[None])
    w = torch.zeros(3, 1, 3, 613, device="cuda")
    for nodes in (1, 11):
        q = torch.randn(nodes, 6, 64, device="cuda").to(dt)
        out = torch.zeros_like(q)
        plan = pool.plan_tree([600], [nodes], 6, weights=True)
        w.zero_()
        for lay in range(3):
            pool.decode_tree_weights(plan, lay, q, None, w[lay], out, bt, 0.1)
        no_error()
        total = w.double().sum(-1)                       # every row's weights add up to one
        assert float((total - 2 * nodes).abs().max()) <= 2 * nodes * 2.0 ** -14
        assert torch.all(w[..., 600 + nodes:] == 0)


@pytest.mark.parametrize("nodes", [1, 20, 45])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_an_infinite_key_has_no_weight(dtype, nodes):
    """A key whose scores are all minus infinity gets the weight zero, and the others what they
    have without it (tokens of 4 q-heads: 4, 80 and 180 rows)."""
    ctx, d, h, hkv, ps, at = 300, 64, 8, 2, 16, 5
    n = ctx + nodes
    g = torch.Generator(device="cuda")
    g.manual_seed(nodes)
    dt = getattr(torch, dtype)
    bt, total = tables([-(-n // ps)], 1)
    pool = make_pool(1, total, ps, hkv, d, dtype)
    k, v = (torch.randn(n, hkv, d, generator=g, device="cuda").to(dt) for _ in range(2))
    q = torch.randn(nodes, h, d, generator=g, device="cuda").to(dt)
    q[:, :, 0] = 1.0
    vis = torch.ones(nodes, n, dtype=torch.bool, device="cuda").tril(ctx)
    vis[:, at] = False
    ref, tol, wt, rel = attend64(q, k, v, 1.0 / math.sqrt(d), dtype, vis)
    want = wt.view(nodes, hkv, -1, n).sum((0, 2))
    wtol = (wt * rel).view(nodes, hkv, -1, n).sum((0, 2)) + \
        (nodes * h // hkv + 4) * 2.0 ** -24 * want + 1e-30
    k[at, :, 0] = -math.inf
    pool.append(0, k, v, bt, torch.arange(n, dtype=torch.int32, device="cuda"),
                torch.zeros(n, dtype=torch.int32, device="cuda"))
    weights = torch.zeros(1, hkv, n, device="cuda")
    out = torch.zeros_like(q)
    pool.decode_tree_weights(pool.plan_tree([ctx], [nodes], h, weights=True), 0, q, None, weights, out, bt,
                             1.0 / math.sqrt(d))
    no_error()
    assert torch.all(weights[0, :, at] == 0.0)
    check(weights[0], want, wtol)
    check(out, ref, tol)


# -- refusals ---------------------------------------------------------------------------------------------
def test_refusals():
    pool = make_pool(2, 8, 16, 2, 64, F16, fill=0.0)
    before = [x.clone() for x in raw(pool)]
    z = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    k, bt, pos, q = z(3, 2, 64), dev([[0, 1], [2, 3]]), dev([0, 1, 2]), z(3, 4, 64)
    rot, w = paged.Rotation(64), z(64)
    norm = lambda **kw: pool.append_norm_rope(**{**dict(  # noqa: E731
        layer=0, q=q, k_new=k, v_new=k, block_tables=bt, positions=pos, rotation=rot), **kw})
    for kw, err in ((dict(layer=2), "layer"), (dict(layer=-1), "layer"),):
        with pytest.raises(IndexError, match=err):
            norm(**kw)
    wide, three = z(3, 6, 64), paged.Rotation(64, sections=[10, 11, 11])
    for kw in (dict(k_new=k.float()), dict(v_new=k[:, :1]), dict(q=q[:2]), dict(q=q[0]),
               dict(q_weight=w[:32]), dict(q_weight=w.float()), dict(k_weight=w[None]),
               dict(q_weight=w, eps=0.0), dict(k_weight=w, eps=-1.0), dict(k_weight=w, eps=math.nan),
               dict(rotation=paged.Rotation(66)), dict(rotation=three, rope_positions=pos),
               dict(rotation=three, rope_positions=dev(np.zeros((3, 2)))),
               dict(rope_positions=dev(np.zeros((3, 3)))), dict(rope_positions=pos.long()),
               dict(q_out=z(3, 3, 64)), dict(positions=pos.long()), dict(rows=dev([0, 1])),
               dict(q_weight=z(65)[1:]), dict(k_new=z(3 * 128 + 1)[1:].view(3, 2, 64)),
               dict(k_new=z(3, 129)[:, :128].unflatten(1, (2, 64))),
               dict(q=wide[:, :4], q_out=wide.view(-1)[:3 * 4 * 64])):
        with pytest.raises(ValueError):
            norm(**kw)
    for axes, pairs, freq, axis in ((5, 1, [1.0], None), (0, 1, [1.0], None), (1, 33, [1.0] * 33, None),
                                    (1, -1, [1.0], None), (2, 1, [1.0], [2]), (1, 1, [math.inf], None),
                                    (1, 1, None, None)):
        f = None if freq is None else np.array(freq)
        x = None if axis is None else np.array(axis, dtype=np.uint8)
        args = ffi.NORM_ROPE_ARGS.pack(
            0, 0, 0, k.data_ptr(), 0, k.data_ptr(), bt.data_ptr(), 0, pos.data_ptr(), 0,
            ffi.np_ptr(f) or 0, ffi.np_ptr(x) or 0, 0, 0, 0, 0, 0, 2, 2, 3, axes, pairs, 1, 1e-6)
        assert ffi.lib.kvc_append_norm_rope(pool.handle, args, None) == ffi.KVC_ERR_INVALID_ARG
    assert ffi.lib.kvc_append_norm_rope(pool.handle, None, None) == ffi.KVC_ERR_INVALID_ARG
    with pytest.raises(ValueError, match="32 bits"):
        norm(layer=1 << 40)

    for bad in (([20, 20], [2], [8]), ([20, 20], [2], [32]), ([20, 20], [1], [16]), ([20], [1, 1], [0, 0]),
                ([20], [0], [0]), ([20], [1], [-16]), ([-1], [1], [0]), ([20], [-1], [0])):
        with pytest.raises(ValueError):
            pool.plan_shared(*bad, 4)
    for heads in (3, 0, -2):
        with pytest.raises(ValueError):
            pool.plan_shared([20], [1], [0], heads)
    with pytest.raises(ValueError):
        pool.plan_shared([20], [1], [0], 4, rows=[-1])
    plan = pool.plan_shared([20, 30, 17], [3], [16], 4, rows=[0, 1, 0])
    out = torch.empty_like(q)
    with pytest.raises(IndexError, match="layer"):
        pool.decode_shared(plan, 2, q, out, bt, 0.1)
    with pytest.raises(IndexError, match="width"):
        pool.decode_shared(plan, 0, q, out, bt[:, :1].contiguous(), 0.1)
    with pytest.raises(IndexError, match="row"):
        pool.decode_shared(plan, 0, q, out, bt[:1], 0.1)
    for args in ((q[:2], out, bt, 0.1), (q, out[:2], bt, 0.1), (q.float(), out, bt, 0.1),
                 (q, out, bt, math.inf), (q, out, bt.long(), 0.1), (q, out, bt[0], 0.1)):
        with pytest.raises(ValueError):
            pool.decode_shared(plan, 0, *args)
    other = make_pool(1, 8, 16, 1, 64, F16, fill=0.0)
    with pytest.raises(ValueError, match="geometry"):
        other.decode_shared(plan, 0, q, out, bt, 0.1)
    with pytest.raises(ValueError, match="built"):
        fresh = paged.SharedPlan()
        ffi.check(ffi.lib.kvc_decode_shared(pool.handle, fresh.handle, 0, q.data_ptr(), out.data_ptr(),
                                            bt.data_ptr(), 2, 0.1, None))

    sums = z(2, 2, 40, t=torch.float32)
    tree = pool.plan_tree([10, 12], [2, 1], 4, weights=True)
    weigh = lambda p, *a: pool.decode_tree_weights(p, 0, q, None, *a)  # noqa: E731
    with pytest.raises(ValueError, match="set_weights"):
        weigh(pool.plan_tree([10, 12], [2, 1], 4), sums, out, bt, 0.1)
    with pytest.raises(IndexError, match="slots"):
        weigh(tree, sums[..., :11].contiguous(), out, bt, 0.1)
    with pytest.raises(IndexError, match="row"):
        weigh(tree, sums[:1], out, bt, 0.1)
    for bad in (sums.double(), sums[:, :1].contiguous(), sums[0], sums.transpose(0, 1)[..., ::2]):
        with pytest.raises(ValueError):
            weigh(tree, bad, out, bt, 0.1)
    with pytest.raises(ValueError, match="row"):
        pool.plan_tree([10, 12], [2, 1], 4, rows=[1, 1], weights=True)
    pool.plan_tree([10, 12], [2, 0], 4, rows=[1, 1], weights=True)     # (one of them has no token)
    pool.plan_tree([10, 12], [2, 1], 4, rows=[1, 1])
    with pytest.raises(ValueError, match="scores"):
        pool.plan_tree([1 << 27], [8], 4, weights=True)
    assert torch.all(sums == 0)

    heavy, lens = z(2, 2, 2, 40, t=torch.float32), dev([20, 20])
    for kw in (dict(budget=0), dict(budget=-1), dict(budget=4, recent=5), dict(budget=4, recent=-1),
               dict(weights=heavy[:1]), dict(weights=heavy[:, :, :1]), dict(weights=heavy[0]),
               dict(weights=heavy.double()), dict(weights_out=heavy[..., :39].contiguous()),
               dict(kept=z(2, 2, 2, 5, t=torch.int32)), dict(kept=z(2, 2, 2, 4, t=torch.int64)),
               dict(ctx_lens=lens.long()), dict(rows=dev([0])), dict(block_tables=bt[0])):
        with pytest.raises(ValueError):
            pool.evict(**{**dict(block_tables=bt, ctx_lens=lens, weights=heavy, budget=4), **kw})
    with pytest.raises(IndexError):
        pool.evict(bt, dev([20, 20, 20]), heavy, 4)
    no_error()
    assert all(torch.equal(a, b) for a, b in zip(raw(pool), before))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_empty_calls(dtype):
    pool = make_pool(1, 8, 16, 2, 64, dtype, fill=0.0)
    z = lambda *s, t=getattr(torch, dtype): torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    bt, none = dev([[0, 1], [2, 3]]), dev([])
    assert pool.append_norm_rope(0, z(0, 4, 64), z(0, 2, 64), z(0, 2, 64), bt, none,
                                 paged.Rotation(64)).shape == (0, 4, 64)
    pool.decode_shared(pool.plan_shared([], [], [], 4), 0, z(0, 4, 64), z(0, 4, 64), bt, 0.1)
    w = z(1, 2, 2, 32, t=torch.float32)
    pool.decode_tree_weights(pool.plan_tree([5], [0], 4, weights=True), 0, z(0, 4, 64), None, w[0],
                             z(0, 4, 64), bt, 0.1)
    assert pool.evict(bt, none, w, 4).shape == (1, 0, 2, 4)
    out = torch.ones(2, 4, 64, device="cuda").to(getattr(torch, dtype))
    pool.decode_shared(pool.plan_shared([0, 0], [2], [0], 4), 0, out, out2 := torch.ones_like(out), bt, 0.1)
    no_error()
    assert torch.all(out2 == 0)
