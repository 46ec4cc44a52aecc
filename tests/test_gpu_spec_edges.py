"""Drafted-token and beam operators where they can go wrong: flat tails far below a peak,
the kernels' variants for large batches, side streams, plans of other pools, scores that
nearly tie.  Bounds are derived from the arithmetic as in tests/test_gpu_spec_ops.py."""

from __future__ import annotations

import math

import numpy as np
import pytest

from conftest import HAS_GPU
from test_gpu_spec_generate import gen  # noqa: F401  (a fixture)
from test_gpu_spec_ops import BF16, F16, F32, dev, no_error, raw

pytestmark = pytest.mark.gpu

if HAS_GPU:
    import torch

    import batch_generate as BG
    import beam
    import kvcache_ffi as ffi
    import paged
    from test_gpu_batch_generate import _model


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


# -- another stream than the current one ----------------------------------------------------------
def _litter():
    """Small tensors of every size on the current stream, full of what no call can use."""
    for n in (1, 3, 8, 64, 200, 1024, 4096, 1 << 16):
        for _ in range(4):
            torch.full((n,), 0x7E7E7E7E, dtype=torch.int32, device="cuda")


def _run(gen, stream, busy):
    bt = gen.bt[:3].clone()
    dec = gen._decoder(bt)
    x = lambda ids: gen.model.embedding[torch.tensor(ids, device="cuda")].contiguous()  # noqa: E731
    prompt, drafts = x([3, 14, 15, 9, 2, 6, 5]), x([5, 9, 11, 3, 60, 7, 8, 2, 4])
    nxt = x([1, 2, 3])
    outs = []
    torch.cuda.synchronize()
    if busy:
        with torch.cuda.stream(stream):
            torch.cuda._sleep(100_000_000)        # some 50 ms, so that all below waits its turn
    for i in range(3):
        outs.append(dec.prefill(i, prompt, stream=stream))
        _litter()
    outs.append(dec.verify(drafts, [[-1, 0, 0]] * 3, stream=stream))
    _litter()
    dec.commit([[0, 2], [0, 1], [0, 2]], stream=stream)
    _litter()
    dec.reorder([[2, 0, 0]], stream=stream)
    _litter()
    outs.append(dec.step(nxt, stream=stream))
    _litter()
    outs += [t for r in range(3) for t in gen.pool.gather(1, bt, r, 0, 10, stream=stream)]
    _litter()
    torch.cuda.synchronize()
    dec.close()
    return outs, bt


def test_decoder_on_a_busy_side_stream(gen):  # noqa: F811
    want, table = _run(gen, None, False)
    for _ in range(3):
        got, bt = _run(gen, torch.cuda.Stream(), True)
        assert torch.equal(table, bt)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    no_error()


def test_outputs_made_for_a_side_stream_are_its_own():
    """The current stream still has writes under way to memory that it has freed."""
    pool = paged.PagedKVCache(1, 8, 16, 2, 64)
    bt, pos = dev([[0, 1, 2, 3]]), dev(np.arange(40))
    k = torch.randn(40, 2, 64, device="cuda").half()
    q = torch.randn(40, 4, 64, device="cuda").half()
    logits, scores = torch.randn(4, 5000, device="cuda"), torch.zeros(1, 4, device="cuda")
    sel = beam.BeamSelector(1, 4, 5000, 8)
    want = [pool.append_rope(0, q, k, k, bt, pos), *sel.select(logits, scores, 8)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    shapes = [(t.shape, t.dtype) for t in want]
    torch.cuda._sleep(100_000_000)
    late = [torch.full(s, 9, dtype=d, device="cuda") for s, d in shapes]
    del late
    got = [pool.append_rope(0, q, k, k, bt, pos, stream=side), *sel.select(logits, scores, 8, stream=side)]
    no_error()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


# -- pieces of every kind after one another on one CTA ---------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tree_restores_values_in_every_piece_of_a_cta(dtype):
    """Wide trees (two groups of rows) and single tokens (one tile) in turn, several pieces a
    CTA, each with drafted V that are not finite: they reach the rows that see them, and the
    rest is what it is with zeros in their place."""
    dt = getattr(torch, dtype)
    seqs, d, h, ps, cols = 1200, 64, 4, 16, 8
    rng = np.random.default_rng(5)
    ctx = rng.integers(0, 60, seqs)
    nodes = np.where(np.arange(seqs) % 2 == 0, 60, 1 + np.arange(seqs) % 5)
    pool = paged.PagedKVCache(1, seqs * cols, ps, 1, d, dtype=dt)
    pool.fill_normal(seed=2)
    bt = dev(rng.permutation(seqs * cols).reshape(seqs, cols))
    total = int(nodes.sum())
    rows = dev(np.repeat(np.arange(seqs), nodes))
    first = np.concatenate([[0], np.cumsum(nodes)[:-1]])
    node = np.arange(total) - np.repeat(first, nodes)
    slots = dev(np.repeat(ctx, nodes) + node)
    k = torch.randn(total, 1, d, device="cuda").to(dt)
    clean = torch.randn(total, 1, d, device="cuda").to(dt)
    hurt = torch.from_numpy(first + rng.integers(0, nodes)).cuda()      # one node of each sequence
    clean[hurt, 0, 7] = 0.0
    odd = clean.clone()
    odd[hurt, 0, 7] = math.inf
    q = torch.randn(total, h, d, device="cuda").to(dt)
    plan = pool.plan_tree(ctx, nodes, h)
    assert plan.info().n_items * 4 <= seqs
    out = []
    for v in (clean, odd):
        pool.append(0, k, v, bt, slots, rows)
        o = torch.zeros_like(q)
        pool.decode_tree(plan, 0, q, None, o, bt, 0.1)
        no_error()
        out.append(o)
    want = out[0].clone()
    at = np.repeat((hurt.cpu().numpy() - first), nodes)
    want[torch.from_numpy(node >= at).cuda(), :, 7] = math.inf
    assert torch.equal(out[1], want)


# -- rotate + append: the variant for many tokens ---------------------------------------------------
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("dtype,d,hkv,h,ps", [
    (F32, 64, 2, 6, 16), (F16, 128, 8, 32, 16), (BF16, 96, 3, 7, 48), (F16, 40, 2, 4, 16),
    (BF16, 256, 1, 3, 32), (F32, 256, 2, 2, 16), (F16, 8, 3, 5, 16), (F32, 12, 1, 2, 16)])
def test_append_rope_of_many_tokens(dtype, d, hkv, h, ps, neox):
    """From 592 tokens on four of them share a CTA; the last CTA has one, two or three."""
    dt = getattr(torch, dtype)
    half = torch.finfo(dt).eps / 2
    slack = 2.0 ** -22 + 3 * 2.0 ** -24 + 2.0 ** -23
    rng = np.random.default_rng(d + h)
    for counts, ctx in (([400, 1, 260], [5, ps - 1, 100000]), ([592], [0]), ([3, 700, 11], [7, 0, 64]),
                        ([1201], [33])):
        n = sum(counts)
        need = [-(-(c + k) // ps) for c, k in zip(ctx, counts)]
        bt = np.zeros((len(ctx), max(need)), dtype=np.int32)
        pages = sum(b - c // ps for b, c in zip(need, ctx))
        perm = iter(rng.permutation(pages))
        for i, c in enumerate(ctx):
            for p in range(c // ps, need[i]):
                bt[i, p] = next(perm)
        pool = paged.PagedKVCache(1, pages, ps, hkv, d, dtype=dt)
        pos = np.concatenate([c + np.arange(k) for c, k in zip(ctx, counts)])
        rows = np.repeat(np.arange(len(ctx)), counts)
        pad = np.unique(np.concatenate([rng.integers(0, n, 9), [n - 1]]))
        slots = pos.copy()
        slots[pad] = -1
        g = torch.Generator(device="cuda")
        g.manual_seed(n)
        qkv = torch.randn(n, h + 2 * hkv, d, generator=g, device="cuda").to(dt)
        q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
        ang = pos + rng.integers(-3, 4, n)
        args = lambda a, b: dict(rows=dev(rows[a:b]), rope_positions=dev(ang[a:b]),  # noqa: E731
                                 freq_base=500000.0, neox=neox)
        for m in raw(pool):
            m.fill_(3.0)
        q_out = torch.full((n, h, d), 5.0, dtype=dt, device="cuda")
        pool.append_rope(0, q, k, v, dev(bt), dev(slots), q_out=q_out, **args(0, n))
        no_error()
        freq = 500000.0 ** (-2.0 * np.arange(d // 2) / d)
        th = torch.from_numpy(ang[:, None].astype(np.float64) * freq).cuda()[:, None]

        def rot(x):
            x = x.double()
            a, b = (x[..., :d // 2], x[..., d // 2:]) if neox else (x[..., 0::2], x[..., 1::2])
            y = [a * th.cos() - b * th.sin(), a * th.sin() + b * th.cos()]
            t = [a.abs() + b.abs()] * 2
            if neox:
                return torch.cat(y, -1), torch.cat(t, -1)
            return torch.stack(y, -1).flatten(-2), torch.stack(t, -1).flatten(-2)

        live = np.setdiff1d(np.arange(n), pad)
        kk, vv = torch.empty_like(k), torch.empty_like(v)
        o = 0
        for i, (c, m) in enumerate(zip(ctx, counts)):
            gk, gv = pool.gather(0, dev(bt), i, c, m)
            kk[o:o + m], vv[o:o + m] = gk, gv
            o += m
        for got, src in ((q_out, q), (kk, k)):
            ref, mag = rot(src)
            tol = half * ref.abs() + slack * mag + (2.0 ** -25 if dtype == F16 else 0)
            assert torch.all((got.double() - ref).abs()[live] <= tol[live])
        assert torch.equal(vv[live], v[live])
        assert torch.all(q_out[pad] == 5.0) and torch.all(kk[pad] == 3.0) and torch.all(vv[pad] == 3.0)
        for m in raw(pool):   # nothing else is written
            assert int((m != 3.0).sum()) <= len(live) * hkv * d
        # few tokens at a time, a CTA each: the same bits
        whole = [m.clone() for m in raw(pool)]
        again = torch.full_like(q_out, 5.0)
        for m in raw(pool):
            m.fill_(3.0)
        for a in range(0, n, 400):
            b = min(n, a + 400)
            pool.append_rope(0, q[a:b], k[a:b], v[a:b], dev(bt), dev(slots[a:b]), q_out=again[a:b],
                             **args(a, b))
        no_error()
        assert torch.equal(again, q_out) and all(torch.equal(a, b) for a, b in zip(whole, raw(pool)))
        pool.close()


# -- selection: many rows over a large vocabulary ---------------------------------------------------
def _select_ref(logits, scores, n_out):
    """Tokens, parents and scores in 64 bits, on the GPU; lower candidates win ties."""
    n, b = scores.shape
    x = logits.double()
    fin = torch.isfinite(x)
    x = torch.where(fin, x, -math.inf)
    top = x.amax(1, keepdim=True)
    some = torch.isfinite(top)
    lse = torch.where(some, top + (x - torch.where(some, top, 0.0)).exp().sum(1, keepdim=True).log(), 0.0)
    cum = scores.double().view(-1, 1)
    s = torch.where(fin & torch.isfinite(cum), cum + (x - lse), -math.inf).view(n, -1)
    best, at = torch.sort(s, dim=1, descending=True, stable=True)
    v = logits.shape[1]
    return at[:, :n_out] % v, at[:, :n_out] // v, best[:, :n_out]


def _check_select(logits, scores, n_out):
    n, b = scores.shape
    sel = beam.BeamSelector(n, b, logits.shape[1], n_out)
    tok, par, best = sel.select(logits, scores, n_out)
    no_error()
    rt, rp, rs = _select_ref(logits, scores, n_out)
    assert torch.equal(par.long(), rp) and torch.equal(tok.long(), rt)
    fin = torch.isfinite(rs)
    assert torch.equal(fin, torch.isfinite(best)) and torch.all(best[~fin] == -math.inf)
    assert torch.all((best.double() - rs).abs()[fin] <= (2.0 ** -17 + 2.0 ** -24 * rs.abs())[fin])
    sel.close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,b,v,k", [(12, 8, 65537, 8), (24, 4, 120000, 32), (24, 8, 100003, 16),
                                     (16, 16, 77777, 32)])
def test_beam_select_many_rows(n, b, v, k, dtype):
    """2, 4, 8 and 8 batches of 512 logits a warp: the running max and sum go over several."""
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(v)
    logits = (3 * torch.randn(n * b, v, generator=g, device="cuda")).to(dt)
    scores = -5 * torch.rand(n, b, generator=g, device="cuda")
    _check_select(logits, scores, k)
    wide = torch.full((n * b, v + 13), math.inf, dtype=dt, device="cuda")    # rows on every alignment
    wide[:, 5:5 + v] = logits
    _check_select(wide[:, 5:5 + v], scores, k)
    # a max that grows with every batch, one that falls, masks, values that are not finite
    ramp = torch.linspace(-20, 20, v, device="cuda")
    logits[0::5] = (logits[0::5].float() + ramp).to(dt)
    logits[1::5] = (logits[1::5].float() - ramp).to(dt)
    logits[2, :v - 3] = -math.inf
    logits[3, 100:] = -math.inf
    logits[4] = -math.inf
    logits[7, ::3] = math.nan
    logits[8, 1::2] = math.inf
    logits[9] = torch.finfo(dt).min
    logits[9, v // 2] = 0.0
    _check_select(logits, scores, k)
    scores[:, 1:] = -math.inf
    scores[1, 0], scores[2, 0] = math.nan, -math.inf
    _check_select(logits, scores, k)
    same = torch.zeros(n * b, v, dtype=dt, device="cuda")      # every candidate ties
    _check_select(same, torch.zeros(n, b, device="cuda"), k)
    peak = same.clone()
    peak[:, 4090:4100] = 7.0                                   # across two warps' runs
    _check_select(peak, torch.zeros(n, b, device="cuda"), k)


# -- commit: contexts that no table holds -------------------------------------------------------------
@pytest.mark.parametrize("ctx", [2 ** 31 - 1, 2 ** 31 - 257, 2 ** 31 - 256, 2 ** 30, -1, -2 ** 31])
def test_commit_reports_contexts_past_every_table(ctx):
    pool = paged.PagedKVCache(1, 4, 16, 1, 64)
    pool.fill_normal(seed=1)
    before = [m.clone() for m in raw(pool)]
    bt = dev([[0, 1], [2, 3]])
    pool.commit_tree(bt, dev([ctx, 3]), dev([[1, 200], [0, 0]]), dev([2, 0]))
    torch.cuda.synchronize()
    assert ffi.device_error(0)[0] == 3
    assert all(torch.equal(a, b) for a, b in zip(before, raw(pool)))


# -- selection: candidates of different beams that nearly tie -------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("v", [700, 32000, 128256])
def test_beam_select_keeps_the_order_of_near_ties(dtype, v):
    """Beams are 2^-16 and more apart, up and down in turn (each is within 2^-17 of its score)."""
    n = 100
    g = torch.Generator(device="cuda")
    g.manual_seed(v)
    x = torch.randn(2 * n, v, generator=g, device="cuda")
    x *= torch.linspace(0.1, 4.0, n, device="cuda").repeat_interleave(2)[:, None]     # flat to peaked
    x[:, 5] = x.amax(1) + 1.0 + torch.rand(2 * n, generator=g, device="cuda")
    logits = x.to(getattr(torch, dtype))
    logp = torch.log_softmax(logits.double(), 1).amax(1).view(n, 2)
    gap = 2.0 ** -16 * (1 + torch.arange(n, device="cuda") % 3) * (1 - 2 * (torch.arange(n, device="cuda") % 2))
    cum = torch.zeros(n, 2, device="cuda")
    cum[:, 1] = (logp[:, 0] - logp[:, 1] + gap).float()
    apart = cum[:, 1].double() + logp[:, 1] - logp[:, 0]
    wide = apart.abs() >= 2.0 ** -16          # (what the scores' own fp32 leaves of the gap)
    assert int(wide.sum()) >= n // 3
    tok, par, _ = beam.BeamSelector(n, 2, v, 2).select(logits, cum, 2)
    no_error()
    assert torch.all(tok == 5)
    assert torch.equal(par[wide, 0].long(), (apart > 0).long()[wide])
    assert torch.equal(par[:, 0] + par[:, 1], torch.ones_like(par[:, 0]))


# -- beam search against a search of its own over the same logits ---------------------------------------
def _search(steps, k, most, penalty, eos):
    """Beam search of one prompt: steps[t] are the (k, vocab) logits of the beams after t tokens."""
    beams, ended = [(0.0, [])], []
    for t in range(most):
        logp = torch.log_softmax(steps[t].double(), 1).cpu().numpy()
        found = sorted(((s + logp[b, w], -b, -w) for b, (s, _) in enumerate(beams)
                        for w in range(logp.shape[1])), reverse=True)[:2 * k]
        kept = []
        for rank, (s, b, w) in enumerate(found):
            ids = beams[-b][1] + [-w]
            if -w == eos:
                if rank < k:
                    ended.append((s / len(ids) ** penalty, ids))
            elif len(kept) < k:
                kept.append((s, ids))
        beams = kept
        if len(ended) >= k:
            break
    else:
        ended += [(s / len(ids) ** penalty, ids) for s, ids in beams]
    return max(ended, key=lambda e: e[0])


@pytest.mark.parametrize("k,penalty,eos_at", [(2, 1.0, None), (3, 0.0, None), (4, 1.0, 1), (4, 2.0, 0),
                                              (3, -0.5, 3), (2, 0.7, 2)])
def test_beam_search_against_a_search_over_the_same_logits(gen, monkeypatch, k, penalty, eos_at):  # noqa: F811
    prompts = [[3, 14, 15, 9, 2, 6, 5], [1] * 17]
    cfg = gen.model.cfg
    old = cfg.eos_token_id
    if eos_at is not None:
        plain, _ = gen.generate_beam_ids(prompts, num_beams=k, max_new_tokens=6, stop_on_eos=False)
        cfg.eos_token_id = plain[0][eos_at]
    seen, real = [], gen._logits

    def logits(h, stream):
        out = real(h, stream)
        seen.append(out.view(len(prompts), k, -1).clone())
        return out
    monkeypatch.setattr(gen, "_logits", logits)
    try:
        ids, scores = gen.generate_beam_ids(prompts, num_beams=k, max_new_tokens=12,
                                            length_penalty=penalty, stop_on_eos=eos_at is not None)
    finally:
        eos, cfg.eos_token_id = cfg.eos_token_id, old
    for i in range(len(prompts)):
        score, want = _search([s[i] for s in seen], k, 12, penalty, eos if eos_at is not None else -1)
        assert ids[i] == want
        # 12 selections, each within 2^-17 and one rounding of a sum below 64
        n = len(want) ** penalty
        assert abs(scores[i] - score) <= 12 * (2.0 ** -17 + 2.0 ** -18) / n + 2.0 ** -40


# -- plans and captures ---------------------------------------------------------------------------------
def test_a_tree_plan_is_not_built_inside_a_capture():
    """An upload from the plan's staging buffer, replayed, would bring what a later build left
    there.  The call is refused, and the capture around it goes on."""
    pool = paged.PagedKVCache(1, 16, 16, 2, 64)
    pool.fill_normal(seed=4)
    bt = dev(np.arange(16).reshape(2, 8))
    q = torch.randn(12, 8, 64, device="cuda").half()
    plan = pool.plan_tree([50, 9], [5, 7], 8)
    want, got = torch.zeros_like(q), torch.zeros_like(q)
    pool.decode_tree(plan, 0, q, None, want, bt, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for p in (plan, None):
            with pytest.raises(ValueError, match="captured"):
                pool.plan_tree([3, 4], [2, 2], 8, plan=p)
        pool.decode_tree(plan, 0, q, None, got, bt, 0.1)
    graph.replay()
    no_error()
    assert plan.n_tokens == 12 and torch.equal(want, got)
    pool.plan_tree([50, 9], [5, 7], 8, plan=plan)      # and builds again outside
    pool.decode_tree(plan, 0, q, None, got.zero_(), bt, 0.1)
    no_error()
    assert torch.equal(want, got)


# -- drafts ---------------------------------------------------------------------------------------------
def test_drafts_with_missing_parents_are_refused(gen):  # noqa: F811
    """Also where the missing ones lie behind what there is room for."""
    prompts = [[3, 14, 15, 9, 2, 6, 5]]
    for draft in (([1, 2, 3, 4], [-1, 0, 1]), ([1, 2, 3, 4, 5, 6], [-1, 0, 1, 2]), ([1], []), ([], [-1])):
        with pytest.raises(ValueError, match="parent"):
            gen.generate_speculative_ids(prompts, lambda i, ids: draft, max_new_tokens=4,
                                         stop_on_eos=False)
    for draft in (([64], [-1]), ([-1], [-1])):
        with pytest.raises(ValueError, match="vocabulary"):
            gen.generate_speculative_ids(prompts, lambda i, ids: draft, max_new_tokens=4,
                                         stop_on_eos=False)
    want, _ = gen.generate_batch_ids(prompts, max_new_tokens=4, stop_on_eos=False)
    got, _ = gen.generate_speculative_ids(prompts, lambda i, ids: ([1] * 90, [-1] * 90), max_new_tokens=4,
                                          stop_on_eos=False)
    assert got == want


# -- a negative scale ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,nodes", [(64, 3), (128, 60), (256, 33), (80, 20)])
def test_tree_with_a_negative_scale_is_the_tree_of_negated_queries(dtype, d, nodes):
    """Bit for bit, in every piece of a CTA: q changes sign where it is copied, and again and
    again for new queries in the same place."""
    dt = getattr(torch, dtype)
    seqs, ctx, cols = 300, 40, 8
    pool = paged.PagedKVCache(1, seqs * cols, 16, 1, d, dtype=dt)
    pool.fill_normal(seed=6)
    bt = dev(np.random.default_rng(d).permutation(seqs * cols).reshape(seqs, cols))
    plan = pool.plan_tree([ctx] * seqs, [nodes] * seqs, 4)
    for k in range(3):
        q = torch.randn(seqs * nodes, 4, d, device="cuda").to(dt)
        a, b = torch.zeros_like(q), torch.zeros_like(q)
        pool.decode_tree(plan, 0, q, None, a, bt, -0.1)
        pool.decode_tree(plan, 0, -q, None, b, bt, 0.1)
        no_error()
        assert torch.equal(a, b)


# -- scores whose rounding outweighs every difference -------------------------------------------------------
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("size", [100.0, 700.0, 1100.0, 1500.0, 2000.0, 2600.0])
def test_tree_with_huge_scores_stays_a_weighted_mean(dtype, size):
    """Scores of 1e5 to 8e7, all nearly equal: whatever the weights, equal values come out as
    they are, up to the probabilities' rounding (h relative each) and the output's.  The max
    creeps up along the context, several tiles a piece."""
    dt = getattr(torch, dtype)
    seqs, hkv, d, ctx, n = 40, 8, 128, 700, 2
    cols = -(-(ctx + n) // 16)
    pool = paged.PagedKVCache(1, seqs * cols, 16, hkv, d, dtype=dt)
    bt = dev(np.arange(seqs * cols).reshape(seqs, cols))
    g = torch.Generator(device="cuda")
    g.manual_seed(int(size))
    pos = torch.arange(ctx + n, dtype=torch.int32, device="cuda")
    v = torch.full((ctx + n, hkv, d), 3.0, dtype=dt, device="cuda")
    creep = torch.linspace(1.0, 1.0 + 2.0 ** -7, ctx + n, device="cuda")[:, None, None]
    for i in range(seqs):
        k = size * creep * (1 + 2.0 ** -10 * torch.randn(ctx + n, hkv, d, generator=g, device="cuda"))
        pool.append(0, k.to(dt), v, bt, pos, torch.full_like(pos, i))
    q = torch.full((seqs * n, hkv, d), size, device="cuda").to(dt)
    out = torch.zeros_like(q)
    pool.decode_tree(pool.plan_tree([ctx] * seqs, [n] * seqs, hkv), 0, q, None, out, bt, 0.088)
    no_error()
    half = torch.finfo(dt).eps / 2
    assert float((out.double() - 3.0).abs().max()) <= 3.0 * (2 * half + 2.0 ** -14)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tree_with_huge_scores_that_grow_by_less_than_a_rescaling(dtype):
    """Scores of 6e7 (a step of fp32 is worth 2^4), the later half 2^7.9 above the first: O is
    not rescaled for that, and the probabilities must still fit their type."""
    dt = getattr(torch, dtype)
    seqs, hkv, d, ctx, n = 40, 8, 128, 700, 2
    cols = -(-(ctx + n) // 16)
    pool = paged.PagedKVCache(1, seqs * cols, 16, hkv, d, dtype=dt)
    bt = dev(np.arange(seqs * cols).reshape(seqs, cols))
    pos = torch.arange(ctx + n, dtype=torch.int32, device="cuda")
    v = torch.full((ctx + n, hkv, d), 3.0, dtype=dt, device="cuda")
    for i in range(seqs):
        k = torch.full((ctx + n, hkv, d), 2000.0 - 8 * i, device="cuda")
        k[:, :, 0] = 0.0
        k[256:, :, 0] = 64.0
        pool.append(0, k.to(dt), v, bt, pos, torch.full_like(pos, i))
    q = torch.full((seqs * n, hkv, d), 1.0, device="cuda")
    q[:, :, 1:] = (1960.0 + 8 * torch.arange(hkv, device="cuda"))[:, None]
    q = q.to(dt)
    out = torch.zeros_like(q)
    pool.decode_tree(pool.plan_tree([ctx] * seqs, [n] * seqs, hkv), 0, q, None, out, bt, 0.0856)
    no_error()
    half = torch.finfo(dt).eps / 2
    assert float((out.double() - 3.0).abs().max()) <= 3.0 * (2 * half + 2.0 ** -14)
