"""Performance cases of the drafted-token and beam operators of the paged KV pool.

Five operators work on the pool together.  A step that verifies drafted tokens
rotates and appends their rows (``append``), attends over the cache and the
drafted tokens' own tree (``tree``) and, once the accepted path is known, moves
its rows together (``commit``).  A step of beam search picks the best
continuations over beams and vocabulary (``select``) and lets the beams' cached
states follow their parents (``reorder``).

``own`` False computes each operator in its plain form, elementary torch
operations in 32 or 64 bits on the same buffers; ``own`` True makes the library
calls.  Pools keep the library's layout in both forms: 16-bit storage holds, for
each page and KV head, 8-position x 16-byte blocks (positions / 8, head_dim / 8,
8 positions, 8 dims), fp32 storage plain rows.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "gfx1150-inference_b200")


# -- cases --------------------------------------------------------------------------------
def listed():
    return [
        # one short sequence, a handful of drafted tokens: the step's latency
        dict(name="append 5 tokens fp32", op="append", dtype="fp32", seqs=1, new_min=5, new_max=5,
             ctx_min=511, ctx_max=511, heads=32, kv_heads=4, dim=64, page=16, neox=False,
             base=10000.0, fused=False, lens=1),
        # the ragged prompts of a batch going in at once, rows cut from a fused QKV product
        dict(name="append 32 prompts bf16", op="append", dtype="bf16", seqs=32, new_min=70,
             new_max=431, ctx_min=0, ctx_max=8000, heads=32, kv_heads=8, dim=128, page=16,
             neox=True, base=500000.0, fused=True, lens=2),
        # a short chain of guesses for one sequence of a small model: latency again
        dict(name="tree 1x4 at 511 fp32", op="tree", dtype="fp32", seqs=1, nodes_min=4,
             nodes_max=4, ctx_min=511, ctx_max=511, heads=32, kv_heads=4, dim=64, page=16, lens=3),
        # an ordinary serving batch with small ragged trees, grouped heads
        dict(name="tree 32x(5..16) ragged fp16", op="tree", dtype="fp16", seqs=32, nodes_min=5,
             nodes_max=16, ctx_min=1024, ctx_max=8192, heads=32, kv_heads=8, dim=128, page=16,
             lens=4),
        # few long sequences, a head group of eight
        dict(name="tree 8x12 at 32k fp16", op="tree", dtype="fp16", seqs=8, nodes_min=12,
             nodes_max=12, ctx_min=32768, ctx_max=32768, heads=64, kv_heads=8, dim=128, page=16,
             lens=5),
        # wide trees over middling contexts: as much arithmetic as memory traffic
        dict(name="tree 16x63 ragged bf16", op="tree", dtype="bf16", seqs=16, nodes_min=63,
             nodes_max=63, ctx_min=3001, ctx_max=9001, heads=32, kv_heads=8, dim=128, page=32,
             lens=6),
        # one sequence's accepted path, and a batch's, in every layer
        dict(name="commit 1 path", op="commit", dtype="fp16", layers=22, seqs=1, nodes_min=9,
             nodes_max=9, path_max=4, ctx_min=700, ctx_max=700, kv_heads=4, dim=64, page=16,
             lens=7),
        dict(name="commit 32 paths", op="commit", dtype="fp16", layers=32, seqs=32, nodes_min=20,
             nodes_max=63, path_max=8, ctx_min=1024, ctx_max=8192, kv_heads=8, dim=128, page=16,
             lens=8),
        # one request with four beams, and a batch of them over a large vocabulary
        dict(name="select 1x4 of 32000 fp32", op="select", dtype="fp32", seqs=1, beams=4,
             vocab=32000, outs=8, live=4, lens=9),
        dict(name="select 24x8 of 128256 fp16", op="select", dtype="fp16", seqs=24, beams=8,
             vocab=128256, outs=16, live=8, lens=10),
        # their states: the open pages of every layer and the page tables
        dict(name="reorder 1x4", op="reorder", dtype="fp16", layers=22, seqs=1, beams=4,
             ctx_min=301, ctx_max=301, kv_heads=4, dim=64, page=16, width=128, lens=11),
        dict(name="reorder 8x8", op="reorder", dtype="bf16", layers=32, seqs=8, beams=8,
             ctx_min=500, ctx_max=4000, kv_heads=8, dim=128, page=32, width=256, lens=12),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "tree", "tree", "commit", "select", "reorder"])
    dtype = rng.choice(["fp16", "bf16", "fp16", "bf16", "fp32"])
    page = rng.choice([16, 16, 32, 48, 64])
    dim = rng.choice([64, 96, 128, 128, 256])
    kv_heads, group = rng.choice([(1, 7), (2, 6), (4, 8), (8, 4), (8, 8), (8, 1), (5, 3)])
    c = dict(op=op, dtype=dtype, lens=rng.randrange(1 << 20))
    if op == "append":
        hi = _spread(rng, 1, 300)
        c.update(seqs=_spread(rng, 1, 16), new_min=max(1, hi // rng.randrange(1, 6)), new_max=hi,
                 ctx_min=0, ctx_max=_spread(rng, 16, 30000), heads=kv_heads * group,
                 kv_heads=kv_heads, dim=min(dim, 128), page=page, neox=rng.random() < 0.5,
                 base=rng.choice([10000.0, 500000.0]), fused=rng.random() < 0.5)
    elif op == "tree":
        ctx = _spread(rng, 1, 16000)
        seqs = _spread(rng, 1, max(1, min(24, 100000 // ctx)))
        nodes = _spread(rng, 1, 64)
        if dtype == "fp32":
            ctx, seqs = min(ctx, 4000), min(seqs, 4)
        if kv_heads * group * dim * nodes > 32 * 128 * 64:
            nodes = max(1, 32 * 128 * 64 // (kv_heads * group * dim))
        c.update(seqs=seqs, nodes_min=max(1, nodes // rng.randrange(1, 4)), nodes_max=nodes,
                 ctx_min=rng.choice([0, ctx // 2, ctx]), ctx_max=ctx, heads=kv_heads * group,
                 kv_heads=kv_heads, dim=dim, page=page)
    elif op == "commit":
        nodes = _spread(rng, 1, 64)
        c.update(layers=_spread(rng, 1, 32), seqs=_spread(rng, 1, 24), nodes_min=1,
                 nodes_max=nodes, path_max=min(nodes, rng.randrange(1, 9)),
                 ctx_min=0, ctx_max=_spread(rng, 8, 9000), kv_heads=min(kv_heads, 8),
                 dim=min(dim, 128), page=page)
    elif op == "select":
        beams = rng.randrange(1, 11)
        c.update(seqs=_spread(rng, 1, 16), beams=beams, vocab=_spread(rng, 50, 130000),
                 outs=min(32, 2 * beams), live=rng.choice([1, beams, beams]))
    else:
        c.update(layers=_spread(rng, 1, 32), seqs=_spread(rng, 1, 6), beams=rng.randrange(1, 9),
                 ctx_min=1, ctx_max=_spread(rng, 8, 3900), kv_heads=min(kv_heads, 8),
                 dim=min(dim, 128), page=page, width=256)
    return c


# -- sizes that a case fixes (the same for every seed) --------------------------------------
def _lengths(case):
    """Per sequence: cached positions, and new tokens / nodes where the case has them."""
    r = np.random.default_rng(case["lens"])
    n = case["seqs"]
    ctx = r.integers(case["ctx_min"], case["ctx_max"] + 1, n) if "ctx_min" in case else None
    lo = case.get("new_min", case.get("nodes_min"))
    new = None if lo is None else r.integers(lo, case.get("new_max", case.get("nodes_max")) + 1, n)
    return ctx, new


def _parents(count, r):
    """A drafted tree of `count` nodes: node i hangs below an earlier one, or the cache."""
    return [-1 if i == 0 else int(r.integers(-1, i)) for i in range(count)]


def _words(case):
    return (case["nodes_max"] + 31) // 32


def _bits(parents, words):
    """One row of mask words per node: itself and everything above it."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | (1 << i))
    m = [[(x >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for x in rows]
    return np.array(m, dtype=np.uint32).reshape(len(parents), words)


def _paths(case):
    """Accepted paths: ascending node numbers per sequence, and how many."""
    _, nodes = _lengths(case)
    r = np.random.default_rng(case["lens"] + 1)
    path = np.zeros((case["seqs"], case["path_max"]), dtype=np.int32)
    count = np.zeros(case["seqs"], dtype=np.int32)
    for i, n in enumerate(nodes):
        k = int(r.integers(min(2, n, case["path_max"]), min(int(n), case["path_max"]) + 1))
        path[i, :k] = np.sort(r.choice(int(n), size=k, replace=False))
        count[i] = k
    return path, count


def _beam_parents(case):
    r = np.random.default_rng(case["lens"] + 2)
    return r.integers(0, case["beams"], (case["seqs"], case["beams"])).astype(np.int32)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    ctx, new = _lengths(case)
    if case["op"] == "append":
        n, row = int(new.sum()), case["dim"] * e
        return {"bytes": 2 * n * row * (case["heads"] + 2 * case["kv_heads"]),
                "flops": 3 * n * case["dim"] * (case["heads"] + case["kv_heads"])}
    if case["op"] == "tree":
        kv = 2 * int((ctx + new).sum()) * case["kv_heads"] * case["dim"] * e
        io = 2 * int(new.sum()) * case["heads"] * case["dim"] * e
        return {"bytes": kv + io,
                "flops": 4 * case["dim"] * case["heads"] * int((new * (ctx + 1)).sum())}
    if case["op"] == "commit":
        path, count = _paths(case)
        live = (np.arange(case["path_max"]) < count[:, None]) & (path != np.arange(case["path_max"]))
        row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * e
        return {"bytes": 2 * max(1, int(live.sum())) * row, "flops": 0}
    if case["op"] == "select":
        n = case["seqs"] * case["beams"] * case["vocab"]
        return {"bytes": n * e + case["seqs"] * case["outs"] * 12, "flops": 3 * n}
    par = _beam_parents(case)
    moved = (par != np.arange(case["beams"])).sum(axis=1)
    row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * e
    tail = ctx % case["page"]
    return {"bytes": 2 * max(1, int((moved * tail).sum())) * row
            + 8 * int((moved * (ctx // case["page"])).sum()), "flops": 0}


# -- pools ------------------------------------------------------------------------------------
class _Memory:
    """Device memory of the library's pool as a torch tensor."""

    def __init__(self, ptr, nbytes, keep):
        self.keep = keep
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1",
                                         "data": (ptr, False), "version": 2}


def _pool_shape(case, layers, pages):
    d, ps = case["dim"], case["page"]
    inner = (ps, d) if case["dtype"] == "fp32" else (ps // 8, d // 8, 8, 8)
    return (layers, pages, case["kv_heads"]) + inner


def _pool(state, case, layers, pages, gen):
    """state["k"], state["v"]: normal values in the pool's layout (and the pool itself)."""
    shape, dt = _pool_shape(case, layers, pages), _DTYPES[case["dtype"]]
    if own:
        paged = _package("paged")
        pool = paged.PagedKVCache(layers, pages, case["page"], case["kv_heads"], case["dim"],
                                  dtype=dt, device=torch.cuda.current_device())
        info, n = pool.info(), math.prod(shape) * dt.itemsize
        state["pool"] = pool
        for key in ("k", "v"):
            mem = torch.as_tensor(_Memory(info[key], n, pool), device="cuda")
            state[key] = mem.view(dt).view(shape)
    else:
        state["k"] = torch.empty(shape, dtype=dt, device="cuda")
        state["v"] = torch.empty(shape, dtype=dt, device="cuda")
    for key in ("k", "v"):
        for layer in range(layers):
            state[key][layer] = torch.randn(shape[1:], generator=gen, device="cuda").to(dt)


def _package(name):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    return __import__(name)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _tables(case, need, r):
    """Page tables for `need` pages per row in a shuffled pool: (table, pages)."""
    total = int(need.sum())
    perm = r.permutation(total).astype(np.int32)
    table = np.zeros((len(need), max(1, int(need.max()))), dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += int(n)
    return table, max(1, total)


# -- states -----------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    r = np.random.default_rng([int(seed), case["lens"]])
    dt = _DTYPES[case["dtype"]]
    s = {"case": case, "op": case["op"]}
    ctx, new = _lengths(case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dt)

    if case["op"] == "append":
        n, hq, hk, d = int(new.sum()), case["heads"], case["kv_heads"], case["dim"]
        need = -(-(ctx + new) // case["page"])
        # pages below the new rows are not touched: the pool holds the others
        first = ctx // case["page"]
        table, pages = _tables(case, need - first, r)
        wide = np.zeros((case["seqs"], int(need.max())), dtype=np.int32)
        for i in range(case["seqs"]):
            wide[i, first[i]:need[i]] = table[i, :need[i] - first[i]]
        _pool(s, case, 1, pages, gen)
        s["bt"] = _cuda(wide)
        s["rows"] = _cuda(np.repeat(np.arange(case["seqs"]), new).astype(np.int32))
        s["pos"] = _cuda(np.concatenate([c + np.arange(k) for c, k in zip(ctx, new)])
                         .astype(np.int32))
        qkv = normal(n, hq + 2 * hk, d)
        s["q"], s["kn"], s["vn"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        if not case["fused"]:
            s["q"], s["kn"], s["vn"] = (s[x].contiguous() for x in ("q", "kn", "vn"))
        s["q_out"] = torch.zeros(n, hq, d, dtype=dt, device="cuda")
    elif case["op"] == "tree":
        n = int(new.sum())
        table, pages = _tables(case, -(-(ctx + new) // case["page"]), r)
        _pool(s, case, 1, pages, gen)
        s["bt"] = _cuda(table)
        mask = np.concatenate([_bits(_parents(int(k), r), _words(case)) for k in new])
        s["mask"] = _cuda(mask.view(np.int32))
        s["q"] = normal(n, case["heads"], case["dim"])
        s["out"] = torch.zeros_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(case["dim"])
        s["ctx"], s["new"] = _cuda(ctx.astype(np.int32)), _cuda(new.astype(np.int32))
        s["seq"] = _cuda(np.repeat(np.arange(case["seqs"]), new))
        s["node"] = _cuda(np.concatenate([np.arange(k) for k in new]))
        if own:  # the plan of a step serves all its layers
            s["plan"] = s["pool"].plan_tree(ctx.tolist(), new.tolist(), case["heads"])
    elif case["op"] == "commit":
        path, count = _paths(case)
        need = -(-(ctx + new) // case["page"])
        first = ctx // case["page"]
        table, pages = _tables(case, need - first, r)
        wide = np.zeros((case["seqs"], int(need.max())), dtype=np.int32)
        for i in range(case["seqs"]):
            wide[i, first[i]:need[i]] = table[i, :need[i] - first[i]]
        _pool(s, case, case["layers"], pages, gen)
        s["bt"], s["ctx"] = _cuda(wide), _cuda(ctx.astype(np.int32))
        s["path"], s["count"] = _cuda(path), _cuda(count)
    elif case["op"] == "select":
        n, b, v = case["seqs"], case["beams"], case["vocab"]
        s["logits"] = (3.0 * torch.randn(n * b, v, generator=gen, device="cuda")).to(dt)
        cum = -4.0 * torch.rand(n, b, generator=gen, device="cuda")
        cum[:, case["live"]:] = -math.inf  # the first step has one beam
        s["cum"] = cum
        s["tokens"] = torch.zeros(n, case["outs"], dtype=torch.int32, device="cuda")
        s["parents"] = torch.zeros_like(s["tokens"])
        s["scores"] = torch.zeros(n, case["outs"], device="cuda")
        if own:
            s["sel"] = _package("beam").BeamSelector(n, b, v, case["outs"],
                                                     device=torch.cuda.current_device())
    else:
        n, b, w = case["seqs"], case["beams"], case["width"]
        # the pool holds the open page of every beam; full pages are only named
        _pool(s, case, case["layers"], n * b, gen)
        table = r.integers(0, n * b, (n * b, w)).astype(np.int32)
        table[np.arange(n * b), np.repeat(np.minimum(ctx // case["page"], w - 1), b)] = \
            r.permutation(n * b)
        s["bt"], s["ctx"] = _cuda(table), _cuda(ctx.astype(np.int32))
        s["parent"] = _cuda(_beam_parents(case))
    return s


# -- one pass -----------------------------------------------------------------------------------
def run(s):
    return {"append": _append, "tree": _tree, "commit": _commit, "select": _select,
            "reorder": _reorder}[s["op"]](s)


def _rows(case, buf, page, t):
    """Rows (n, layers, kv_heads, dim) of positions t of pages `page`."""
    if case["dtype"] == "fp32":
        return buf[:, page, :, t]
    got = buf[:, page, :, t // 8, :, t % 8]
    return got.reshape(*got.shape[:-2], case["dim"])


def _set_rows(case, buf, page, t, rows):
    if case["dtype"] == "fp32":
        buf[:, page, :, t] = rows
    else:
        buf[:, page, :, t // 8, :, t % 8] = rows.reshape(*rows.shape[:-1], case["dim"] // 8, 8)


def _rotate(x, pos, base, neox):
    """Angles of far positions in 64 bits, the rotation in 32."""
    d = x.shape[-1]
    inv = base ** (-torch.arange(0, d, 2, device=x.device, dtype=torch.float64) / d)
    ang = (pos.double()[:, None] * inv)[:, None]
    cos, sin = ang.cos().float(), ang.sin().float()
    x = x.float()
    if neox:
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)


def _append(s):
    case = s["case"]
    if own:
        s["pool"].append_rope(0, s["q"], s["kn"], s["vn"], s["bt"], s["pos"], rows=s["rows"],
                              q_out=s["q_out"], freq_base=case["base"], neox=case["neox"])
        return s["q_out"], s["k"], s["v"]
    pos = s["pos"].long()
    page = s["bt"][s["rows"].long(), pos // case["page"]].long()
    dt = _DTYPES[case["dtype"]]
    s["q_out"].copy_(_rotate(s["q"], pos, case["base"], case["neox"]).to(dt))
    k = _rotate(s["kn"], pos, case["base"], case["neox"]).to(dt)
    _set_rows(case, s["k"], page, pos % case["page"], k[:, None])
    _set_rows(case, s["v"], page, pos % case["page"], s["vn"][:, None])
    return s["q_out"], s["k"], s["v"]


def _cached(case, buf, bt):
    """fp32 (sequences, kv_heads, positions, dim) of all pages of the tables."""
    x = buf[0][bt.long()].float()
    if case["dtype"] != "fp32":  # (seqs, pages, heads, t / 8, d / 8, 8, 8)
        x = x.transpose(-3, -2).flatten(-2).flatten(-3, -2)
    return x.transpose(1, 2).flatten(2, 3)


def _tree(s):
    case = s["case"]
    if own:
        s["pool"].decode_tree(s["plan"], 0, s["q"], s["mask"], s["out"], s["bt"], s["scale"])
        return s["out"]
    n, h, hk, d = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    most = case["nodes_max"]
    k, v = _cached(case, s["k"], s["bt"]), _cached(case, s["v"], s["bt"])
    length = k.shape[2]
    q = torch.zeros(n, most, h, d, device="cuda")
    q[s["seq"], s["node"]] = s["q"].float()
    q = q.view(n, most, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    # who sees what: the cached positions, and the nodes of the mask's bits
    j = torch.arange(most, device="cuda")
    seen = (s["mask"][:, j // 32] >> (j % 32)) & 1
    nodes = torch.zeros(n, most, most, dtype=torch.bool, device="cuda")
    nodes[s["seq"], s["node"]] = seen.bool()
    at = torch.arange(length, device="cuda")
    rel = at[None] - s["ctx"][:, None]                                    # (n, length)
    drafted = (rel >= 0) & (rel < s["new"][:, None])
    ok = nodes.gather(2, rel.clamp(0, most - 1).long()[:, None].expand(n, most, length))
    ok = (rel < 0)[:, None] | (drafted[:, None] & ok)
    p = (q @ k.transpose(-1, -2)) * s["scale"]
    ok = ok[:, None].repeat_interleave(h // hk, dim=2)
    p = p.masked_fill_(~ok, -math.inf)
    p = (p - p.amax(dim=-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    out = (p @ v) / total.masked_fill(total == 0, 1.0)
    out = out.view(n, hk, most, h // hk, d).permute(0, 2, 1, 3, 4).reshape(n, most, h, d)
    s["out"].copy_(out[s["seq"], s["node"]].to(s["out"].dtype))
    return s["out"]


def _commit(s):
    case = s["case"]
    if own:
        s["pool"].commit_tree(s["bt"], s["ctx"], s["path"], s["count"])
        return s["k"], s["v"]
    j = torch.arange(case["path_max"], device="cuda")
    src = torch.where(j < s["count"][:, None], s["path"], j)  # past the path: onto itself
    src, dst = s["ctx"][:, None] + src, s["ctx"][:, None] + j
    live = (j < s["count"][:, None]).flatten()
    last = s["bt"].shape[1] - 1
    row = torch.arange(case["seqs"], device="cuda")[:, None]
    ps = case["page"]
    src_page = s["bt"][row, (src // ps).clamp(max=last)].flatten().long()
    dst_page = s["bt"][row, (dst // ps).clamp(max=last)].flatten().long()
    src_page, dst_page = src_page[live], dst_page[live]
    src_t, dst_t = (src % ps).flatten()[live].long(), (dst % ps).flatten()[live].long()
    _set_rows(case, s["k"], dst_page, dst_t, _rows(case, s["k"], src_page, src_t))
    _set_rows(case, s["v"], dst_page, dst_t, _rows(case, s["v"], src_page, src_t))
    return s["k"], s["v"]


def _select(s):
    case = s["case"]
    if own:
        s["sel"].select(s["logits"], s["cum"], case["outs"],
                        out=(s["tokens"], s["parents"], s["scores"]))
        return s["tokens"], s["parents"], s["scores"]
    n, b, v = case["seqs"], case["beams"], case["vocab"]
    x = s["logits"].double()  # candidates of different beams next to each other: 64 bits
    top = x.amax(dim=1, keepdim=True)
    lse = top + (x - top).exp().sum(dim=1, keepdim=True).log()
    score = (s["cum"].double().view(-1, 1) + (x - lse)).view(n, b * v)
    best, at = torch.sort(score, dim=1, descending=True, stable=True)
    at = at[:, :case["outs"]]
    s["tokens"].copy_(at % v)
    s["parents"].copy_(torch.div(at, v, rounding_mode="floor"))
    s["scores"].copy_(best[:, :case["outs"]])
    return s["tokens"], s["parents"], s["scores"]


def _reorder(s):
    case = s["case"]
    if own:
        s["pool"].reorder_beams(s["bt"], s["parent"], s["ctx"])
        return s["bt"], s["k"], s["v"]
    n, b, w, ps = case["seqs"], case["beams"], case["width"], case["page"]
    old = s["bt"].view(n, b, w)
    row = torch.arange(n, device="cuda")[:, None]
    parent = s["parent"].long()
    col = (s["ctx"].long() // ps).clamp(max=w - 1)
    mine = old.gather(2, col.view(n, 1, 1).expand(n, b, 1))[..., 0].long()   # open pages
    theirs = mine.gather(1, parent)
    t = torch.arange(ps, device="cuda")
    open_rows = (t[None] < (s["ctx"] % ps)[:, None]).repeat_interleave(b, dim=0)  # (n * b, ps)
    if case["dtype"] == "fp32":
        move = open_rows.view(1, n * b, 1, ps, 1)
    else:
        move = open_rows.view(1, n * b, 1, ps // 8, 1, 8, 1)
    mine, theirs = mine.flatten(), theirs.flatten()
    s["k"][:, mine] = torch.where(move, s["k"][:, theirs], s["k"][:, mine])
    s["v"][:, mine] = torch.where(move, s["v"][:, theirs], s["v"][:, mine])
    full = torch.arange(w, device="cuda") < (s["ctx"] // ps)[:, None, None]
    s["bt"].copy_(torch.where(full, old[row, parent], old).view(n * b, w))
    return s["bt"], s["k"], s["v"]


# -- the operators' definitions in 64 bits -------------------------------------------------------
def _dense(case, buf):
    """fp64 (layers, pages, heads, positions, dim) of a pool."""
    if case["dtype"] == "fp32":
        return buf.double()
    x = buf.double().permute(0, 1, 2, 3, 5, 4, 6)
    return x.reshape(*buf.shape[:3], case["page"], case["dim"])


def _laid(case, x):
    """_dense undone."""
    if case["dtype"] == "fp32":
        return x
    d, ps = case["dim"], case["page"]
    return x.reshape(*x.shape[:3], ps // 8, 8, d // 8, 8).permute(0, 1, 2, 3, 5, 4, 6).contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    ctx, new = _lengths(case)
    if case["op"] == "select":
        n, b, v = case["seqs"], case["beams"], case["vocab"]
        out = torch.zeros(n, case["outs"], dtype=torch.float64, device="cuda")
        for i in range(n):
            logp = torch.log_softmax(s["logits"][i * b:(i + 1) * b].double(), dim=1)
            score = (logp + s["cum"][i].double()[:, None]).flatten()
            out[i] = score.topk(case["outs"]).values
        return None, None, out
    k, v = _dense(case, s["k"]), _dense(case, s["v"])
    bt, ps = s["bt"].cpu().numpy(), case["page"]
    if case["op"] == "append":
        d = case["dim"]
        freq = np.power(float(case["base"]), -2.0 * np.arange(d // 2) / d)
        ang = torch.from_numpy(s["pos"].cpu().numpy().astype(np.float64)[:, None] * freq).cuda()
        turn = torch.polar(torch.ones_like(ang), ang)[:, None]

        def rot(x):
            x = x.double()
            if case["neox"]:
                y = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * turn
                return torch.cat([y.real, y.imag], dim=-1)
            y = torch.view_as_complex(x.unflatten(-1, (d // 2, 2)).contiguous()) * turn
            return torch.view_as_real(y).flatten(-2)

        kn, vn, at = rot(s["kn"]), s["vn"].double(), 0
        for i in range(case["seqs"]):
            for c in range(int(ctx[i]), int(ctx[i] + new[i])):
                k[0, bt[i, c // ps], :, c % ps] = kn[at]
                v[0, bt[i, c // ps], :, c % ps] = vn[at]
                at += 1
        return rot(s["q"]), _laid(case, k), _laid(case, v)
    if case["op"] == "tree":
        hk, g, d = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
        mask = s["mask"].cpu().numpy().view(np.uint32)
        out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
        for i in range(case["seqs"]):
            c, m = int(ctx[i]), int(new[i])
            pages = torch.from_numpy(bt[i, :-(-(c + m) // ps)].astype(np.int64)).cuda()
            ki = k[0, pages].transpose(0, 1).reshape(hk, -1, d)[:, :c + m]
            vi = v[0, pages].transpose(0, 1).reshape(hk, -1, d)[:, :c + m]
            ok = np.ones((m, c + m), dtype=bool)
            for a in range(m):
                ok[a, c:] = [(int(mask[at + a, x // 32]) >> (x % 32)) & 1 for x in range(m)]
            ok = torch.from_numpy(ok).cuda()
            qi = s["q"][at:at + m].double().view(m, hk, g, d)
            sc = torch.einsum("mhgd,hld->hgml", qi, ki) * s["scale"]
            w = torch.softmax(sc.masked_fill(~ok, -math.inf), dim=-1)
            out[at:at + m] = torch.einsum("hgml,hld->mhgd", w, vi).reshape(m, hk * g, d)
            at += m
        return out
    if case["op"] == "commit":
        path, count = _paths(case)
        k0, v0 = k.clone(), v.clone()
        for i in range(case["seqs"]):
            for j in range(int(count[i])):
                a, z = int(ctx[i] + path[i, j]), int(ctx[i]) + j
                k[:, bt[i, z // ps], :, z % ps] = k0[:, bt[i, a // ps], :, a % ps]
                v[:, bt[i, z // ps], :, z % ps] = v0[:, bt[i, a // ps], :, a % ps]
        return _laid(case, k), _laid(case, v)
    par, b = _beam_parents(case), case["beams"]
    k0, v0 = k.clone(), v.clone()
    for i in range(case["seqs"]):
        col, t = int(ctx[i]) // ps, int(ctx[i]) % ps
        for x in range(b):
            if t:
                z, a = bt[i * b + x, col], bt[i * b + par[i, x], col]
                k[:, z, :, :t], v[:, z, :, :t] = k0[:, a, :, :t], v0[:, a, :, :t]
    return None, _laid(case, k), _laid(case, v)
