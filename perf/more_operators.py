"""Performance cases of four further operators of the paged KV pool.

``norm``    a step's q and K heads normalised, rotated (by one position or by one per
            axis of an image or a video) and appended with their V rows, in one pass
``shared``  attention of a decode batch whose sequences share long prefixes: a prefix's
            pages are read once for all of its members
``weigh``   attention that also adds its weights up, per cached slot and KV head
``evict``   the slots with the least weight leave the cache, the others move together

``own`` False computes each operator in its plain form, elementary torch operations in
32 or 64 bits on the same buffers; ``own`` True makes the library calls.  Pools keep the
library's layout in both forms: 16-bit storage holds, for each page and KV head,
8-position x 16-byte blocks (positions / 8, head_dim / 8, 8 positions, 8 dims), fp32
storage plain rows.
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
_EPS = 1e-6


# -- cases --------------------------------------------------------------------------------
def listed():
    return [
        # one token of one sequence: the step's latency
        dict(name="norm 1 token fp32", op="norm", dtype="fp32", seqs=1, new_min=1, new_max=1,
             ctx_min=511, ctx_max=511, heads=32, kv_heads=4, dim=64, page=16, rotary=64,
             neox=True, base=10000.0, sections="", order="blocks", fused=False, lens=1),
        # a decode step of a serving batch, rows cut from a fused QKV product
        dict(name="norm 48 tokens bf16", op="norm", dtype="bf16", seqs=48, new_min=1, new_max=1,
             ctx_min=100, ctx_max=8000, heads=32, kv_heads=8, dim=128, page=16, rotary=128,
             neox=True, base=500000.0, sections="", order="blocks", fused=True, lens=2),
        # prompts with images going in at once: positions in time, height and width
        dict(name="norm 12 image prompts fp16", op="norm", dtype="fp16", seqs=12, new_min=333,
             new_max=1201, ctx_min=0, ctx_max=2000, heads=32, kv_heads=8, dim=128, page=32,
             rotary=128, neox=True, base=500000.0, sections="24,20,20", order="cyclic",
             fused=True, lens=3),
        # four answers to one short question of a small model: latency again
        dict(name="shared 4 on 512 fp16", op="shared", dtype="fp16", groups=1, members_min=4,
             members_max=4, prefix_min=512, prefix_max=512, own_min=1, own_max=40, heads=32,
             kv_heads=4, dim=64, page=16, lens=4),
        # a serving batch in front of a handful of system prompts, some requests alone
        dict(name="shared 9 groups ragged fp16", op="shared", dtype="fp16", groups=9,
             members_min=1, members_max=12, prefix_min=500, prefix_max=6000, own_min=50,
             own_max=1200, heads=32, kv_heads=8, dim=128, page=32, lens=5),
        # many requests on one long document: the prefix is compute, not memory
        dict(name="shared 96 on 24k bf16", op="shared", dtype="bf16", groups=1, members_min=96,
             members_max=96, prefix_min=24576, prefix_max=24576, own_min=30, own_max=700,
             heads=64, kv_heads=8, dim=128, page=16, lens=6),
        # one short sequence, one token
        dict(name="weigh 1x1 at 511 fp32", op="weigh", dtype="fp32", seqs=1, new_min=1, new_max=1,
             ctx_min=511, ctx_max=511, heads=32, kv_heads=4, dim=64, page=16, lens=7),
        # a decode step of an ordinary serving batch, grouped heads
        dict(name="weigh 32x1 ragged fp16", op="weigh", dtype="fp16", seqs=32, new_min=1,
             new_max=1, ctx_min=1024, ctx_max=8192, heads=32, kv_heads=8, dim=128, page=16,
             lens=8),
        # prompts that go in piece by piece, every token's weights counted
        dict(name="weigh 4x(20..100) bf16", op="weigh", dtype="bf16", seqs=4, new_min=20,
             new_max=100, ctx_min=700, ctx_max=4001, heads=32, kv_heads=8, dim=128, page=32,
             lens=9),
        # a small model's one sequence, cut back by a few pages
        dict(name="evict 1 of 600 to 512 fp16", op="evict", dtype="fp16", layers=22, seqs=1,
             ctx_min=600, ctx_max=600, budget=512, recent=64, kv_heads=4, dim=64, page=16,
             lens=10),
        # a batch of long prompts cut to its budget after they went in
        dict(name="evict 8 ragged to 1024 bf16", op="evict", dtype="bf16", layers=32, seqs=8,
             ctx_min=900, ctx_max=3100, budget=1024, recent=200, kv_heads=8, dim=128, page=32,
             lens=11),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "shared", "shared", "weigh", "evict"])
    dtype = rng.choice(["fp16", "bf16", "fp16", "bf16", "fp32"])
    page = rng.choice([16, 16, 32, 48, 64])
    dim = rng.choice([64, 96, 128, 128, 256])
    kv_heads, group = rng.choice([(1, 7), (2, 6), (4, 8), (8, 4), (8, 8), (8, 1), (5, 3)])
    c = dict(op=op, dtype=dtype, lens=rng.randrange(1 << 20))
    if op == "norm":
        hi = _spread(rng, 1, 500)
        rotary = rng.choice([dim, dim, dim // 2])
        a = rotary // 2
        sections = rng.choice(["", f"{a}", f"{a // 2},{a - a // 2}",
                               f"{a - 2 * (a // 3)},{a // 3},{a // 3}"])
        c.update(seqs=_spread(rng, 1, 16), new_min=max(1, hi // rng.randrange(1, 6)), new_max=hi,
                 ctx_min=0, ctx_max=_spread(rng, 16, 30000), heads=kv_heads * group,
                 kv_heads=kv_heads, dim=dim, page=page, rotary=rotary, neox=rng.random() < 0.7,
                 base=rng.choice([10000.0, 500000.0]), sections=sections,
                 order=rng.choice(["blocks", "cyclic", "ladders"]), fused=rng.random() < 0.5)
    elif op == "shared":
        groups = rng.randrange(1, 7)
        members = _spread(rng, 1, 64 // groups)
        prefix = _spread(rng, 16, 16000)
        if dtype == "fp32":
            members, prefix, groups = min(members, 12), min(prefix, 3000), min(groups, 3)
        c.update(groups=groups, members_min=max(1, members // rng.randrange(1, 4)),
                 members_max=members, prefix_min=rng.choice([0, prefix // 2, prefix]),
                 prefix_max=prefix, own_min=1, own_max=_spread(rng, 1, 1500),
                 heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page)
    elif op == "weigh":
        ctx = _spread(rng, 1, 12000)
        new = rng.choice([1, 1, _spread(rng, 1, 64)])
        seqs = _spread(rng, 1, max(1, min(24, 100000 // ctx // new)))
        if dtype == "fp32":
            ctx, seqs = min(ctx, 4000), min(seqs, 4)
        c.update(seqs=seqs, new_min=max(1, new // rng.randrange(1, 4)), new_max=new,
                 ctx_min=rng.choice([0, ctx // 2, ctx]), ctx_max=ctx, heads=kv_heads * group,
                 kv_heads=kv_heads, dim=min(dim, 128) if new > 8 else dim, page=page)
    else:
        ctx = _spread(rng, 64, 3000)
        budget = max(1, int(ctx * rng.uniform(0.2, 1.0)))
        c.update(layers=_spread(rng, 1, 32), seqs=_spread(rng, 1, 6),
                 ctx_min=rng.choice([1, ctx // 2, ctx]), ctx_max=ctx, budget=budget,
                 recent=rng.choice([0, budget // 8, budget // 2]), kv_heads=kv_heads,
                 dim=min(dim, 128), page=page)
    return c


# -- sizes that a case fixes (the same for every seed) --------------------------------------
def _lengths(case):
    """Per sequence: cached positions, and new tokens where the case has them."""
    r = np.random.default_rng(case["lens"])
    n = case["seqs"]
    ctx = r.integers(case["ctx_min"], case["ctx_max"] + 1, n)
    new = r.integers(case["new_min"], case["new_max"] + 1, n) if "new_min" in case else None
    return ctx, new


def _groups(case):
    """A shared batch: members and prefix of each group, and each member's whole length."""
    r = np.random.default_rng(case["lens"])
    n, ps = case["groups"], case["page"]
    members = r.integers(case["members_min"], case["members_max"] + 1, n)
    prefix = r.integers(case["prefix_min"], case["prefix_max"] + 1, n) // ps * ps
    lens = np.repeat(prefix, members) + r.integers(case["own_min"], case["own_max"] + 1,
                                                   int(members.sum()))
    return members, prefix, lens


def _sections(case):
    """Pairs of each axis."""
    return [int(x) for x in case["sections"].split(",")] if case["sections"] else []


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "shared":
        members, prefix, lens = _groups(case)
        own_rows = int((lens - np.repeat(prefix, members)).sum())
        kv = 2 * (int(prefix.sum()) + own_rows) * case["kv_heads"] * case["dim"] * e
        io = 2 * len(lens) * case["heads"] * case["dim"] * e
        return {"bytes": kv + io, "flops": 4 * case["dim"] * case["heads"] * int(lens.sum())}
    ctx, new = _lengths(case)
    if case["op"] == "norm":
        n, row = int(new.sum()), case["dim"] * e
        return {"bytes": 2 * n * row * (case["heads"] + 2 * case["kv_heads"]),
                "flops": 7 * n * case["dim"] * (case["heads"] + case["kv_heads"])}
    if case["op"] == "weigh":
        kv = 2 * int((ctx + new).sum()) * case["kv_heads"] * case["dim"] * e
        io = 2 * int(new.sum()) * case["heads"] * case["dim"] * e
        sums = 4 * int((2 * ctx + new).sum()) * case["kv_heads"]
        seen = int((new * ctx + new * (new + 1) // 2).sum())
        return {"bytes": kv + io + sums, "flops": 4 * case["dim"] * case["heads"] * seen}
    full = ctx > case["budget"]
    heads = case["layers"] * case["kv_heads"]
    keep = int(np.minimum(ctx, case["budget"]).sum())
    moved = int(full.sum()) * case["budget"]
    return {"bytes": heads * (4 * moved * case["dim"] * e + 4 * int(ctx.sum()) + 8 * keep),
            "flops": 0}


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


def _tables(need, r):
    """Page tables for `need` pages per row in a shuffled pool: (table, pages)."""
    total = int(need.sum())
    perm = r.permutation(total).astype(np.int32)
    table = np.zeros((len(need), max(1, int(need.max()))), dtype=np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += int(n)
    return table, max(1, total)


def _axes_positions(ctx, count, axes, r):
    """Rotary positions (count, axes) of a prompt: text, an image, text.  Text counts up on
    every axis; an image keeps its first axis and counts rows and columns on the others."""
    at, out = int(ctx), []
    while len(out) < count:
        for _ in range(int(r.integers(5, 60))):
            out.append([at] * axes)
            at += 1
        h, w = int(r.integers(4, 25)), int(r.integers(4, 25))
        for i in range(h * w):
            out.append([at, at + i // w, at + i % w][:axes])
        at += max(h, w)
    return np.array(out[:count], dtype=np.int32)


# -- states -----------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    r = np.random.default_rng([int(seed), case["lens"]])
    dt = _DTYPES[case["dtype"]]
    s = {"case": case, "op": case["op"]}
    ps, d, hk = case["page"], case["dim"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dt)

    if case["op"] == "norm":
        ctx, new = _lengths(case)
        n, hq = int(new.sum()), case["heads"]
        # pages below the new rows are not touched: the pool holds the others
        need, first = -(-(ctx + new) // ps), ctx // ps
        table, pages = _tables(need - first, r)
        wide = np.zeros((case["seqs"], int(need.max())), dtype=np.int32)
        for i in range(case["seqs"]):
            wide[i, first[i]:need[i]] = table[i, :need[i] - first[i]]
        _pool(s, case, 1, pages, gen)
        s["bt"] = _cuda(wide)
        s["rows"] = _cuda(np.repeat(np.arange(case["seqs"]), new).astype(np.int32))
        s["pos"] = _cuda(np.concatenate([c + np.arange(k) for c, k in zip(ctx, new)])
                         .astype(np.int32))
        axes = len(_sections(case))
        s["turn"] = None
        if axes:
            s["turn"] = _cuda(np.concatenate([_axes_positions(c, k, axes, r)
                                              for c, k in zip(ctx, new)]))
        qkv = normal(n, hq + 2 * hk, d)
        s["q"], s["kn"], s["vn"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        if not case["fused"]:
            s["q"], s["kn"], s["vn"] = (s[x].contiguous() for x in ("q", "kn", "vn"))
        s["qw"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dt)
        s["kw"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dt)
        s["q_out"] = torch.zeros(n, hq, d, dtype=dt, device="cuda")
        if own:  # one table of angles serves all steps and layers
            s["rotation"] = _package("paged").Rotation(
                case["rotary"], freq_base=case["base"], sections=_sections(case) or None,
                order=case["order"], neox=case["neox"])
    elif case["op"] == "shared":
        members, prefix, lens = _groups(case)
        group = np.repeat(np.arange(len(members)), members)
        table, pages = _tables(np.concatenate([-(-lens // ps) - prefix[group] // ps,
                                               prefix // ps]), r)
        wide = np.zeros((len(lens), int((-(-lens // ps)).max())), dtype=np.int32)
        for i, g in enumerate(group):
            a, b = int(prefix[g]) // ps, -(-int(lens[i]) // ps)
            wide[i, :a] = table[len(lens) + g, :a]
            wide[i, a:b] = table[i, :b - a]
        _pool(s, case, 1, pages, gen)
        s["bt"] = _cuda(wide)
        s["lens"] = _cuda(lens.astype(np.int32))
        s["q"] = normal(len(lens), case["heads"], d)
        s["out"] = torch.zeros_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(d)
        if own:  # the plan of a step serves all its layers
            s["plan"] = s["pool"].plan_shared(lens.tolist(), members.tolist(), prefix.tolist(),
                                              case["heads"])
    elif case["op"] == "weigh":
        ctx, new = _lengths(case)
        n = int(new.sum())
        table, pages = _tables(-(-(ctx + new) // ps), r)
        _pool(s, case, 1, pages, gen)
        s["bt"] = _cuda(table)
        s["q"] = normal(n, case["heads"], d)
        s["out"] = torch.zeros_like(s["q"])
        # what earlier steps have added up
        s["weights"] = torch.rand(case["seqs"], hk, table.shape[1] * ps, generator=gen,
                                  device="cuda").square_().mul_(4.0)
        s["scale"] = 1.0 / math.sqrt(d)
        s["ctx"], s["new"] = _cuda(ctx.astype(np.int32)), _cuda(new.astype(np.int32))
        s["seq"] = _cuda(np.repeat(np.arange(case["seqs"]), new))
        s["node"] = _cuda(np.concatenate([np.arange(k) for k in new]))
        if own:
            s["plan"] = s["pool"].plan_tree(ctx.tolist(), new.tolist(), case["heads"],
                                            weights=True)
    else:
        ctx, _ = _lengths(case)
        table, pages = _tables(-(-ctx // ps), r)
        _pool(s, case, case["layers"], pages, gen)
        s["bt"], s["ctx"] = _cuda(table), _cuda(ctx.astype(np.int32))
        shape = (case["layers"], case["seqs"], hk, table.shape[1] * ps)
        # a few slots draw most of the weight
        s["weights"] = torch.randn(shape, generator=gen, device="cuda").mul_(1.5).exp_()
        s["left"] = torch.zeros_like(s["weights"])
        s["kept"] = torch.zeros(shape[:3] + (case["budget"],), dtype=torch.int32, device="cuda")
    return s


# -- one pass -----------------------------------------------------------------------------------
def run(s):
    return {"norm": _norm, "shared": _shared, "weigh": _weigh, "evict": _evict}[s["op"]](s)


def _pair_table(case):
    """(inverse frequency, axis) of each rotated pair, in 64 bits."""
    half, sec = case["rotary"] // 2, _sections(case) or [case["rotary"] // 2]
    base, j = float(case["base"]), torch.arange(case["rotary"] // 2, dtype=torch.float64)
    inv = base ** (-j / half)
    if case["order"] == "cyclic":
        a = (torch.arange(half) % len(sec))
        turn = torch.arange(half) // len(sec)
        return inv, torch.where(turn < torch.tensor(sec)[a], a, torch.zeros_like(a))
    axis = torch.repeat_interleave(torch.arange(len(sec)), torch.tensor(sec))
    if case["order"] == "ladders":
        inv = torch.cat([base ** (-torch.arange(n, dtype=torch.float64) / n) for n in sec])
    return inv, axis


def _normed(x, w):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + _EPS) * w.float()


def _rotate(x, cos, sin, rot, neox):
    """The first `rot` dims of x turned by the pairs' angles, in 32 bits."""
    y, rest = x[..., :rot], x[..., rot:]
    if neox:
        a, b = y[..., :rot // 2], y[..., rot // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    else:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([y, rest], dim=-1)


def _norm(s):
    case = s["case"]
    if own:
        s["pool"].append_norm_rope(0, s["q"], s["kn"], s["vn"], s["bt"], s["pos"], s["rotation"],
                                   rows=s["rows"], rope_positions=s["turn"], q_weight=s["qw"],
                                   k_weight=s["kw"], eps=_EPS, q_out=s["q_out"])
        return s["q_out"], s["k"], s["v"]
    inv, axis = _pair_table(case)
    inv, axis = inv.cuda(), axis.cuda()
    turn = s["pos"][:, None] if s["turn"] is None else s["turn"]
    ang = (turn[:, axis].double() * inv)[:, None]                # (n, 1, pairs)
    cos, sin = ang.cos().float(), ang.sin().float()
    dt, rot = _DTYPES[case["dtype"]], case["rotary"]
    s["q_out"].copy_(_rotate(_normed(s["q"], s["qw"]), cos, sin, rot, case["neox"]).to(dt))
    k = _rotate(_normed(s["kn"], s["kw"]), cos, sin, rot, case["neox"]).to(dt)
    pos = s["pos"].long()
    page, t = s["bt"][s["rows"].long(), pos // case["page"]].long(), pos % case["page"]
    for buf, rows in ((s["k"], k), (s["v"], s["vn"])):
        if case["dtype"] == "fp32":
            buf[0, page, :, t] = rows
        else:
            buf[0, page, :, t // 8, :, t % 8] = rows.unflatten(-1, (-1, 8))
    return s["q_out"], s["k"], s["v"]


def _dense(case, x):
    """(..., positions, dim) of pages (..., the pool's layout of one head)."""
    if case["dtype"] == "fp32":
        return x
    return x.transpose(-3, -2).flatten(-2).flatten(-3, -2)


def _cached(case, buf, bt):
    """fp32 (sequences, kv_heads, positions, dim) of the pages of the tables."""
    return _dense(case, buf[0][bt.long()].float()).transpose(1, 2).flatten(2, 3)


def _shared(s):
    case = s["case"]
    if own:
        s["pool"].decode_shared(s["plan"], 0, s["q"], s["out"], s["bt"], s["scale"])
        return s["out"]
    members, prefix, lens = _groups(case)
    hk, d, ps = case["kv_heads"], case["dim"], case["page"]
    at = 0
    for m, p in zip(members.tolist(), prefix.tolist()):
        bt = s["bt"][at:at + m]
        q = s["q"][at:at + m].float().view(m, hk, -1, d)
        last = -(-int(lens[at:at + m].max()) // ps)
        kp, vp = (_cached(case, s[x], bt[:1, :p // ps])[0] for x in ("k", "v"))
        ko, vo = (_cached(case, s[x], bt[:, p // ps:last]) for x in ("k", "v"))
        # (kv_heads, members * group, prefix) and (members, kv_heads, group, own)
        rows = m * q.shape[2]
        sp = (q.transpose(0, 1).reshape(hk, rows, d) @ kp.transpose(-1, -2)) * s["scale"]
        so = (q @ ko.transpose(-1, -2)) * s["scale"]
        seen = p + torch.arange(so.shape[-1], device="cuda") < s["lens"][at:at + m, None]
        so = so.masked_fill(~seen[:, None, None], -math.inf)
        sp = sp.view(hk, m, q.shape[2], p).transpose(0, 1)
        top = so.amax(dim=-1, keepdim=True)
        if p:
            top = torch.maximum(top, sp.amax(dim=-1, keepdim=True))
        eo, ep = (so - top).exp(), (sp - top).exp()
        total = eo.sum(dim=-1, keepdim=True) + ep.sum(dim=-1, keepdim=True)
        out = eo @ vo + (ep.transpose(0, 1).reshape(hk, rows, p) @ vp).view(
            hk, m, -1, d).transpose(0, 1)
        s["out"][at:at + m] = (out / total).view(m, -1, d).to(s["out"].dtype)
        at += m
    return s["out"]


def _weigh(s):
    case = s["case"]
    if own:
        s["pool"].decode_tree_weights(s["plan"], 0, s["q"], None, s["weights"], s["out"], s["bt"],
                                      s["scale"])
        return s["out"], s["weights"]
    n, h, hk, d = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    most = int(_lengths(case)[1].max())
    k, v = _cached(case, s["k"], s["bt"]), _cached(case, s["v"], s["bt"])
    length = k.shape[2]
    q = torch.zeros(n, most, h, d, device="cuda")
    q[s["seq"], s["node"]] = s["q"].float()
    q = q.view(n, most, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    at = torch.arange(length, device="cuda")
    rel = at[None] - s["ctx"][:, None]                                    # (n, length)
    node = torch.arange(most, device="cuda")
    ok = rel[:, None] <= node[:, None]                                    # (n, most, length)
    p = (q @ k.transpose(-1, -2)) * s["scale"]
    p = p.masked_fill_(~ok[:, None].repeat_interleave(h // hk, dim=2), -math.inf)
    p = (p - p.amax(dim=-1, keepdim=True)).exp_()
    p = p / p.sum(dim=-1, keepdim=True)
    out = (p @ v).view(n, hk, most, h // hk, d).permute(0, 2, 1, 3, 4).reshape(n, most, h, d)
    s["out"].copy_(out[s["seq"], s["node"]].to(s["out"].dtype))
    p = p.view(n, hk, most, h // hk, length)
    p = p * (node < s["new"][:, None]).view(n, 1, most, 1, 1)             # padded rows
    add = p.sum(dim=(2, 3))
    fresh = ((rel >= 0) & (rel < s["new"][:, None]))[:, None]             # slots of new tokens
    s["weights"].copy_(torch.where(fresh, add, s["weights"] + add))
    return s["out"], s["weights"]


def _move(case, buf, bt, kept):
    """Every kept row of every layer and head to its new place."""
    shape, ps = kept.shape, case["page"]

    def along(dim):
        view = [1, 1, 1, 1]
        view[dim] = -1
        return torch.arange(shape[dim], device="cuda").view(view).expand(shape)

    live = kept >= 0
    layer, row, head, z = (along(i)[live] for i in range(4))
    a = kept[live].long()
    pa, pz = bt[row, a // ps].long(), bt[row, z // ps].long()
    if case["dtype"] == "fp32":
        buf[layer, pz, head, z % ps] = buf[layer, pa, head, a % ps]
    else:
        a, z = a % ps, z % ps
        buf[layer, pz, head, z // 8, :, z % 8] = buf[layer, pa, head, a // 8, :, a % 8]


def _evict(s):
    case = s["case"]
    if own:
        s["pool"].evict(s["bt"], s["ctx"], s["weights"], case["budget"], recent=case["recent"],
                        weights_out=s["left"], kept=s["kept"])
        return s["kept"], s["left"], s["k"], s["v"]
    w, budget = s["weights"], case["budget"]
    slot = torch.arange(w.shape[-1], device="cuda")
    ctx = s["ctx"].view(1, -1, 1, 1)
    key = torch.where(slot >= ctx - case["recent"], math.inf, w)
    key = torch.where(slot >= ctx, -math.inf, key)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    if order.shape[-1] < budget:
        order = torch.nn.functional.pad(order, (0, budget - order.shape[-1]), value=w.shape[-1])
    kept = torch.where(order < ctx, order, w.shape[-1]).sort(dim=-1).values
    live = kept < ctx
    s["kept"].copy_(torch.where(live, kept, -1))
    left = w.gather(-1, kept.clamp(max=w.shape[-1] - 1))
    cut = min(budget, w.shape[-1])
    s["left"][..., :cut] = torch.where(live, left, s["left"].new_zeros(()))[..., :cut]
    _move(case, s["k"], s["bt"], s["kept"])
    _move(case, s["v"], s["bt"], s["kept"])
    return s["kept"], s["left"], s["k"], s["v"]


# -- the operators' definitions in 64 bits -------------------------------------------------------
def _rows64(case, buf, pages, length):
    """fp64 (kv_heads, length, dim) of one sequence's pages of layer 0."""
    x = buf[0, torch.from_numpy(pages.astype(np.int64)).cuda()].double()
    if case["dtype"] != "fp32":      # (pages, heads, t / 8, d / 8, 8, 8)
        x = x.permute(0, 1, 2, 4, 3, 5).reshape(len(pages), case["kv_heads"], case["page"],
                                                case["dim"])
    return x.transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :length]


def exact(case, seed):
    s = prepare(case, seed)
    bt, ps, d, hk = s["bt"].cpu().numpy(), case["page"], case["dim"], case["kv_heads"]
    if case["op"] == "norm":
        pos, rot = s["pos"].cpu().numpy(), case["rotary"]
        turn = s["turn"].cpu().numpy() if s["turn"] is not None else pos[:, None]
        sec = _sections(case) or [rot // 2]
        ang = np.zeros((len(pos), rot // 2))
        for j in range(rot // 2):
            if case["order"] == "cyclic":
                axis = j % len(sec) if j // len(sec) < sec[j % len(sec)] else 0
            else:
                axis = next(a for a in range(len(sec)) if j < sum(sec[:a + 1]))
            power = j / (rot // 2)
            if case["order"] == "ladders":
                power = (j - sum(sec[:axis])) / sec[axis]
            ang[:, j] = turn[:, axis].astype(np.float64) * float(case["base"]) ** -power
        ang = torch.from_numpy(ang).cuda()
        z = torch.polar(torch.ones_like(ang), ang)[:, None]

        def turned(x, w):
            x = x.double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / d + _EPS).sqrt() * w.double()
            y = x[..., :rot]
            if case["neox"]:
                y = torch.complex(y[..., :rot // 2].contiguous(),
                                  y[..., rot // 2:].contiguous()) * z
                y = torch.cat([y.real, y.imag], dim=-1)
            else:
                y = torch.view_as_complex(y.unflatten(-1, (-1, 2)).contiguous()) * z
                y = torch.view_as_real(y).flatten(-2)
            return torch.cat([y, x[..., rot:]], dim=-1)

        k, v, rows = s["k"].double(), s["v"].double(), s["rows"].cpu().numpy()
        for buf, new in ((k, turned(s["kn"], s["kw"])), (v, s["vn"].double())):
            page = torch.from_numpy(bt[rows, pos // ps].astype(np.int64)).cuda()
            t = torch.from_numpy((pos % ps).astype(np.int64)).cuda()
            if case["dtype"] == "fp32":
                buf[0, page, :, t] = new
            else:
                for u in range(d // 8):
                    buf[0, page, :, t // 8, u, t % 8] = new[..., 8 * u:8 * u + 8]
        return turned(s["q"], s["qw"]), k, v
    if case["op"] == "shared":
        _, _, lens = _groups(case)
        if int(lens.sum()) * case["heads"] > 3e8:
            return None
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, n in enumerate(lens.tolist()):
            ki, vi = (_rows64(case, s[x], bt[i, :-(-n // ps)], n) for x in ("k", "v"))
            sc = torch.einsum("hgd,hld->hgl", s["q"][i].double().view(hk, -1, d), ki) * s["scale"]
            out[i] = torch.einsum("hgl,hld->hgd", torch.softmax(sc, dim=-1), vi).reshape(-1, d)
        return out
    if case["op"] == "weigh":
        ctx, new = _lengths(case)
        out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
        weights = s["weights"].double()
        for i in range(case["seqs"]):
            c, m = int(ctx[i]), int(new[i])
            ki, vi = (_rows64(case, s[x], bt[i, :-(-(c + m) // ps)], c + m) for x in ("k", "v"))
            sc = torch.einsum("mhgd,hld->hgml", s["q"][at:at + m].double().view(m, hk, -1, d), ki)
            late = torch.ones(m, c + m, dtype=torch.bool, device="cuda").triu(diagonal=c + 1)
            w = torch.softmax((sc * s["scale"]).masked_fill(late, -math.inf), dim=-1)
            out[at:at + m] = torch.einsum("hgml,hld->mhgd", w, vi).reshape(m, -1, d)
            weights[i, :, c:c + m] = 0.0
            weights[i, :, :c + m] += w.sum(dim=(1, 2))
            at += m
        return out, weights
    # rows move as they are: their own type holds them
    ctx, w = s["ctx"].cpu().numpy(), s["weights"].cpu().numpy()
    left, budget, recent = torch.zeros_like(s["left"], dtype=torch.float64), case["budget"], case["recent"]
    k0, v0 = s["k"], s["v"]
    k1, v1 = k0.clone(), v0.clone()
    for i, n in enumerate(ctx.tolist()):
        m = min(n, budget)
        if n > budget:
            old = n - recent
            best = np.argsort(-w[:, i, :, :old], axis=-1, kind="stable")[..., :budget - recent]
            tail = np.broadcast_to(np.arange(old, n), best.shape[:2] + (recent,))
            keep = np.sort(np.concatenate([best, tail], axis=-1), axis=-1)
        else:
            keep = np.broadcast_to(np.arange(n), w.shape[:1] + (hk, n))
        left[:, i, :, :m] = torch.from_numpy(np.take_along_axis(w[:, i], keep, -1).astype(
            np.float64)).cuda()
        if n <= budget:
            continue
        lay = torch.arange(w.shape[0], device="cuda")[:, None]
        z = torch.arange(m, device="cuda")[None]
        table = torch.from_numpy(bt[i].astype(np.int64)).cuda()
        for h in range(hk):
            a = torch.from_numpy(keep[:, h].astype(np.int64)).cuda()
            for old_buf, buf in ((k0, k1), (v0, v1)):
                if case["dtype"] == "fp32":
                    buf[lay, table[z // ps], h, z % ps] = old_buf[lay, table[a // ps], h, a % ps]
                else:
                    buf[lay, table[z // ps], h, z % ps // 8, :, z % 8] = \
                        old_buf[lay, table[a // ps], h, a % ps // 8, :, a % 8]
    return None, left, k1, v1
