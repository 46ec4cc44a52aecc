"""Drafted tokens and beams through the layers: BatchDecoder.verify / commit / reorder
and the two generation loops on top of them, on the seeded model of
tests/golden/engine_model.py.

* A verified tree gives every node what decoding its branch token by token gives: the
  layers' own bound, 5e-3 * max(1, max|ref|) per layer (tests/test_gpu_layer_batch.py),
  times the model's two layers.  Rows appended by a step and by a verify come from
  projections of the same kernels, and only the rotation differs (32-bit against 64-bit
  angles): a few fp16 steps.
* After a commit, decoding goes on as if the path had been decoded token by token.
* Speculative generation yields greedy generation's tokens, whatever is drafted.
* A beam's score is the log probability of its tokens: recomputed from one prefill of
  the whole hypothesis, whose logits (fp16, values below 32) may differ by the layer bound
  and one fp16 step; two log softmax terms of it per token.
"""

from __future__ import annotations

import numpy as np
import pytest

from conftest import HAS_GPU

pytestmark = pytest.mark.gpu

if HAS_GPU:
    import torch

    import batch_generate as BG
    import kvcache_ffi as ffi
    import paged
    from test_gpu_batch_generate import _golden, _model

BOUND = 2 * 5e-3


@pytest.fixture
def gen(cuda_device):
    cfg, tensors = _model()
    g = BG.BatchGenerator(BG.BatchModel.from_tensors(cfg, tensors), max_batch=8, max_seq_len=64)
    yield g
    g.close()
    torch.cuda.synchronize()
    assert ffi.device_error(0, clear=True) == (0, 0)


def _x(gen, ids):
    return gen.model.embedding[torch.tensor(ids, dtype=torch.long, device="cuda")].contiguous()


def _close(a, b):
    a, b = a.float(), b.float()
    assert float((a - b).abs().max()) <= BOUND * max(1.0, float(b.abs().max()))


TREES = [[-1, 0, 0, 1, 1, 2, 3, 0], [], [-1, -1, 1]]
DRAFT = [[5, 9, 11, 3, 60, 7, 8, 2], [], [4, 30, 12]]
PROMPTS = [[3, 14, 15, 9, 2, 6, 5], [10, 20], [1] * 17]


def _prefilled(gen):
    dec = gen._decoder(gen.bt[:3].contiguous())
    for i, p in enumerate(PROMPTS):
        dec.prefill(i, _x(gen, p))
    return dec


def _branch(tree, j):
    path = []
    while j >= 0:
        path.append(j)
        j = tree[j]
    return path[::-1]


def test_verified_tree_and_committed_path_match_decoding(gen):
    dec = _prefilled(gen)
    h = dec.verify(_x(gen, sum(DRAFT, [])), TREES)
    assert list(dec.ctx) == [7, 2, 17]
    rows = {}
    for i in (0, 2):                      # every node's branch, decoded as a prompt of its own
        o = 0 if i == 0 else len(DRAFT[0])
        for j in range(len(TREES[i])):
            branch = _branch(TREES[i], j)
            one = gen._decoder(gen.bt[4:5].contiguous())
            want = one.prefill(0, _x(gen, PROMPTS[i] + [DRAFT[i][a] for a in branch]))
            rows[i, j] = [gen.pool.gather(l, gen.bt, 4, 0, len(PROMPTS[i]) + len(branch))
                          for l in range(2)]
            one.close()
            _close(h[o + j:o + j + 1], want[-1:])
    paths = [[0, 1, 3, 6], [], [1, 2]]
    dec.commit(paths)
    assert list(dec.ctx) == [11, 2, 19]
    for i, j in ((0, 6), (2, 2)):         # the cache holds the branch's rows, side by side
        for l in range(2):
            for got, want in zip(gen.pool.gather(l, gen.bt, i, 0, int(dec.ctx[i])), rows[i, j][l]):
                _close(got, want)
    nxt = dec.step(_x(gen, [1, 2, 3]))
    for i, ids in ((0, PROMPTS[0] + [5, 9, 3, 8, 1]), (1, PROMPTS[1] + [2]),
                   (2, PROMPTS[2] + [30, 12, 3])):
        one = gen._decoder(gen.bt[4:5].contiguous())
        _close(nxt[i:i + 1], one.prefill(0, _x(gen, ids))[-1:])
        one.close()
    dec.close()


def test_verify_and_commit_refuse_what_does_not_fit(gen):
    dec = _prefilled(gen)
    x = _x(gen, [1, 2])
    with pytest.raises(ValueError):
        dec.verify(x, [[-1, 0], []])
    with pytest.raises(ValueError):
        dec.verify(x, [[-1], [], []])
    with pytest.raises(ValueError):
        dec.verify(x, [[-1, 1], [], []])          # a parent that comes later
    with pytest.raises(IndexError):
        dec.verify(_x(gen, [1] * 60), [list(range(-1, 59)), [], []])
    with pytest.raises(RuntimeError):
        dec.commit([[], [], []])
    dec.verify(x, [[-1, 0], [], []])
    for bad in ([[0], []], [[1, 0], [], []], [[2], [], []], [[0], [0], []]):
        with pytest.raises(ValueError):
            dec.commit(bad)
    dec.commit([[0, 1], [], []])
    with pytest.raises(RuntimeError):
        dec.commit([[0, 1], [], []])              # a commit uses its verify up
    with pytest.raises(ValueError):
        dec.reorder([[0, 1, 2]])                  # rows of different lengths
    with pytest.raises(ValueError):
        dec.reorder([[0, 3, 1]])
    empty = dec.verify(_x(gen, []), [[], [], []])
    assert empty.shape[0] == 0
    dec.commit([[], [], []])
    dec.close()


@pytest.mark.parametrize("kind", ["right", "wrong", "mixed", "none"])
def test_speculative_generation_is_greedy_generation(gen, kind):
    meta, _ = _golden()
    want, _ = gen.generate_batch_ids(meta["prompts"], max_new_tokens=10, stop_on_eos=False)
    full = [list(p) + w for p, w in zip(meta["prompts"], want)]

    def drafter(i, ids):
        nxt = full[i][len(ids):len(ids) + 3]
        if kind == "none":
            return [], []
        if kind == "wrong":
            return [(t + 1) % 64 for t in nxt], list(range(-1, len(nxt) - 1))
        if kind == "right":
            return nxt, list(range(-1, len(nxt) - 1))
        # right and wrong siblings on every level
        toks, par, above = [], [], -1
        for t in nxt:
            toks += [(t + 7) % 64, t]
            par += [above, above]
            above = len(toks) - 1
        return toks, par

    got, m = gen.generate_speculative_ids(meta["prompts"], drafter, max_new_tokens=10,
                                          stop_on_eos=False)
    assert got == want
    assert m["steps"] == {"right": 3, "wrong": 9, "none": 9}.get(kind, m["steps"])
    if kind == "mixed":
        assert m["accepted"] > 0
    gen.model.cfg.eos_token_id = want[0][4]
    got, _ = gen.generate_speculative_ids(meta["prompts"], drafter, max_new_tokens=10)
    ref, _ = gen.generate_batch_ids(meta["prompts"], max_new_tokens=10)
    assert got == ref
    gen.model.cfg.eos_token_id = -1


def _logp(gen, prompt, ids):
    """Sum of the log probabilities of ids behind prompt, from one prefill, and its bound."""
    one = gen._decoder(gen.bt[7:8].contiguous())
    h = one.prefill(0, _x(gen, prompt + ids[:-1]))[len(prompt) - 1:]
    logits = gen._logits(h.contiguous(), torch.cuda.current_stream())
    one.close()
    lp = torch.log_softmax(logits.double(), dim=1)
    top = float(logits.float().abs().max())
    tol = 2 * len(ids) * (BOUND * max(1.0, top) + 2.0 ** -10 * max(1.0, top))
    return float(sum(lp[j, t] for j, t in enumerate(ids))), tol


def test_beam_search_scores_are_log_probabilities(gen):
    prompts = [PROMPTS[0], PROMPTS[2]]
    outs, scores = gen.generate_beam_ids(prompts, num_beams=3, max_new_tokens=20,
                                         length_penalty=0.0, stop_on_eos=False)
    greedy, _ = gen.generate_beam_ids(prompts, num_beams=1, max_new_tokens=20, length_penalty=0.0,
                                      stop_on_eos=False)
    plain, _ = gen.generate_batch_ids(prompts, max_new_tokens=20, stop_on_eos=False)
    assert greedy == plain                        # one beam is greedy decoding
    for p, ids, s in zip(prompts, outs, scores):
        assert len(ids) == 20
        lp, tol = _logp(gen, p, ids)
        assert abs(lp - s) <= tol
    again, s2 = gen.generate_beam_ids(prompts, num_beams=3, max_new_tokens=20, length_penalty=0.0,
                                      stop_on_eos=False)
    assert again == outs and s2 == scores         # the generator's own tables are as they were
    gen.model.cfg.eos_token_id = outs[0][2]
    ended, s3 = gen.generate_beam_ids(prompts, num_beams=3, max_new_tokens=20)
    for p, ids, s in zip(prompts, ended, s3):
        lp, tol = _logp(gen, p, ids)
        assert abs(lp / len(ids) - s) <= tol / len(ids)
    gen.model.cfg.eos_token_id = -1
    for bad in (dict(num_beams=0), dict(num_beams=17), dict(num_beams=5), dict(max_new_tokens=60)):
        with pytest.raises(ValueError):
            gen.generate_beam_ids(prompts, **{**dict(num_beams=2, max_new_tokens=4), **bad})


def test_reordered_beams_decode_like_their_own_sequences(gen):
    """Beams that swap, merge and split while their open pages fill up: every beam's cache
    is that of its own token sequence decoded alone."""
    rng = np.random.default_rng(0)
    k = 4
    dec = gen._decoder(gen.bt[:k].clone())
    prompt = [7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18, 19]
    dec.prefill(0, _x(gen, prompt))
    dec.ctx[:] = len(prompt)
    seqs = [list(prompt) for _ in range(k)]
    for step in range(24):
        par = np.zeros((1, k), dtype=np.int32) if step == 0 else rng.integers(0, k, (1, k))
        dec.reorder(par)
        toks = rng.integers(0, 64, k).tolist()
        seqs = [seqs[p] + [t] for p, t in zip(par[0], toks)]
        h = dec.step(_x(gen, toks))
    for b in range(k):
        one = gen._decoder(gen.bt[7:8].contiguous())
        want = one.prefill(0, _x(gen, seqs[b]))
        _close(h[b:b + 1], want[-1:])
        for l in range(2):
            for x, y in zip(gen.pool.gather(l, dec.bt, b, 0, len(seqs[b])),
                            gen.pool.gather(l, gen.bt, 7, 0, len(seqs[b]))):
                _close(x, y)
        one.close()
    dec.close()
