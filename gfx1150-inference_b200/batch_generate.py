"""Batched generate_batch_ids on the paged pool.

The reference's ``LlamaInferenceEngine.generate_batch_ids``
(src/inference.py:415-457) serves a batch by running ``generate_ids`` for one
prompt after another: every token of every sequence is one pass over all layers
(``forward_layer_cached`` per layer, src/layer.py:221-263), then the final
RMSNorm and the LM head on the last position (src/inference.py:233-253) and the
sampler.  ``BatchGenerator`` produces the same tokens with every sequence of the
batch advancing together:

* each prompt is prefilled into its own block-table rows of one paged pool
  (``paged.BatchDecoder.prefill``, chunked like ``prefill_tokens`` when asked);
* then every decode step runs all sequences' next tokens through each layer in
  one ``kvc_forward_layer_paged`` call (``BatchDecoder.step``), the final RMSNorm
  (``kvc_rmsnorm``) and the LM head (``kvc_linear``) on the whole batch, and the
  sampler per sequence.

Greedy decoding (temperature 0, no repetition penalty) takes the argmax of each
sequence's fp16 logits, as ``sample_next_token`` does (src/inference.py:51-121).
Any other sampling goes through a caller-supplied ``sampler`` with that
function's signature (the reference's own ``sample_next_token``), fed each
sequence's logits on the host and a ``numpy`` generator seeded ``seed + i`` for
prompt i, exactly like the sequential loop.  A sequence that has stopped (EOS)
keeps riding along in the batch; its extra tokens are discarded.

Two loops have no counterpart in the reference: ``generate_speculative_ids`` verifies
a tree of drafted tokens per step and yields greedy decoding's tokens (up to rounding)
in fewer steps, and ``generate_beam_ids`` is beam search.
"""

from __future__ import annotations

import time
from dataclasses import dataclass
from typing import Callable, Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

import kvcache_ffi as ffi
import paged

# GGUF names of one layer's projections in forward_layer_cached's order
_PROJ = ["attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down"]
# GGML type ids the kernels take (KVC_WTYPE_*); F32 (0) is converted to F16
_F32, _F16 = 0, 1
_KERNEL_TYPES = {1, 2, 8, 12, 14}


@dataclass
class ModelConfig:
    layers: int
    hidden: int
    intermediate: int
    heads: int
    kv_heads: int
    head_dim: int
    vocab: int
    eps: float = 1e-5
    rope_base: float = 10000.0
    rope_neox: bool = False
    eos_token_id: int = -1


def _f16_rows(raw: np.ndarray, typ: int, n: int, k: int) -> np.ndarray:
    if typ == _F16:
        return np.frombuffer(memoryview(np.ascontiguousarray(raw)), dtype=np.float16).reshape(n, k)
    if typ == _F32:
        return np.frombuffer(memoryview(np.ascontiguousarray(raw)), dtype=np.float32).reshape(n, k).astype(np.float16)
    raise ValueError(f"GGML type {typ} is not a float table")


class BatchModel:
    """The weights generation needs, resident on one GPU: per layer the two norm
    weights and the seven GGML-typed projections (paged.DeviceLayerWeights), the
    token-embedding table as fp16 rows, the output norm and the LM head."""

    def __init__(self, cfg: ModelConfig, layers: List[paged.DeviceLayerWeights],
                 embedding: torch.Tensor, out_norm: torch.Tensor, head: torch.Tensor,
                 head_type: int, device: int):
        self.cfg, self.layers, self.embedding = cfg, layers, embedding
        self.out_norm, self.head, self.head_type, self.device = out_norm, head, head_type, device

    @classmethod
    def from_tensors(cls, cfg: ModelConfig, tensors: Dict[str, Tuple[np.ndarray, int, tuple]],
                     embedding: Optional[np.ndarray] = None, device: int = 0) -> "BatchModel":
        """tensors: GGUF name -> (raw bytes, GGML type id, (n, k) row-major shape),
        the layout of a llama GGUF file (``token_embd.weight``, ``blk.{l}.*``,
        ``output_norm.weight``, ``output.weight``, or the tied embedding).  The
        embedding table is given as fp16 rows when ``token_embd.weight`` is
        quantized (the reference dequantizes rows with its own code)."""
        dev = torch.device("cuda", device)

        def to_dev(a: np.ndarray) -> torch.Tensor:
            return torch.from_numpy(np.ascontiguousarray(a)).to(dev)

        def weight(name: str):
            raw, typ, shape = tensors[name]
            n, k = shape
            if typ == _F32:
                raw, typ = _f16_rows(raw, typ, n, k).view(np.uint8).reshape(-1), _F16
            if typ not in _KERNEL_TYPES:
                raise ValueError(f"{name}: GGML type {typ} is not supported by the kernels")
            return to_dev(np.frombuffer(memoryview(np.ascontiguousarray(raw)), dtype=np.uint8)), typ

        def norm(name: str) -> torch.Tensor:
            raw, typ, shape = tensors[name]
            return to_dev(_f16_rows(raw, typ, 1, cfg.hidden).reshape(-1))

        layers = []
        for l in range(cfg.layers):
            p = f"blk.{l}."
            ws = [weight(p + n + ".weight") for n in _PROJ]
            layers.append(paged.DeviceLayerWeights(norm(p + "attn_norm.weight"),
                                                   norm(p + "ffn_norm.weight"),
                                                   [w for w, _ in ws], [t for _, t in ws],
                                                   cfg.hidden, cfg.intermediate))
        if embedding is None:
            raw, typ, shape = tensors["token_embd.weight"]
            embedding = _f16_rows(raw, typ, shape[0], shape[1])
        if embedding.shape != (cfg.vocab, cfg.hidden):
            raise ValueError(f"the embedding table is {embedding.shape}, expected "
                             f"({cfg.vocab}, {cfg.hidden})")
        head_name = "output.weight" if "output.weight" in tensors else "token_embd.weight"
        head, head_type = weight(head_name)
        if cfg.vocab % 16:
            raise ValueError("the LM head kernel needs a vocabulary that is a multiple of 16")
        return cls(cfg, layers, to_dev(np.asarray(embedding, np.float16)),
                   norm("output_norm.weight"), head, head_type, device)

    @classmethod
    def from_reference_engine(cls, engine, device: int = 0) -> "BatchModel":
        """The weights of a gfx1150-inference ``LlamaInferenceEngine`` moved to the
        GPU once (see ``tensors_from_reference_engine``)."""
        cfg, tensors, embedding = tensors_from_reference_engine(engine)
        return cls.from_tensors(cfg, tensors, embedding=embedding, device=device)


def tensors_from_reference_engine(engine):
    """(ModelConfig, tensors, embedding rows) of a gfx1150-inference
    ``LlamaInferenceEngine``: its layer configuration (LlamaLayerConfig), every
    tensor of its GGUF file read through its WeightStreamer, and the token
    embedding dequantized row by row with the engine's own ``embed_tokens``
    (src/tokenizer.py:336).  Host memory only."""
    import sys

    lc = engine.layer_cfg
    gg = engine.streamer.gguf
    tensors = {}
    for name, info in gg.tensors.items():
        view = np.array(engine.streamer.get_tensor_view(name), copy=True)
        shape = tuple(int(d) for d in info.shape_row_major)
        tensors[name] = (view.view(np.uint8).reshape(-1), int(info.ggml_type), shape)
    mod = sys.modules[type(engine).__module__]
    emb_info = gg.tensors["token_embd.weight"]
    vocab = int(emb_info.shape_row_major[0])
    embedding = mod.embed_tokens(list(range(vocab)), emb_info,
                                 engine.streamer.get_tensor_view("token_embd.weight"),
                                 lc.hidden_size)
    tok = getattr(engine, "tokenizer", None)
    cfg = ModelConfig(layers=int(engine.num_layers), hidden=lc.hidden_size,
                      intermediate=lc.intermediate_size, heads=lc.num_heads,
                      kv_heads=lc.num_kv_heads, head_dim=lc.head_dim, vocab=vocab,
                      eps=float(lc.rms_norm_eps), rope_base=float(lc.rope_freq_base),
                      rope_neox=bool(lc.rope_neox),
                      eos_token_id=int(tok.eos_token_id) if tok is not None else -1)
    return cfg, tensors, np.asarray(embedding, np.float16)


class BatchGenerator:
    """generate_batch_ids for a batch of up to ``max_batch`` prompts of up to
    ``max_seq_len`` positions (prompt + new tokens), on one paged pool."""

    def __init__(self, model: BatchModel, max_batch: int, max_seq_len: int, page_size: int = 16):
        cfg = model.cfg
        self.model, self.max_batch, self.max_seq_len = model, int(max_batch), int(max_seq_len)
        self.pages_per_seq = (self.max_seq_len + page_size - 1) // page_size
        self.pool = paged.PagedKVCache(cfg.layers, self.max_batch * self.pages_per_seq, page_size,
                                       cfg.kv_heads, cfg.head_dim, dtype=torch.float16,
                                       device=model.device)
        table = np.arange(self.max_batch * self.pages_per_seq, dtype=np.int32)
        self.bt = torch.from_numpy(table.reshape(self.max_batch, self.pages_per_seq)).to(
            torch.device("cuda", model.device))

    def _logits(self, h: torch.Tensor, stream) -> torch.Tensor:
        """Final RMSNorm and LM head of rows h (m, hidden) -> fp16 logits (m, vocab)."""
        m = self.model
        n = int(h.shape[0])
        normed = torch.empty_like(h)
        sp = int(stream.cuda_stream) or None
        ffi.check(ffi.lib.kvc_rmsnorm(int(h.data_ptr()), None, None, int(m.out_norm.data_ptr()),
                                      int(normed.data_ptr()), n, m.cfg.hidden, float(m.cfg.eps),
                                      sp))
        logits = torch.empty((n, m.cfg.vocab), dtype=torch.float16, device=h.device)
        ffi.check(ffi.lib.kvc_linear(int(normed.data_ptr()), n, m.cfg.hidden,
                                     int(m.head.data_ptr()), m.head_type, m.cfg.vocab,
                                     int(logits.data_ptr()), sp))
        return logits

    def generate_batch_ids(
        self,
        batch_prompt_ids: Sequence[Sequence[int]],
        max_new_tokens: int = 16,
        temperature: float = 0.0,
        top_k: int = 40,
        top_p: float = 0.95,
        repetition_penalty: float = 1.0,
        stop_on_eos: bool = True,
        seed: Optional[int] = 42,
        prefill_chunk_size: Optional[int] = None,
        sampler: Optional[Callable] = None,
    ) -> Tuple[List[List[int]], Dict[str, float]]:
        """The arguments and result of the reference's generate_batch_ids
        (src/inference.py:415-457): the generated ids of each prompt and batch
        metrics.  ``sampler`` (the reference's sample_next_token) is required
        unless decoding is greedy (temperature 0, repetition penalty 1)."""
        cfg = self.model.cfg
        prompts = [[int(t) for t in p] for p in batch_prompt_ids]
        b = len(prompts)
        if b > self.max_batch:
            raise ValueError(f"{b} prompts exceed the generator's max_batch {self.max_batch}")
        if max_new_tokens < 0:
            raise ValueError(f"max_new_tokens must be >= 0 (got {max_new_tokens})")
        for p in prompts:
            if not p:
                raise ValueError("prompt_ids must not be empty")
            if len(p) + max_new_tokens > self.max_seq_len:
                raise ValueError(f"len(prompt_ids) ({len(p)}) + max_new_tokens ({max_new_tokens}) "
                                 f"exceeds max_seq_len ({self.max_seq_len})")
            if min(p) < 0 or max(p) >= cfg.vocab:
                raise ValueError("a token id is outside the vocabulary")
        greedy = (temperature == 0.0 or top_k == 1) and repetition_penalty == 1.0
        if not greedy and sampler is None:
            raise ValueError("non-greedy decoding needs sampler= (e.g. the reference's "
                             "sample_next_token)")
        t0 = time.perf_counter()
        outs: List[List[int]] = [[] for _ in range(b)]
        if b == 0 or max_new_tokens == 0:
            return outs, {"batch_size": float(b), "total_tokens_generated": 0.0,
                          "total_time_s": 0.0, "tokens_per_sec": 0.0}
        stream = torch.cuda.current_stream(self.model.device)
        rngs = [np.random.default_rng(None if seed is None else seed + i) for i in range(b)]
        hist = [list(p) for p in prompts]
        dec = paged.BatchDecoder(self.pool, self.model.layers, self.bt[:b].contiguous(),
                                 cfg.heads, [0] * b, eps=cfg.eps, freq_base=cfg.rope_base,
                                 neox=cfg.rope_neox)
        emb = self.model.embedding

        def pick(logits: torch.Tensor) -> List[int]:
            if greedy:
                return [int(t) for t in torch.argmax(logits.float(), dim=1).tolist()]
            host = logits.cpu().numpy()
            return [int(sampler(host[i], temperature=temperature, top_k=top_k, top_p=top_p,
                                repetition_penalty=repetition_penalty, generated_ids=hist[i],
                                rng=rngs[i])) for i in range(b)]

        try:
            last = []
            for i, p in enumerate(prompts):  # prefill, full or chunked (prefill_tokens)
                ids = torch.tensor(p, dtype=torch.long, device=emb.device)
                step = len(p) if not prefill_chunk_size or prefill_chunk_size <= 0 else prefill_chunk_size
                for s0 in range(0, len(p), step):
                    h = dec.prefill(i, emb[ids[s0:s0 + step]].contiguous(), stream=stream)
                last.append(h[-1:])
            nxt = pick(self._logits(torch.cat(last), stream))
            done = [False] * b
            for i in range(b):
                outs[i].append(nxt[i])
                hist[i].append(nxt[i])
            for _ in range(max_new_tokens - 1):
                for i in range(b):
                    if stop_on_eos and outs[i][-1] == cfg.eos_token_id:
                        done[i] = True
                if all(done):
                    break
                ids = torch.tensor([o[-1] for o in outs], dtype=torch.long, device=emb.device)
                h = dec.step(emb[ids].contiguous(), stream=stream)
                nxt = pick(self._logits(h, stream))
                for i in range(b):
                    if not done[i]:
                        outs[i].append(nxt[i])
                        hist[i].append(nxt[i])
        finally:
            dec.close()
        t = time.perf_counter() - t0
        total = float(sum(len(o) for o in outs))
        return outs, {"batch_size": float(b), "total_tokens_generated": total,
                      "total_time_s": t, "tokens_per_sec": total / max(t, 1e-9)}

    def _check_prompts(self, batch_prompt_ids, rows: int, max_new_tokens: int) -> List[List[int]]:
        prompts = [[int(t) for t in p] for p in batch_prompt_ids]
        if len(prompts) * rows > self.max_batch:
            raise ValueError(f"{len(prompts)} prompts of {rows} rows exceed the generator's "
                             f"max_batch {self.max_batch}")
        if max_new_tokens < 0:
            raise ValueError(f"max_new_tokens must be >= 0 (got {max_new_tokens})")
        for p in prompts:
            if not p:
                raise ValueError("prompt_ids must not be empty")
            if len(p) + max_new_tokens > self.max_seq_len:
                raise ValueError(f"len(prompt_ids) ({len(p)}) + max_new_tokens ({max_new_tokens}) "
                                 f"exceeds max_seq_len ({self.max_seq_len})")
            if min(p) < 0 or max(p) >= self.model.cfg.vocab:
                raise ValueError("a token id is outside the vocabulary")
        return prompts

    def _decoder(self, bt: torch.Tensor) -> paged.BatchDecoder:
        cfg = self.model.cfg
        return paged.BatchDecoder(self.pool, self.model.layers, bt, cfg.heads,
                                  [0] * int(bt.shape[0]), eps=cfg.eps, freq_base=cfg.rope_base,
                                  neox=cfg.rope_neox)

    def generate_speculative_ids(
        self,
        batch_prompt_ids: Sequence[Sequence[int]],
        drafter: Callable[[int, List[int]], Tuple[Sequence[int], Sequence[int]]],
        max_new_tokens: int = 16,
        stop_on_eos: bool = True,
    ) -> Tuple[List[List[int]], Dict[str, float]]:
        """Greedy generation that verifies drafted tokens, several per step.
        ``drafter(i, ids)`` is given prompt i's ids so far and returns (tokens, parents) of
        a drafted tree: parents[j] is the node above token j, smaller than j, or -1 for
        a token right behind the ids; empty for no draft.  Every step runs the last
        token and its draft through the layers at once (``BatchDecoder.verify``), follows
        the drafted tokens that are the argmax of the node above them, keeps that path
        (``commit``) and adds the argmax behind it: the ids are those of greedy decoding
        whatever is drafted, up to rounding.  (Several tokens of a step are rotated by angles of
        64 bits where single ones have the reference's 32, and their sums run in another
        order, so where two logits are within a few fp16 steps the other may win.)
        Metrics count the steps and the drafted and accepted tokens."""
        cfg = self.model.cfg
        prompts = self._check_prompts(batch_prompt_ids, 1, max_new_tokens)
        b = len(prompts)
        t0 = time.perf_counter()
        outs: List[List[int]] = [[] for _ in range(b)]
        stats = {"batch_size": float(b), "steps": 0.0, "drafted": 0.0, "accepted": 0.0}
        if b and max_new_tokens:
            stream = torch.cuda.current_stream(self.model.device)
            dec = self._decoder(self.bt[:b].contiguous())
            emb = self.model.embedding
            try:
                last = []
                for i, p in enumerate(prompts):
                    ids = torch.tensor(p, dtype=torch.long, device=emb.device)
                    last.append(dec.prefill(i, emb[ids].contiguous(), stream=stream)[-1:])
                first = torch.argmax(self._logits(torch.cat(last), stream).float(), dim=1).tolist()
                for i in range(b):
                    outs[i].append(int(first[i]))

                def done(i: int) -> bool:
                    return len(outs[i]) >= max_new_tokens or (
                        stop_on_eos and outs[i][-1] == cfg.eos_token_id)

                while not all(done(i) for i in range(b)):
                    tokens, trees = [], []
                    for i in range(b):
                        if done(i):
                            trees.append([])
                            continue
                        # node 0 is the last token, whose row is not cached yet
                        toks, par = drafter(i, prompts[i] + outs[i])
                        # a path of k tokens yields k + 1, and the cache holds all but the last
                        room = min(max_new_tokens - len(outs[i]) - 1,
                                   self.max_seq_len - int(dec.ctx[i]) - 1,
                                   ffi.MAX_TREE_NODES - 1)
                        if len(toks) != len(par):
                            raise ValueError("the draft needs one parent per token")
                        toks, par = [int(t) for t in toks][:room], [int(q) for q in par][:room]
                        if any(not 0 <= t < cfg.vocab for t in toks):
                            raise ValueError("a drafted token id is outside the vocabulary")
                        tokens += [outs[i][-1]] + toks
                        trees.append([-1] + [q + 1 for q in par])
                        stats["drafted"] += len(toks)
                    ids = torch.tensor(tokens, dtype=torch.long, device=emb.device)
                    h = dec.verify(emb[ids].contiguous(), trees, stream=stream)
                    best = torch.argmax(self._logits(h, stream).float(), dim=1).tolist()
                    paths, o = [], 0
                    for i, tree in enumerate(trees):
                        path, at = [], 0
                        if tree:
                            path, new = [0], []
                            while True:
                                new.append(int(best[o + at]))
                                nxt = [j for j in range(at + 1, len(tree))
                                       if tree[j] == at and tokens[o + j] == new[-1]]
                                if not nxt or (stop_on_eos and new[-1] == cfg.eos_token_id):
                                    break
                                at = nxt[0]
                                path.append(at)
                            outs[i] += new
                            stats["accepted"] += len(path) - 1
                        paths.append(path)
                        o += len(tree)
                    dec.commit(paths, stream=stream)
                    stats["steps"] += 1
            finally:
                dec.close()
        t = time.perf_counter() - t0
        total = float(sum(len(o) for o in outs))
        stats.update(total_tokens_generated=total, total_time_s=t, tokens_per_sec=total / max(t, 1e-9))
        return outs, stats

    def generate_beam_ids(
        self,
        batch_prompt_ids: Sequence[Sequence[int]],
        num_beams: int = 4,
        max_new_tokens: int = 16,
        length_penalty: float = 1.0,
        stop_on_eos: bool = True,
    ) -> Tuple[List[List[int]], List[float]]:
        """Beam search: for each prompt the ids of the best of ``num_beams`` beams and its
        score, the sum of its tokens' log probabilities over len ** length_penalty.  Each
        beam is a row of the batch (max_batch >= prompts * num_beams); every step picks
        the continuations on the GPU (``beam.BeamSelector``) and lets the beams' cached
        states follow their parents (``BatchDecoder.reorder``).  A prompt ends when
        num_beams of its hypotheses have ended, or at max_new_tokens."""
        import beam

        cfg, k = self.model.cfg, int(num_beams)
        if not 1 <= k <= ffi.MAX_BEAMS:
            raise ValueError(f"num_beams must be in [1, {ffi.MAX_BEAMS}]")
        if cfg.vocab < 2 * k:
            raise ValueError("the vocabulary is smaller than two beams' continuations")
        prompts = self._check_prompts(batch_prompt_ids, k, max_new_tokens)
        n = len(prompts)
        if n == 0 or max_new_tokens == 0:
            return [[] for _ in prompts], [0.0] * n
        stream = torch.cuda.current_stream(self.model.device)
        emb = self.model.embedding
        dec = self._decoder(self.bt[:n * k].clone())      # (reorder permutes the table)
        sel = beam.BeamSelector(n, k, cfg.vocab, 2 * k, device=self.model.device)
        ended: List[List[Tuple[float, List[int]]]] = [[] for _ in range(n)]
        live: List[List[List[int]]] = [[[] for _ in range(k)] for _ in range(n)]

        def norm(score: float, length: int) -> float:
            return score / length ** length_penalty

        try:
            last = []
            for i, p in enumerate(prompts):     # the prompt goes into the first beam's row
                ids = torch.tensor(p, dtype=torch.long, device=emb.device)
                h = dec.prefill(i * k, emb[ids].contiguous(), stream=stream)[-1:]
                dec.ctx[i * k:(i + 1) * k] = len(p)
                last.append(h.expand(k, -1))
            h = torch.cat(last).contiguous()
            scores = torch.full((n, k), -float("inf"), device=emb.device)
            scores[:, 0] = 0.0
            for step in range(max_new_tokens):
                tok, par, best = sel.select(self._logits(h, stream), scores, 2 * k, stream=stream)
                tok, par, best = tok.tolist(), par.tolist(), best.tolist()
                parents = np.zeros((n, k), dtype=np.int32)
                nxt = np.zeros((n, k), dtype=np.int64)
                run = np.full((n, k), -np.inf, dtype=np.float32)
                for i in range(n):
                    if len(ended[i]) >= k:      # finished: rides along
                        parents[i] = np.arange(k)
                        continue
                    grown = []
                    for rank in range(2 * k):
                        ids = live[i][par[i][rank]] + [tok[i][rank]]
                        if stop_on_eos and tok[i][rank] == cfg.eos_token_id:
                            if rank < k:
                                ended[i].append((norm(best[i][rank], len(ids)), ids))
                        elif len(grown) < k:
                            j = len(grown)
                            parents[i, j], nxt[i, j] = par[i][rank], tok[i][rank]
                            run[i, j] = best[i][rank]
                            grown.append(ids)
                    live[i] = grown
                if step + 1 == max_new_tokens or all(len(e) >= k for e in ended):
                    break
                dec.reorder(parents, stream=stream)
                scores = torch.from_numpy(run).to(emb.device)
                ids = torch.from_numpy(nxt.reshape(-1)).to(emb.device)
                h = dec.step(emb[ids].contiguous(), stream=stream)
        finally:
            dec.close()
            sel.close()
        outs, finals = [], []
        for i in range(n):
            hyps = list(ended[i])
            if len(hyps) < k:
                hyps += [(norm(float(run[i, j]), len(ids)), ids) for j, ids in enumerate(live[i])
                         if np.isfinite(run[i, j])]
            score, ids = max(hyps, key=lambda x: x[0])
            outs.append(ids)
            finals.append(score)
        return outs, finals

    def close(self):
        self.pool.close()
