"""Beam search's selection on the GPU (kvc_beam_select of libkvcache.so).

A step of beam search over the paged pool: ``BeamSelector.select`` picks the best
continuations of each sequence from its beams' logits, and
``paged.PagedKVCache.reorder_beams`` lets the cached states follow their parents.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

import kvcache_ffi as ffi
from paged import _TORCH_CODE, _made_on, _on, _stream_on


class BeamSelector:
    """Workspace and calls of the selection, for up to ``max_seqs`` sequences of up to
    ``max_beams`` beams over ``vocab`` tokens with up to ``max_out`` results each.
    Calls of one selector must be ordered on one stream."""

    def __init__(self, max_seqs: int, max_beams: int, vocab: int, max_out: int, device: int = 0):
        h = ctypes.c_void_p()
        ffi.check(ffi.lib.kvc_beam_create(int(max_seqs), int(max_beams), int(vocab), int(max_out),
                                          int(device), ctypes.byref(h)))
        self.handle = h
        self.device = int(device)

    def select(self, logits: torch.Tensor, scores: torch.Tensor, n_out: int,
               out: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None, stream=None
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """The ``n_out`` best (beam, token) pairs of each sequence by scores[seq, beam] +
        log softmax(logits)[token], best first; equal scores go to the lower beam, then
        the lower token.  Scores are within 2^-17 (and their rounding), so candidates of
        different beams less than 2^-16 apart may change places.  logits: (sequences *
        beams, vocab) fp16, bf16 or fp32, rows may be strided; scores: (sequences, beams)
        fp32, -inf for a beam not in use.  Returns (tokens int32, parents int32, scores
        fp32), each (sequences, n_out)."""
        dev = self.device
        code = _TORCH_CODE.get(logits.dtype)
        if code is None:
            raise ValueError(f"unsupported dtype {logits.dtype}")
        if scores.dim() != 2 or logits.dim() != 2:
            raise ValueError("logits and scores must have two dimensions")
        n, beams = scores.shape
        vocab = logits.shape[1]
        if logits.shape[0] != n * beams:
            raise ValueError("logits needs one row per beam")
        if logits.get_device() != dev:
            raise ValueError(f"logits must be on cuda:{dev}")
        st = logits.stride()
        if (vocab > 1 and st[1] != 1) or (n * beams > 1 and st[0] < vocab):
            raise ValueError("a row of logits must be packed")
        if out is None:
            with _made_on(stream, dev):
                tokens = torch.empty((n, n_out), dtype=torch.int32, device=logits.device)
                out = (tokens, torch.empty_like(tokens),
                       torch.empty((n, n_out), dtype=torch.float32, device=logits.device))
        tokens, parents, best = out
        m = n * n_out
        ffi.check(ffi.lib.kvc_beam_select(
            self.handle, logits.data_ptr(), code, st[0] if n * beams > 1 else vocab,
            _on(scores, "scores", torch.float32, 0, dev), n, beams, vocab, n_out,
            _on(tokens, "tokens", torch.int32, m, dev),
            _on(parents, "parents", torch.int32, m, dev),
            _on(best, "scores out", torch.float32, m, dev), _stream_on(stream, dev)))
        return out

    def close(self):
        if self.handle is not None:
            ffi.check(ffi.lib.kvc_beam_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
