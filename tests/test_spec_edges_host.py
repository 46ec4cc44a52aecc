"""Host side of the drafted-token and beam operators where it can go wrong (no GPU):
calls that are refused before any device work, and what the decoder remembers."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import paged
from test_spec_host import _pool


def test_a_mask_without_words_is_not_a_chain():
    pool, plan = _pool(), paged.TreePlan()
    plan.n_tokens, plan.num_heads = 3, 4
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    bt = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="word"):
        pool.decode_tree(plan, 0, q, torch.zeros(3, 0, dtype=torch.int32), q, bt, 0.1)
    plan.close()


class _Elsewhere:
    """A weight on another GPU."""
    is_cuda = True

    def is_contiguous(self):
        return True

    def get_device(self):
        return 1

    def data_ptr(self):
        return 256


def test_layer_weights_on_another_device_are_refused():
    pool, plan = _pool(), paged.TreePlan()
    plan.n_tokens, plan.num_heads = 1, 4
    x = torch.zeros(1, 256, dtype=torch.float16)
    lw = paged.DeviceLayerWeights(x[0], x[0], [_Elsewhere()] * 7, [1] * 7, 256, 512)
    with pytest.raises(ValueError, match="weights"):
        pool.forward_layer_tree(plan, 0, x, x, lw, None, torch.zeros(1, 4, dtype=torch.int32))
    plan.close()


class _Cache:
    """Takes a decoder's calls and remembers the streams that they name."""
    num_layers, page_size = 2, 16

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name not in ("plan", "plan_tree", "forward_layer", "forward_layer_tree", "commit_tree",
                        "reorder_beams"):
            raise AttributeError(name)

        def call(*args, **kw):
            self.calls.append((name, kw.get("stream", args[-1] if args else None)))
            return paged.TreePlan() if name == "plan_tree" else None
        return call


def _decoder(rows=3, ctx=10):
    return paged.BatchDecoder(_Cache(), [object(), object()], torch.zeros((rows, 4), dtype=torch.int32),
                              8, [ctx] * rows)


def test_what_a_decoder_makes_belongs_to_the_stream_it_is_given(monkeypatch):
    """The allocator may hand memory of the current stream to another tensor as soon as the
    call has returned, so nothing that the kernels on `stream` use is made elsewhere."""
    state = {"on": None}
    made = []

    class On:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            state["on"] = self.stream

        def __exit__(self, *_):
            state["on"] = None

    class Stream:
        cuda_stream = 77

    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda ptr, device=None: ("stream", ptr))
    monkeypatch.setattr(torch.cuda, "stream", On)
    for name in ("from_numpy", "empty_like"):
        real = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, _real=real, _name=name, **k: (
            made.append((_name, state["on"])), _real(*a, **k))[1])
    dec, s = _decoder(), Stream()
    x = torch.zeros((3, 16), dtype=torch.float16)
    dec.verify(x, [[-1], [-1], [-1]], stream=s)
    dec.commit([[0], [0], [0]], stream=s)
    dec.reorder([[1, 1, 2]], stream=s)
    dec.step(x, stream=s)
    dec.prefill(0, x, stream=s)
    assert {n for n, _ in made} == {"from_numpy", "empty_like"} and len(made) >= 13
    assert all(on == ("stream", 77) for _, on in made)
    assert all(at is s for _, at in dec.cache.calls) and len(dec.cache.calls) == 11
    made.clear()
    dec.verify(x, [[-1], [-1], [-1]])          # none given: the current stream
    assert made and all(on is None for _, on in made)
    dec.close()


def test_a_reorder_drops_the_verify_before_it():
    """Only cached positions follow their parents: the drafted rows behind them stay, and a
    commit would keep another beam's."""
    dec = _decoder()
    x = torch.zeros((6, 16), dtype=torch.float16)
    dec.verify(x, [[-1, 0]] * 3)
    dec.reorder([[1, 2, 0]])
    with pytest.raises(RuntimeError, match="verify"):
        dec.commit([[0, 1]] * 3)
    assert list(dec.ctx) == [10] * 3
    dec.verify(x, [[-1, 0]] * 3)
    with pytest.raises(ValueError):
        dec.reorder([[1, 2, 3]])              # refused: nothing moved, the verify stands
    dec.commit([[0, 1], [0], []])
    assert list(dec.ctx) == [12, 11, 10]
    dec.close()


@pytest.mark.parametrize("apart", [2 ** 31, 2 ** 32, 2 ** 32 + 512])
def test_tokens_too_far_apart_are_refused(apart):
    """2^32 would arrive as 0 (packed rows), 2^32 + 512 as 512."""
    t = torch.empty(apart + 128, dtype=torch.float16, device="meta").as_strided((2, 2, 64), (apart, 64, 1))
    with pytest.raises(ValueError, match="apart"):
        paged._token_rows(t, "q", torch.float16, (2, 2, 64), t.get_device())
    near = t.as_strided((2, 2, 64), (2 ** 31 - 8, 64, 1))
    assert paged._token_rows(near, "q", torch.float16, (2, 2, 64), t.get_device())[1] == 2 ** 31 - 8
    assert paged._token_rows(t[:1], "q", torch.float16, (1, 2, 64), t.get_device())[1] == 128


@pytest.mark.parametrize("kind", [list, lambda a: np.array(a, dtype=np.int64)])
def test_lengths_past_32_bits_are_refused(kind):
    """2^32 + 5 cached positions are not 5."""
    pool = _pool()
    for args in (([2 ** 32 + 5], [3]), ([5], [2 ** 32 + 3]), ([2 ** 31], [1])):
        with pytest.raises(ValueError, match="32 bits"):
            pool.plan_tree(kind(args[0]), kind(args[1]), 4)
    with pytest.raises(ValueError, match="32 bits"):
        pool.plan_tree([5], [3], 4, rows=kind([2 ** 32]))


def test_reorder_takes_the_decoder_s_rows_of_a_longer_table():
    seen = []

    class Cache(_Cache):
        def reorder_beams(self, table, parents, lens, stream=None):
            seen.append((table.data_ptr(), table.shape, parents.tolist(), lens.tolist()))

    bt = torch.zeros((6, 4), dtype=torch.int32)
    dec = paged.BatchDecoder(Cache(), [object(), object()], bt, 8, [10, 10, 7, 7])
    dec.reorder([[1, 0], [1, 1]])
    assert seen == [(bt.data_ptr(), (4, 4), [[1, 0], [1, 1]], [10, 7])]
    dec.close()
