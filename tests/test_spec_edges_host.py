"""Host side of the drafted-token and beam operators where it can go wrong (no GPU):
calls that are refused before any device work, and what the decoder remembers."""

from __future__ import annotations

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
