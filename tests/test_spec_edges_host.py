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
