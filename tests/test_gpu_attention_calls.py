"""GPU tests of the attention calls' arguments beyond shapes and types."""
from __future__ import annotations

import pytest
import torch

import attention_ref as ref
from test_gpu_attention import _paged, _randn, att  # noqa: F401  (att: a fixture)

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_a_mask_needs_max_tree_of_at_most_64(cuda_device, att):
    news, lens = [5], [70]
    k, v, table = _paged(1, lens, 2, 64, 16, BF16)
    q, mask = _randn(2, 5, 4, 64), torch.full((5,), 31, dtype=torch.int64, device="cuda")
    args = q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), ref.cumulative(news, cuda_device)
    for most in (65, 4096):
        with pytest.raises(ValueError, match="names 64 tokens"):
            att.tree_attention(*args, max_tree=most, tree_mask=mask)
        att.tree_attention(*args, max_tree=most)
    att.tree_attention(*args, max_tree=64, tree_mask=mask)
