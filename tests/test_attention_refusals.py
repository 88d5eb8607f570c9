"""Refusals of the attention entry points that need no GPU."""
from __future__ import annotations

import ctypes
import random

import pytest
import torch

from test_attention_validation import ENTRY, GOOD, PTR, SHAPE, _structs, lib  # noqa: F401  (lib: a fixture)


@pytest.mark.parametrize("max_tree", [65, 1 << 20])
def test_a_masked_tree_has_at_most_64_tokens(lib, max_tree):
    mirror, _ = _structs()["tree"]
    args = mirror(**{**GOOD["tree"], "mask": PTR, "max_tree": max_tree})
    assert getattr(lib, ENTRY["tree"])(ctypes.addressof(args), None) == SHAPE


# ------------------------------------------------- out apart from the inputs
def _places(t):
    at = t.storage_offset() + sum(torch.arange(n).view([-1 if d == i else 1 for i in range(3)]) * s
                                  for d, (n, s) in enumerate(zip(t.shape, t.stride())))
    return set(at.flatten().tolist())


def test_overlaps_are_found_place_by_place():
    from svdflash_b200.kernels.attention import _overlap
    rng = random.Random(5)
    buffer = torch.zeros(4000)
    found = []
    for _ in range(4000):
        views = []
        for _ in range(2):
            n, h, d = rng.randrange(1, 5), rng.randrange(1, 4), rng.choice([4, 8])
            token, head = rng.choice([8, 16, 24, 32, 64, 72, 100]), rng.choice([4, 8, 12, 16, 24, 64, 200])
            views.append(buffer.as_strided((n, h, d), (token, head, 1), rng.choice([0, 4, 8, 16, 24, 40, 100, 300])))
        want = bool(_places(views[0]) & _places(views[1]))
        assert _overlap(*views) == _overlap(*views[::-1]) == want, [(v.shape, v.stride(), v.storage_offset()) for v in views]
        found.append(want)
    assert 0.2 < sum(found) / len(found) < 0.8


def test_overlaps_of_usual_layouts_need_no_search(monkeypatch):
    from svdflash_b200.kernels import attention
    qkv = torch.zeros(300, 6, 8)
    heads_first = torch.zeros(6, 300, 8).transpose(0, 1)
    blocks = torch.zeros(20, 2, 64)
    monkeypatch.setattr(attention.torch, "arange", None)     # the search would call it
    for a, b in [(qkv[:, :4], qkv[:, 4:]), (qkv[:, 4:], qkv[:, :4]), (qkv[:, ::2], qkv[:, 1::2]), (qkv[:100], qkv[100:]),
                 (heads_first[:, :4], heads_first[:, 4:]), (heads_first[:, ::2], heads_first[:, 1::2]),
                 (qkv, torch.zeros(300, 6, 8)), (blocks[:, :1], blocks[:, 1:])]:
        assert not attention._overlap(a, b)
