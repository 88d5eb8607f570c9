"""Refusals of the attention entry points that need no GPU."""
from __future__ import annotations

import ctypes
import math
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


# --------------------------------------------------- yarn's magnitude and ends
YARN = dict(type="yarn", factor=40.0, original_max_position_embeddings=4096)


@pytest.mark.parametrize("more,want", [
    ({}, 0.1 * math.log(40) + 1), (dict(mscale=1.0), 0.1 * math.log(40) + 1), (dict(mscale=1.0, mscale_all_dim=1.0), 1.0),
    (dict(mscale=0.707, mscale_all_dim=1.0), (0.0707 * math.log(40) + 1) / (0.1 * math.log(40) + 1)),
    (dict(mscale=1.0, mscale_all_dim=0.5, attention_factor=1.25), 1.25), (dict(mscale=1.0, mscale_all_dim=0.5, factor=1.0), 1.0)])
def test_yarn_magnitude(more, want):
    from svdflash_b200.kernels import attention as att
    got = att.rope_frequencies(64, device="cpu", scaling={**YARN, **more})[1]
    assert got == pytest.approx(want, rel=1e-12)


@pytest.mark.parametrize("more", [dict(mscale=0.7), dict(mscale_all_dim=0.7), dict(mscale=0.7, mscale_all_dim=0), dict(mscale=0)])
def test_half_of_yarns_magnitude_is_refused(more):
    from svdflash_b200.kernels import attention as att
    with pytest.raises(ValueError, match="mscale"):
        att.rope_frequencies(64, device="cpu", scaling={**YARN, **more})


def test_yarn_between_its_ends():
    """The share of the stretched frequency grows evenly with the pair's index between the ends, whole pairs or not."""
    from svdflash_b200.kernels import attention as att
    half, base = 32, 10000.0
    ends = [half * math.log(4096 / (2 * math.pi * turns)) / math.log(base) for turns in (32, 1)]
    for more, (first, last) in (({}, (math.floor(ends[0]), math.ceil(ends[1]))), (dict(truncate=False), ends)):
        freq, _ = att.rope_frequencies(64, base=base, device="cpu", scaling={**YARN, **more})
        for i in range(half):
            plain = base ** (-i / half)
            share = min(1.0, max(0.0, (i - first) / (last - first)))
            assert freq[i].item() == pytest.approx(plain * (1 - share) + plain / 40 * share, rel=1e-6)
