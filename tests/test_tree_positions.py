"""Positions of drafted trees from a paging step's successive ones (torch expressions: no GPU needed)."""
from __future__ import annotations

import random

import pytest
import torch


def _step(held, news, extra):
    from svdflash_b200.kernels.attention import PageStep
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    positions = [h + i for h, n in zip(held, news) for i in range(n)] + [0] * extra

    def ints(x):
        return torch.tensor(x, dtype=torch.int32)
    return PageStep(torch.zeros(len(positions), dtype=torch.int64), ints(positions), ints(cu),
                    ints([h + n for h, n in zip(held, news)]), ints([5]), ints([0]))


def _signed(bits):
    return bits - (1 << 64) if bits >> 63 else bits


@pytest.mark.parametrize("held,news,extra", [
    ([0], [1], 0), ([40], [6], 0), ([7, 0, 1000], [64, 0, 26], 0), ([0, 3], [0, 5], 9), ([9] * 5, [0, 0, 64, 0, 1], 2)])
def test_a_token_takes_its_depth_behind_the_context(held, news, extra):
    from svdflash_b200.kernels.attention import tree_positions
    rng = random.Random(sum(held) + sum(news))
    masks, want = [], []
    for h, n in zip(held, news):
        rows, depth = [], []
        for i in range(n):
            parent = rng.randrange(-1, i)                      # -1: a root
            rows.append((rows[parent] if parent >= 0 else 0) | 1 << i)
            depth.append(depth[parent] + 1 if parent >= 0 else 0)
        masks += [_signed(r) for r in rows]
        want += [h + d for d in depth]
    masks += [-1] * extra
    got = tree_positions(_step(held, news, extra), torch.tensor(masks, dtype=torch.int64))
    assert got.dtype == torch.int32
    assert got.tolist() == want + [0] * extra                  # entries of nobody stay what they are


def test_a_chain_keeps_its_positions():
    from svdflash_b200.kernels.attention import tree_positions
    step = _step([5, 17], [64, 3], 0)
    chain = [_signed((1 << (i + 1)) - 1) for n in (64, 3) for i in range(n)]
    assert torch.equal(tree_positions(step, torch.tensor(chain)), step.positions)


def test_masks_of_another_shape_or_type_are_refused():
    from svdflash_b200.kernels.attention import tree_positions
    step = _step([5], [4], 0)
    with pytest.raises(ValueError, match="dimensions do not match"):
        tree_positions(step, torch.ones(3, dtype=torch.int64))
    with pytest.raises(TypeError, match="int64"):
        tree_positions(step, torch.ones(4, dtype=torch.int32))
