"""GPU tests of the paging step over lengths that no request has: they must not reach anything outside the table, the
free list and the outputs.  The plain form counts in Python's unbounded integers, cut where the operator says."""
from __future__ import annotations

import random

import pytest
import torch

from test_gpu_attention import att  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
MOST = 2 ** 31 - 1


def _plain(table, held, added, free, count, block, tokens):
    table, width = [list(r) for r in table], len(table[0])
    left = max(0, min(count, len(free)))
    slots, positions, cu, lens, taken = [-1] * tokens, [0] * tokens, [0], [], 0
    for b, (h, n) in enumerate(zip(held, added)):
        h = max(h, 0)
        n = min(max(n, 0), MOST - h)
        have, need = min(-(-h // block), width), min(-(-(h + n) // block), width)
        for i in range(have, need):
            table[b][i] = free[left - 1 - taken] if taken < left else -1
            taken += 1
        for t in range(cu[-1], min(cu[-1] + n, MOST, tokens)):
            pos = h + t - cu[-1]
            page = table[b][pos // block] if pos // block < width else -1
            slots[t], positions[t] = page * block + pos % block if page >= 0 else -1, pos
        begin = cu[-1]
        cu.append(min(begin + n, MOST))
        lens.append(h + cu[-1] - begin)
    return table, slots, positions, cu, lens, max(left - taken, 0), max(taken - left, 0)


HOSTILE = [MOST, MOST - 1, MOST - 15, MOST - 16, 2 ** 30, 2 ** 31 - 70, -1, -2 ** 31, 0, 1, 17, 60]


@pytest.mark.parametrize("batch,block,tokens", [(1, 16, 9), (12, 16, 50), (144, 16, 300), (144, 1, 40), (1500, 64, 700), (144, 16, 0)])
def test_lengths_that_no_request_has(cuda_device, att, batch, block, tokens):
    rng = random.Random(batch + block)
    pairs = [(h, n) for h in HOSTILE for n in HOSTILE] if batch == 144 else \
        [(MOST, 5)] if batch == 1 else [(h, 5) for h in HOSTILE] if batch == 12 else \
        [(rng.choice(HOSTILE + [3, 40]), rng.choice([0, 1, 1, 7, rng.choice(HOSTILE)])) for _ in range(batch)]
    held, added = [h for h, _ in pairs], [n for _, n in pairs]
    width, free, count = 5, list(range(500, 500 + 300)), 290
    wide = torch.full((batch + 2, 40), -9, dtype=torch.int32, device="cuda")       # what lies around the table stays
    table = wide[1:1 + batch, 20:20 + width]
    start = [[1000 * b + i for i in range(width)] for b in range(batch)]
    table.copy_(torch.tensor(start, dtype=torch.int32))
    args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (held, added, free, [count])]
    got = att.page_step(table, *args, block, tokens)
    want = _plain(start, held, added, free, count, block, tokens)
    assert table.tolist() == want[0]
    assert got.slots.tolist() == want[1]
    assert got.positions.tolist() == want[2]
    assert got.cu_seqlens.tolist() == want[3]
    assert got.seq_lens.tolist() == want[4]
    assert (got.free_count.tolist(), got.missing.tolist()) == ([want[5]], [want[6]])
    table.fill_(-9)
    assert (wide == -9).all()


def test_more_tokens_than_said_still_take_their_blocks(cuda_device, att):
    """num_tokens below the sum (none at all, to take blocks ahead): the table is the same."""
    held, added = [5, 0, 40, 16], [60, 33, 0, 1]
    args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (held, added, list(range(30)), [30])]
    tables = []
    for tokens in (sum(added), 50, 1, 0):
        table = torch.full((4, 6), -9, dtype=torch.int32, device="cuda")
        got = att.page_step(table, *args, 16, tokens)
        tables.append(table.tolist())
        want = _plain([[-9] * 6] * 4, held, added, list(range(30)), 30, 16, tokens)
        assert (tables[-1], got.cu_seqlens.tolist(), got.free_count.tolist()) == (want[0], want[3], [want[5]])
        assert got.slots.tolist() == want[1]
    assert all(t == tables[0] for t in tables)


@pytest.mark.parametrize("each", [2 ** 21 - 1, 2 ** 21])
def test_sums_of_many_long_requests(cuda_device, att, each):
    """1100 requests: their tokens add up to 2^31 and more."""
    batch, block = 1100, 64
    args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([3] * batch, [each] * batch, list(range(40)), [40])]
    table = torch.full((batch, 2), -9, dtype=torch.int32, device="cuda")
    got = att.page_step(table, *args, block, 20)
    want = _plain([[-9, -9]] * batch, [3] * batch, [each] * batch, list(range(40)), 40, block, 20)
    assert table.tolist() == want[0] and got.slots.tolist() == want[1] and got.positions.tolist() == want[2]
    assert got.cu_seqlens.tolist() == want[3] and got.seq_lens.tolist() == want[4]
    assert (got.free_count.tolist(), got.missing.tolist()) == ([want[5]], [want[6]])
