"""Plain 64-bit forms of the attention operators for the tests, and the error
bounds that their results are held to.

The bound of attention, per element, with u the unit roundoff of the 16-bit
type (bf16 2^-8, fp16 2^-11), A = sum_j p_j |v_j| and n keys:

* the output is rounded once: u |o|;
* each probability is rounded to the type before the product with v: u A (in
  fp16 a probability under 2^-14 of the row's largest has the absolute error
  2^-25 instead, and there are at most n of them: n 2^-25 max|v|);
* scores, exponentials and sums in fp32: a score of products of N(0, 1)
  elements over D = 128 is off by at most D 2^-24 sum|q_i k_i| s < 1e-4, which
  a probability takes on as a relative error: 2e-4 A with the exponential's and
  the sum's.
"""
from __future__ import annotations

import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def attend(q, k, v, seen, scale):
    """(out, bound term A, n 2^-25 max|v|) for q [n, D], k, v [m, D], seen [n, m], in float64.
    Keys that are not seen are left out altogether, whatever they hold."""
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    tiny = torch.zeros_like(out)
    for i in range(q.shape[0]):
        ids = seen[i].nonzero()[:, 0]
        if ids.numel() == 0:
            continue
        p = torch.softmax((k[ids] @ q[i]) * scale, 0)
        out[i] = p @ v[ids]
        mag[i] = p @ v[ids].abs()
        tiny[i] = ids.numel() * 2.0 ** -25 * v[ids].abs().max()
    return out, mag, tiny


def attend_all(q, k, v, seen, scale):
    """attend() for every row at once: only where all values are finite."""
    w = (q.double() @ k.double().T * scale).masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(torch.softmax(w, 1), nan=0.0)
    v = v.double()
    tiny = (seen.sum(1, keepdim=True) * 2.0 ** -25 * v.abs().max()).expand(-1, v.shape[1])
    return p @ v, p @ v.abs(), tiny


def check(got, want, mag, tiny, dtype, what=""):
    u = UNIT[dtype]
    bound = 1.01 * u * (want.abs() + mag) + 2e-4 * mag + 2 * tiny + 1e-30
    err = (got.double() - want).abs()
    assert torch.isfinite(got.float()).all(), f"{what}: non-finite output"
    worst = (err / bound).max().item()
    assert worst <= 1.0, f"{what}: error is {worst:.3f} of its bound (largest {err.max().item():.3e})"


def cumulative(lens, device):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(device)


def prompt_seen(n, m, causal, device):
    rows, keys = torch.arange(n, device=device), torch.arange(m, device=device)
    if not causal:
        return torch.ones(n, m, dtype=torch.bool, device=device)
    return keys[None, :] <= rows[:, None] + (m - n)


def prompt(q, k, v, lq, lk, causal=True, scale=None, rowwise=False):
    """(out, A, tiny) over packed sequences of lq queries and lk keys."""
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    group = q.shape[1] // k.shape[1]
    outs = [torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(3)]
    q0 = k0 = 0
    for n, m in zip(lq, lk):
        if n and m:
            seen = prompt_seen(n, m, causal, q.device)
            for h in range(q.shape[1]):
                got = (attend if rowwise else attend_all)(q[q0:q0 + n, h], k[k0:k0 + m, h // group],
                                                          v[k0:k0 + m, h // group], seen, scale)
                for o, g in zip(outs, got):
                    o[q0:q0 + n, h] = g
        q0, k0 = q0 + n, k0 + m
    return outs


def gather(cache, table_row, head, length):
    """The first `length` tokens of one request and head, [length, D]."""
    block = cache.shape[2]
    pages = table_row[: -(-length // block)].long()
    return cache[pages, head].reshape(-1, cache.shape[3])[:length]


def tree_seen(n, length, mask_rows, device):
    seen = torch.zeros(n, length, dtype=torch.bool, device=device)
    first = length - n
    seen[:, :max(first, 0)] = True
    for i in range(n):
        for j in range(n):
            if first + j < 0:
                continue
            if mask_rows is None:
                seen[i, first + j] = j <= i
            else:
                seen[i, first + j] = j < 64 and bool((int(mask_rows[i]) >> j) & 1)
    return seen


def tree(q, k_cache, v_cache, table, lens, news, masks, scale=None, rowwise=False):
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    group = q.shape[1] // k_cache.shape[1]
    outs = [torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(3)]
    q0 = 0
    for b, (n, length) in enumerate(zip(news, lens)):
        if n and length:
            rows = None if masks is None else masks[q0:q0 + n].tolist()
            seen = tree_seen(n, length, rows, q.device)
            for h in range(q.shape[1]):
                kk = gather(k_cache, table[b], h // group, length)
                vv = gather(v_cache, table[b], h // group, length)
                got = (attend if rowwise else attend_all)(q[q0:q0 + n, h], kk, vv, seen, scale)
                for o, g in zip(outs, got):
                    o[q0:q0 + n, h] = g
        q0 += n
    return outs


def rope(x, positions, inv_freq, interleaved, scale):
    """(rotated x, |a| + |b| per element) in float64."""
    half = inv_freq.shape[0]
    theta = positions.double()[:, None] * inv_freq.double()[None]
    cos, sin = (theta.cos() * scale)[:, None], (theta.sin() * scale)[:, None]
    y = x.double().clone()
    mag = torch.zeros_like(y)
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    mag[..., first] = mag[..., second] = (a.abs() + b.abs()) * abs(scale)
    return y, mag


def pages(table, held, added, free, count, block):
    """The paging step in Python: (table, slots, positions, cu, lens, count, missing)."""
    table = [list(r) for r in table]
    width = len(table[0])
    left = max(0, min(count, len(free)))
    slots, positions, cu, taken = [], [], [0], 0
    for b, (h, n) in enumerate(zip(held, added)):
        h, n = max(h, 0), max(n, 0)
        have, need = min(-(-h // block), width), min(-(-(h + n) // block), width)
        for i in range(have, need):
            table[b][i] = free[left - 1 - taken] if taken < left else -1
            taken += 1
        for pos in range(h, h + n):
            page = table[b][pos // block] if pos // block < width else -1
            slots.append(page * block + pos % block if page >= 0 else -1)
            positions.append(pos)
        cu.append(cu[-1] + n)
    return (table, slots, positions, cu, [max(h, 0) + max(n, 0) for h, n in zip(held, added)],
            max(left - taken, 0), max(taken - left, 0))
