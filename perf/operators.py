"""Cases of the attention operators beside the SVD MLP: prompt attention, tree attention over the paged cache, rotary
positions with the cache write, and the paging step that gives both their block tables and slots.

`run` computes an operator in its plain form (elementary torch operations in fp32), or, with `own` set, through
`svdflash_b200.kernels.attention`.  Head counts are the decoder layers' own (32 query and 8 key/value heads of 128 at
hidden 4096, 64 and 8 at hidden 8192) and generic ones beside them; lengths run from one token to long contexts.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DEVICE = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_module = None


def _attention():
    """The framework's operators (imported only when `own` is set)."""
    global _module
    if _module is None:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neuronmlp-on-tpu_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from svdflash_b200.kernels import attention
        _module = attention
    return _module


# --------------------------------------------------------------------- cases
def listed():
    return [
        # prompt attention: packed prompts, causal; `past` is what of each sequence came before this call's queries
        # the shortest prompt a chat turn sends: latency
        dict(name="prompt_short", op="prompt", type="bf16", heads=32, kv_heads=8, dim=128, batch=1, low=33, high=33, past=0),
        # a batch of mixed requests admitted together, one key/value head per query head
        dict(name="prompt_ragged", op="prompt", type="f16", heads=16, kv_heads=16, dim=64, batch=24, low=1, high=700, past=0),
        # prompts prefilled in chunks: each chunk's queries see the whole prefix
        dict(name="prompt_chunk", op="prompt", type="bf16", heads=32, kv_heads=8, dim=128, batch=4, low=1, high=512, past=5600),
        # one long document
        dict(name="prompt_long", op="prompt", type="bf16", heads=32, kv_heads=8, dim=128, batch=1, low=8192, high=8192, past=0),
        # tree attention over the paged cache; tree 1 is ordinary decoding
        # one user, a long conversation
        dict(name="decode_long", op="tree", type="bf16", heads=32, kv_heads=8, dim=128, batch=1, low=65537, high=65537, tree=1, block=16),
        # a full serving batch with contexts of very different lengths
        dict(name="decode_batch", op="tree", type="bf16", heads=32, kv_heads=8, dim=128, batch=64, low=1, high=16384, tree=1, block=16),
        # drafted trees of up to 26 tokens on short contexts
        dict(name="tree_small", op="tree", type="f16", heads=16, kv_heads=2, dim=64, batch=8, low=100, high=2100, tree=26, block=64),
        # drafted trees of up to 64 tokens on long contexts, 64 query heads
        dict(name="tree_wide", op="tree", type="bf16", heads=64, kv_heads=8, dim=128, batch=4, low=20001, high=32768, tree=64, block=32),
        # rotary positions and the cache write
        # one decoding step of a batch: interleaved pairs in half of the head
        dict(name="rope_decode", op="rope", type="f16", heads=32, kv_heads=8, dim=128, tokens=64, rotary=64, interleaved=True, block=16, last=16384, scale=1.0, keys=False),
        # a whole prompt at a long context's positions; its rotated keys also go to prompt attention
        dict(name="rope_prompt", op="rope", type="bf16", heads=32, kv_heads=8, dim=128, tokens=8192, rotary=128, interleaved=False, block=16, last=131072, scale=1.2, keys=True),
        # the paging step before each forward pass
        # a decoding step of a few requests
        dict(name="pages_decode", op="pages", batch=8, low=1, high=4000, new=1, block=16),
        # a scheduler tick that admits prompts beside a large decoding batch
        dict(name="pages_mixed", op="pages", batch=1024, low=0, high=8000, new=300, block=16),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


_HEADS = [(32, 8), (16, 16), (64, 8), (8, 1), (28, 4), (12, 2), (5, 5)]


def draw(rng):
    op = rng.choice(["prompt", "prompt", "tree", "tree", "rope", "pages"])
    if op == "prompt":
        while True:
            heads, kv = rng.choice(_HEADS)
            high = _log(rng, 1, 8192)
            c = dict(op=op, type=rng.choice(["bf16", "f16"]), heads=heads, kv_heads=kv, dim=rng.choice([64, 128]),
                     batch=_log(rng, 1, 32), low=_log(rng, 1, high), high=high,
                     past=rng.choice([0, 0, _log(rng, 1, 8192)]))
            if c["batch"] * heads * high * (high + c["past"]) <= 32 * 8192 * 8192:
                return c
    if op == "tree":
        while True:
            heads, kv = rng.choice(_HEADS)
            high = _log(rng, 1, 65536)
            c = dict(op=op, type=rng.choice(["bf16", "f16"]), heads=heads, kv_heads=kv, dim=rng.choice([64, 128]),
                     batch=_log(rng, 1, 128), low=_log(rng, 1, high), high=high,
                     tree=rng.choice([1, 1, _log(rng, 2, 64)]), block=rng.choice([16, 32, 64, 128]))
            if c["batch"] * (high + 64) * kv * c["dim"] <= 4 * 32832 * 8 * 128 and c["batch"] * high * heads * c["tree"] <= 4 * 32768 * 64 * 64:
                return c
    if op == "rope":
        heads, kv = rng.choice(_HEADS[:4])
        dim = rng.choice([64, 128])
        return dict(op=op, type=rng.choice(["bf16", "f16"]), heads=heads, kv_heads=kv, dim=dim, tokens=_log(rng, 1, 4096),
                    rotary=rng.choice([dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                    block=rng.choice([16, 32, 64]), last=_log(rng, 64, 131072), scale=rng.choice([1.0, 1.2]), keys=rng.random() < 0.5)
    high = _log(rng, 1, 8000)
    return dict(op=op, batch=_log(rng, 1, 1024), low=rng.randrange(0, high + 1), high=high, new=_log(rng, 1, 300),
                block=rng.choice([16, 32, 64, 128]))


def _spread(case, what, low, high, n):
    """n whole numbers between low and high, spread over their logarithm; the last is `high`."""
    rng = random.Random("%s %s %s %s" % (what, low, high, n))
    got = [min(high, max(low, _log(rng, max(low, 1), max(high, 1)))) if high > 0 else 0 for _ in range(n)]
    if low == 0:
        got = [0 if rng.random() < 0.1 else v for v in got]
    if got:
        got[-1] = high
    return got


def _lengths(case):
    """Query tokens and key tokens of each request (prompt, tree), or tokens held and tokens added (pages)."""
    n = case["batch"]
    first = _spread(case, "len", case["low"], case["high"], n)
    if case["op"] == "prompt":
        past = _spread(case, "past", 0, case["past"], n)
        return first, [a + b for a, b in zip(first, past)]
    if case["op"] == "tree":
        new = _spread(case, "tree", max(1, case["tree"] * 3 // 4), case["tree"], n)  # most trees are full or nearly
        return new, [a + b for a, b in zip(new, first)]
    return first, _spread(case, "new", 0 if n > 8 else 1, case["new"], n)


# -------------------------------------------------------------------- inputs
def _rng(seed):
    return torch.Generator(device=DEVICE).manual_seed(int(seed))


def _cumulative(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).to(DEVICE)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32)


def _tables(lens, block, g, spare=3):
    """A block table for requests of these lengths, with blocks in random order; unused entries are -1."""
    need = [-(-v // block) for v in lens]
    width = max(need + [1])
    order = torch.randperm(sum(need) + spare, generator=g, device=DEVICE).to(torch.int32)
    counts = torch.tensor(need, device=DEVICE)
    starts = counts.cumsum(0) - counts
    col = torch.arange(width, device=DEVICE)
    at = (starts[:, None] + col).clamp(max=sum(need) + spare - 1)
    table = torch.where(col < counts[:, None], order[at], torch.full_like(order[at], -1))
    return table.contiguous(), sum(need) + spare


def prepare(case, seed):
    g = _rng(seed)
    op = case["op"]
    s = dict(op=op, case=case)
    if op == "prompt":
        t = _TYPES[case["type"]]
        lq, lk = _lengths(case)
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        if case["past"]:
            q = _normal(g, sum(lq), h, d).to(t)
            kv = _normal(g, sum(lk), 2 * hk, d).to(t)
            k, v = kv[:, :hk], kv[:, hk:]
        else:  # the projections write q, k and v beside one another
            qkv = _normal(g, sum(lq), h + 2 * hk, d).to(t)
            q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        s.update(q=q, k=k, v=v, cu_q=_cumulative(lq), cu_k=_cumulative(lk), max_q=max(lq), max_k=max(lk))
    elif op == "tree":
        t = _TYPES[case["type"]]
        new, lens = _lengths(case)
        h, hk, d, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
        table, blocks = _tables(lens, block, g)
        rng = random.Random(int(seed))
        masks = []
        for n in new:  # each token hangs on one of the eight before it
            rows = []
            for i in range(n):
                up = rows[rng.randrange(max(0, i - 8), i)] if i else 0
                rows.append(up | 1 << i)
            masks += [r - (1 << 64) if r >> 63 else r for r in rows]
        s.update(q=_normal(g, sum(new), h, d).to(t), k_cache=_normal(g, blocks, hk, block, d).to(t),
                 v_cache=_normal(g, blocks, hk, block, d).to(t), table=table, cu_q=_cumulative(new),
                 lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE),
                 mask=torch.tensor(masks, dtype=torch.int64, device=DEVICE) if case["tree"] > 1 else None,
                 max_q=max(new), max_k=max(lens))
    elif op == "rope":
        t = _TYPES[case["type"]]
        h, hk, d, n, block = case["heads"], case["kv_heads"], case["dim"], case["tokens"], case["block"]
        qkv = _normal(g, n, h + 2 * hk, d).to(t)
        blocks = -(-n // block) + 1
        slots = torch.randperm(blocks * block, generator=g, device=DEVICE)[:n]
        if n > 1:
            slots[n // 2] = -1  # a padded token: rotated, written nowhere
        half = case["rotary"] // 2
        freq = torch.tensor([10000.0 ** (-i / half) for i in range(half)], dtype=torch.float64)
        s.update(q=qkv[:, :h], k=qkv[:, h:h + hk], v=qkv[:, h + hk:], slots=slots,
                 inv_freq=freq.to(torch.float32).to(DEVICE),
                 positions=torch.randint(0, case["last"], (n,), generator=g, device=DEVICE, dtype=torch.int32),
                 k_cache=_normal(g, blocks, hk, block, d).to(t), v_cache=_normal(g, blocks, hk, block, d).to(t))
    else:
        held, new = _lengths(case)
        block = case["block"]
        total = [a + b for a, b in zip(held, new)]
        table, used = _tables(held, block, g, spare=0)
        width = -(-max(total + [1]) // block) + 2
        wide = torch.full((len(held), width), -1, dtype=torch.int32, device=DEVICE)
        cols = min(width, table.shape[1])
        wide[:, :cols] = table[:, :cols]
        extra = sum(-(-a // block) for a in total) - sum(-(-a // block) for a in held) + 7
        free = used + torch.randperm(extra, generator=g, device=DEVICE).to(torch.int32)
        s.update(table=wide, held=torch.tensor(held, dtype=torch.int32, device=DEVICE),
                 new=torch.tensor(new, dtype=torch.int32, device=DEVICE), free=free,
                 free_count=torch.tensor([extra], dtype=torch.int32, device=DEVICE), tokens=sum(new))
    return s


# ----------------------------------------------------------------- one pass
def run(s):
    return {"prompt": _run_prompt, "tree": _run_tree, "rope": _run_rope, "pages": _run_pages}[s["op"]](s)


def _run_prompt(s):
    if own:
        return _attention().prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])
    return _plain_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["max_q"], s["max_k"])


def _run_tree(s):
    c = s["case"]
    if own:
        return _attention().tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu_q"],
                                           max_tree=c["tree"], tree_mask=s["mask"])
    return _plain_tree(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu_q"], s["mask"], s["max_q"],
                       s["max_k"])


def _run_rope(s):
    c = s["case"]
    if own:
        q, k = _attention().rope_cache(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["inv_freq"], s["k_cache"],
                                       s["v_cache"], interleaved=c["interleaved"], scale=c["scale"], return_k=c["keys"])
        return {"q": q, "k": k, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    q = _plain_rope(s["q"], s["positions"], s["inv_freq"], c["interleaved"], c["scale"])
    k = _plain_rope(s["k"], s["positions"], s["inv_freq"], c["interleaved"], c["scale"])
    _plain_write(s["k_cache"], s["slots"], k)
    _plain_write(s["v_cache"], s["slots"], s["v"])
    return {"q": q, "k": k if c["keys"] else None, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _run_pages(s):
    c = s["case"]
    if own:
        p = _attention().page_step(s["table"], s["held"], s["new"], s["free"], s["free_count"], c["block"], s["tokens"])
        return {"table": s["table"], "slots": p.slots, "positions": p.positions, "cu": p.cu_seqlens, "lens": p.seq_lens,
                "free_count": p.free_count, "missing": p.missing}
    return _plain_pages(s["table"], s["held"], s["new"], s["free"], s["free_count"], c["block"], s["tokens"])


# --------------------------------------------------------------- plain forms
def _softmax_times(scores, seen, v):
    """softmax(scores) v over the keys that are `seen`; rows that see nothing give zeros.
    scores [batch, kv head, group, row, key], v [batch, kv head, key, dim]."""
    scores = torch.where(seen, scores, torch.full_like(scores[..., :1], float("-inf")))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    b, hk, group, rows, keys = p.shape
    out = torch.matmul(p.reshape(b, hk, group * rows, keys), v).reshape(b, hk, group, rows, -1)
    return out / torch.where(total > 0, total, torch.ones_like(total))


def _padded(x, cu, longest):
    """Packed [N, heads, dim] as [batch, heads, longest, dim] in fp32, zeros beyond each length; and the places."""
    at = cu[:-1, None].long() + torch.arange(longest, device=x.device)
    held = at < cu[1:, None]
    at = at.clamp(max=max(x.shape[0] - 1, 0))
    return torch.where(held[..., None, None], x[at].float(), torch.zeros((), device=x.device)).transpose(1, 2), at, held


def _plain_prompt(q, k, v, cu_q, cu_k, max_q, max_k):
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    qp, at, held = _padded(q, cu_q, max_q)
    kp, vp = _padded(k, cu_k, max_k)[0], _padded(v, cu_k, max_k)[0]
    b = qp.shape[0]
    scores = torch.matmul(qp.reshape(b, hk, -1, d), kp.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    scores = scores.reshape(b, hk, h // hk, max_q, -1)
    lq, lk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    row, col = torch.arange(max_q, device=q.device), torch.arange(max_k, device=q.device)
    seen = (col <= row[:, None] + (lk - lq)[:, None, None]) & (col < lk[:, None, None])
    out = _softmax_times(scores, seen[:, None, None], vp)
    out = out.reshape(b, h, max_q, d).transpose(1, 2)
    return out[held].to(q.dtype)


def _plain_tree(q, k_cache, v_cache, table, lens, cu_q, mask, max_q, max_k):
    h, hk, d, block = q.shape[1], k_cache.shape[1], q.shape[2], k_cache.shape[2]
    qp, at, held = _padded(q, cu_q, max_q)
    b = qp.shape[0]
    pages = -(-max_k // block)
    blocks = table[:, :pages].clamp(min=0).long()
    col = torch.arange(pages * block, device=q.device)
    there = (col < lens[:, None])[:, None, :, None]
    zero = torch.zeros((), device=q.device)
    kp = torch.where(there, k_cache[blocks].float().transpose(1, 2).reshape(b, hk, pages * block, d), zero)
    vp = torch.where(there, v_cache[blocks].float().transpose(1, 2).reshape(b, hk, pages * block, d), zero)
    new = cu_q[1:] - cu_q[:-1]
    node = col - (lens - new)[:, None]                      # place in the tree; negative in the context
    if mask is None:
        inside = node[:, None] <= torch.arange(max_q, device=q.device)[:, None]
    else:
        inside = (mask[at][:, :, None] >> node.clamp(0, 63)[:, None]) & 1 == 1
    seen = ((node < 0)[:, None] | inside) & (col < lens[:, None])[:, None]
    scores = torch.matmul(qp.reshape(b, hk, -1, d), kp.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    scores = scores.reshape(b, hk, h // hk, max_q, -1)
    out = _softmax_times(scores, seen[:, None, None], vp)
    return out.reshape(b, h, max_q, d).transpose(1, 2)[held].to(q.dtype)


def _plain_rope(x, positions, inv_freq, interleaved, scale):
    angle = positions[:, None, None].float() * inv_freq
    cos, sin = torch.cos(angle) * scale, torch.sin(angle) * scale
    half = inv_freq.shape[0]
    turned, rest = x[..., :2 * half].float(), x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned.to(x.dtype), rest), -1)


def _plain_write(cache, slots, x):
    block = cache.shape[2]
    keep = slots >= 0
    # a token that is written nowhere repeats what a written one puts into its place
    first = torch.argmax(keep.to(torch.int32))
    at = torch.where(keep, slots, slots[first])
    cache[at // block, :, at % block] = torch.where(keep[:, None, None], x, x[first])


def _plain_pages(table, held, new, free, free_count, block, tokens):
    total = held + new
    have, need = (held + block - 1) // block, (total + block - 1) // block
    extra = need - have
    taken = extra.cumsum(0) - extra
    col = torch.arange(table.shape[1], device=table.device)
    fresh = (col >= have[:, None]) & (col < need[:, None])
    at = taken[:, None] + col - have[:, None]
    left = free_count[0]
    # blocks come off the end of the free list
    block_ids = free[(left - 1 - at).clamp(0, free.shape[0] - 1).long()]
    table.copy_(torch.where(fresh & (at < left), block_ids, torch.where(fresh, torch.full_like(table, -1), table)))
    cu = torch.cat((torch.zeros_like(new[:1]), new)).cumsum(0).to(torch.int32)
    token = torch.arange(tokens, device=table.device)
    who = torch.searchsorted(cu[1:].contiguous(), token.to(torch.int32), right=True).clamp(max=held.shape[0] - 1)
    place = token - cu[who] + held[who]
    page = table[who, (place // block).clamp(max=table.shape[1] - 1)].long()
    slots = torch.where(page >= 0, page * block + place % block, torch.full_like(page, -1))
    used = extra.sum().to(torch.int32)
    missing = (used - left).clamp(min=0).reshape(1)
    return {"table": table, "slots": slots, "positions": place.to(torch.int32), "cu": cu, "lens": total,
            "free_count": (left - used).clamp(min=0).reshape(1), "missing": missing}


# ---------------------------------------------------------- from 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        return None
    if case["op"] == "rope":
        return _exact_rope(s, case)
    h, hk = case["heads"], case["kv_heads"]
    group = h // hk
    scale = 1.0 / math.sqrt(case["dim"])
    lq, lk = _lengths(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    q0 = k0 = 0
    for b, (n, m) in enumerate(zip(lq, lk)):
        rows = torch.arange(n, device=DEVICE)
        keys = torch.arange(m, device=DEVICE)
        if case["op"] == "prompt":
            allowed = keys[None, :] <= rows[:, None] + (m - n)
        else:
            pages = s["table"][b, : -(-m // case["block"])].long()
            allowed = torch.zeros(n, m, dtype=torch.bool, device=DEVICE)
            allowed[:, : m - n] = True
            if s["mask"] is None:
                allowed[:, m - n:] = rows[None, :] <= rows[:, None]
            else:
                bits = s["mask"][q0:q0 + n]
                for j in range(n):
                    allowed[:, m - n + j] = (bits >> j) & 1 == 1
        for head in range(h):
            kv = head // group
            if case["op"] == "prompt":
                key, val = s["k"][k0:k0 + m, kv].double(), s["v"][k0:k0 + m, kv].double()
            else:
                key = s["k_cache"][pages, kv].reshape(-1, case["dim"])[:m].double()
                val = s["v_cache"][pages, kv].reshape(-1, case["dim"])[:m].double()
            w = (s["q"][q0:q0 + n, head].double() @ key.T * scale).masked_fill(~allowed, -math.inf)
            out[q0:q0 + n, head] = torch.softmax(w, dim=1) @ val
        q0, k0 = q0 + n, k0 + m
    return out


def _exact_rope(s, case):
    half, block = case["rotary"] // 2, case["block"]
    theta = s["positions"].double()[:, None] * s["inv_freq"].double()[None]
    turn = torch.polar(torch.full_like(theta, case["scale"]), theta)[:, None]
    got = {}
    for name in ("q", "k"):
        x = s[name].double().clone()
        if case["interleaved"]:
            first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
        else:
            first, second = slice(0, half), slice(half, 2 * half)
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        got[name] = x
    for name, x in (("k_cache", got["k"]), ("v_cache", s["v"].double())):
        cache = s[name].double().clone()
        for token, slot in enumerate(s["slots"].tolist()) if x.shape[0] <= 64 else ():
            if slot >= 0:
                cache[slot // block, :, slot % block] = x[token]
        if x.shape[0] > 64:
            keep = (s["slots"] >= 0).nonzero()[:, 0]
            at = s["slots"][keep]
            cache[at // block, :, at % block] = x[keep]
        got[name] = cache
    if not case["keys"]:
        got["k"] = None
    return got


# ---------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "pages":
        held, new = _lengths(case)
        block = case["block"]
        fresh = sum(-(-(a + b) // block) - -(-a // block) for a, b in zip(held, new))
        # read held, new, the blocks taken and each written token's page; write them, slots, positions, offsets, lengths
        return {"bytes": 16.0 * len(held) + 8.0 * fresh + 12.0 * sum(new) + 16, "flops": 0.0}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "rope":
        n = case["tokens"]
        moved = n * d * (2 * h + 4 * hk + (hk if case["keys"] else 0))  # q in and out; k and v in and into the cache; k out
        return {"bytes": 2.0 * moved + 12.0 * n, "flops": 3.0 * n * case["rotary"] * (h + hk)}
    lq, lk = _lengths(case)
    if op == "prompt":
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(lq, lk))
    else:
        pairs = sum(n * (m - n) + n for n, m in zip(lq, lk))  # the context, and each token itself
    return {"bytes": 2.0 * d * (2 * h * sum(lq) + 2 * hk * sum(lk)), "flops": 4.0 * pairs * h * d}
