"""GPU tests of the attention operators against their plain 64-bit forms
(attention_ref.py, which derives the bounds)."""
from __future__ import annotations

import random

import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def att():
    from svdflash_b200.kernels import attention
    return attention


def _randn(seed, *shape, dtype=BF16, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=device).to(dtype)


def _status(device):
    from svdflash_b200.kernels import ops
    ops.check_device_status(device)


# ------------------------------------------------------------------- prompt
def _qkv(seed, nq, nk, h, hk, d, dtype):
    """q, k, v as views of one buffer (nq == nk) or of two."""
    if nq == nk:
        x = _randn(seed, nq, h + 2 * hk, d, dtype=dtype)
        return x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    kv = _randn(seed + 1, nk, 2 * hk, d, dtype=dtype)
    return _randn(seed, nq, h, d, dtype=dtype), kv[:, :hk], kv[:, hk:]


PROMPTS = [
    # lq, lk (None: the same), heads, kv heads, head_dim, dtype
    ([1], None, 4, 1, 128, BF16),
    ([1], None, 1, 1, 64, F16),
    ([2, 1, 3], None, 3, 3, 128, F16),
    ([63, 64, 65], None, 4, 2, 64, BF16),
    ([127, 128, 129], None, 4, 2, 128, BF16),
    ([255, 256, 257], None, 2, 1, 128, F16),
    ([300, 1, 0, 511, 17], None, 8, 2, 128, BF16),
    ([0, 0, 40], None, 2, 2, 64, F16),
    ([513, 700], None, 5, 5, 64, BF16),
    ([1025], None, 28, 4, 128, BF16),
    ([1, 1, 1], [1, 300, 129], 8, 1, 128, BF16),
    ([100, 7, 256], [356, 1000, 256], 4, 2, 128, F16),
    ([33, 130], [161, 131], 4, 4, 64, BF16),
    ([200, 10, 300], [100, 0, 299], 4, 2, 128, BF16),   # more queries than keys: rows that see nothing
    ([2049], None, 2, 1, 64, F16),
]


@pytest.mark.parametrize("lq,lk,h,hk,d,dtype", PROMPTS)
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_matches_the_formula(cuda_device, att, lq, lk, h, hk, d, dtype, causal):
    lk = lq if lk is None else lk
    q, k, v = _qkv(sum(lq) + d, sum(lq), sum(lk), h, hk, d, dtype)
    out = att.prompt_attention(q, k, v, ref.cumulative(lq, cuda_device), ref.cumulative(lk, cuda_device), causal=causal)
    want, mag, tiny = ref.prompt(q, k, v, lq, lk, causal)
    ref.check(out, want, mag, tiny, dtype, f"{lq} {lk}")
    _status(cuda_device)


def _behind(t, rows):
    """`t` with `rows` rows of NaN behind it, which no sequence holds."""
    return torch.cat([t, torch.full((rows, *t.shape[1:]), float("nan"), dtype=t.dtype, device=t.device)])


@pytest.mark.parametrize("lq,lk,h,hk,d,dtype", PROMPTS)
@pytest.mark.parametrize("causal,scale", [(True, None), (False, None), (True, -0.05), (False, 0.0)])
def test_prompt_in_long_tensors(cuda_device, att, lq, lk, h, hk, d, dtype, causal, scale):
    """The tiles for long walks over the keys are taken by the tensors' lengths."""
    lk = lq if lk is None else lk
    q, k, v = _qkv(sum(lq) + d, sum(lq), sum(lk), h, hk, d, dtype)
    want, mag, tiny = ref.prompt(q, k, v, lq, lk, causal, scale)
    k, v = _behind(k, 1500 * len(lq)), _behind(v, 1500 * len(lq))
    cq, ck = ref.cumulative(lq, cuda_device), ref.cumulative(lk, cuda_device)
    outs = [att.prompt_attention(q, k, v, cq, ck, causal=causal, scale=scale) for _ in range(2)]
    _status(cuda_device)
    ref.check(outs[0], want, mag, tiny, dtype, f"{lq} {lk}")
    assert torch.equal(*outs)


@pytest.mark.parametrize("scale", [0.0, 0.02, 1.0, -0.125])
def test_prompt_scale(cuda_device, att, scale):
    lq = [140, 65]
    q, k, v = _qkv(5, 205, 205, 4, 2, 128, BF16)
    cu = ref.cumulative(lq, cuda_device)
    # the scores' error grows with the scale: keep them as small as the bound assumes
    q = (q.float() / max(1.0, abs(scale) * 128 ** 0.5)).to(BF16)
    out = att.prompt_attention(q, k, v, cu, scale=scale)
    ref.check(out, *ref.prompt(q, k, v, lq, lq, True, scale), BF16, f"scale {scale}")


def test_prompt_large_scores(cuda_device, att):
    """Scores far above the exponential's range: the running maximum keeps the sums finite, one key wins."""
    n, d = 300, 128
    q, k, v = _qkv(6, n, n, 2, 1, d, BF16)
    q, k = (q * 40).contiguous(), (k * 40).contiguous()
    cu = ref.cumulative([n], cuda_device)
    out = att.prompt_attention(q, k, v, cu)
    want, mag, tiny = ref.prompt(q, k, v, [n], [n])
    # scores of about 1600 * sqrt(128) are known to 128 * 2^-24 of their terms' sum: up to 0.2 in a probability
    # where two keys are that close, so only rows with a clear winner are compared
    s = (q[:, 0].double() @ k[:, 0].double().T * d ** -0.5).masked_fill(~ref.prompt_seen(n, n, True, cuda_device), -1e30)
    top = s.topk(2, dim=1).values
    clear = (top[:, 0] - top[:, 1]) > 20
    assert clear.sum() > n // 2
    ref.check(out[clear][:, :1], want[clear][:, :1], mag[clear][:, :1], tiny[clear][:, :1], BF16, "winner")
    assert torch.isfinite(out.float()).all()


def test_prompt_sequences_do_not_touch(cuda_device, att):
    """NaN and infinities of one sequence stay there, and rows of no sequence give zeros."""
    lq = [100, 30, 129, 61]
    q, k, v = (t.contiguous() for t in _qkv(7, sum(lq) + 40, sum(lq) + 40, 4, 2, 128, BF16))
    cu = ref.cumulative(lq, cuda_device)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for t in (q, k, v):
            t[100:130] = bad
            t[sum(lq):] = bad
        out = att.prompt_attention(q, k, v, cu)
        want, mag, tiny = ref.prompt(q, k, v, [100], [100])
        ref.check(out[:100], want[:100], mag[:100], tiny[:100], BF16, "before")
        w, m, t = ref.prompt(q[130:320], k[130:320], v[130:320], lq[2:], lq[2:])
        ref.check(out[130:320], w, m, t, BF16, "after")
        assert (out[sum(lq):] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d,dtype", [(128, BF16), (64, F16)])
def test_prompt_masked_places_do_not_matter(cuda_device, att, bad, d, dtype):
    """What a later token's key or value holds does not reach the rows before it."""
    n = 333
    q, k, v = (t.contiguous() for t in _qkv(8, n, n, 2, 1, d, dtype))
    for at in (70, 200, 332):
        k2, v2 = k.clone(), v.clone()
        k2[at:] = bad
        v2[at:] = bad
        out = att.prompt_attention(q, k2, v2, ref.cumulative([n], cuda_device))
        want, mag, tiny = ref.prompt(q[:at], k[:at], v[:at], [at], [at])
        ref.check(out[:at], want, mag, tiny, dtype, f"{bad} from {at}")


def test_prompt_strides_and_outputs(cuda_device, att):
    lq = [150, 43]
    n, h, hk, d = 193, 4, 2, 128
    cu = ref.cumulative(lq, cuda_device)
    base, kb, vb = _randn(9, n, h, d), _randn(10, n, hk, d), _randn(11, n, hk, d)
    want, mag, tiny = ref.prompt(base, kb, vb, lq, lq)
    heads_first = base.transpose(0, 1).contiguous().transpose(0, 1)               # [h, n, d] in memory
    odd = torch.empty(n, h * d + 1, dtype=BF16, device="cuda")[:, 1:].view(n, h, d)  # rows off 16 bytes
    odd.copy_(base)
    last = torch.empty(n, h, d, 2, dtype=BF16, device="cuda")[..., 0]             # no unit stride in the head
    last.copy_(base)
    for q in (base, heads_first, odd, last):
        ref.check(att.prompt_attention(q, kb, vb, cu), want, mag, tiny, BF16, "strides")
    k1 = _randn(12, n, 1, d).expand(n, hk, d)                                     # one key head, broadcast
    w1, m1, t1 = ref.prompt(base, k1, vb, lq, lq)
    ref.check(att.prompt_attention(base, k1, vb, cu), w1, m1, t1, BF16, "broadcast")
    wide = torch.full((n, h + 3, d + 8), 7.0, dtype=BF16, device="cuda")
    out = wide[:, 1:1 + h, :d]
    assert att.prompt_attention(base, kb, vb, cu, out=out) is out
    ref.check(out, want, mag, tiny, BF16, "out")
    out.fill_(7.0)
    assert (wide == 7.0).all()                                                    # nothing beside it was written


def test_prompt_offsets_beyond_32_bits(cuda_device, att):
    n, h, hk, d, step = 70, 2, 1, 128, 1 << 25
    big = torch.empty(n * step, dtype=BF16, device="cuda")                        # 4.7 GB: the last rows are past 2^31 elements
    q, k, v = (big.as_strided((n, m, d), (step, d, 1), at) for m, at in ((h, 0), (hk, 1024), (hk, 2048)))
    for t, seed in ((q, 13), (k, 14), (v, 15)):
        t.copy_(_randn(seed, *t.shape))
    out = big.as_strided((n, h, d), (step, d, 1), 4096)
    cu = ref.cumulative([n - 3, 3], cuda_device)
    att.prompt_attention(q, k, v, cu, out=out)
    ref.check(out, *ref.prompt(q, k, v, [n - 3, 3], [n - 3, 3]), BF16, "far rows")


def test_prompt_streams_graphs_and_repeats(cuda_device, att):
    lq = [300, 77]
    q, k, v = _qkv(16, 377, 377, 8, 2, 128, BF16)
    cu = ref.cumulative(lq, cuda_device)
    first = att.prompt_attention(q, k, v, cu)
    for _ in range(5):
        assert torch.equal(att.prompt_attention(q, k, v, cu), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = att.prompt_attention(q, k, v, cu)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(first)
    with torch.cuda.graph(graph, stream=side):
        att.prompt_attention(q, k, v, cu, out=out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)


# --------------------------------------------------------------------- tree
def _paged(seed, lens, hk, d, block, dtype, spare=3):
    """Caches whose unused places hold NaN, and a table with -1 beyond each request's blocks."""
    need = [-(-m // block) for m in lens]
    rng = random.Random(seed)
    ids = list(range(sum(need) + spare))
    rng.shuffle(ids)
    width = max(need + [1]) + 1
    rows, at = [], 0
    for m in need:
        rows.append(ids[at:at + m] + [-1] * (width - m))
        at += m
    table = torch.tensor(rows, dtype=torch.int32, device="cuda")
    shape = (len(ids), hk, block, d)
    k = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
    v = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
    for b, m in enumerate(lens):
        for i in range(need[b]):
            fill = min(block, m - i * block)
            k[rows[b][i], :, :fill] = _randn(seed + 7 * b + i, hk, fill, d, dtype=dtype)
            v[rows[b][i], :, :fill] = _randn(seed + 7 * b + i + 9999, hk, fill, d, dtype=dtype)
    return k, v, table


def _masks(seed, news):
    rng = random.Random(seed)
    out = []
    for n in news:
        rows = []
        for i in range(n):
            rows.append((rows[rng.randrange(max(0, i - 4), i)] if i else 0) | 1 << i)
        out += [r - (1 << 64) if r >> 63 else r for r in rows]
    return torch.tensor(out, dtype=torch.int64, device="cuda")


TREES = [
    # new tokens, lengths with them, heads, kv heads, head_dim, block, dtype, masked
    ([1], [1], 4, 1, 128, 16, BF16, False),
    ([1], [17], 1, 1, 64, 16, F16, False),
    ([1, 1, 1, 1], [1, 16, 63, 64], 32, 8, 128, 16, BF16, False),
    ([1, 1, 1], [65, 4097, 1000], 8, 8, 64, 32, F16, False),
    ([1, 1], [3000, 5], 64, 8, 128, 128, BF16, False),
    ([1] * 5, [700, 0, 129, 2500, 1], 28, 4, 128, 16, BF16, False),   # an empty request
    ([1, 1, 1], [9, 2047, 300], 5, 5, 128, 8, F16, False),
    ([4, 4], [4, 300], 8, 2, 128, 16, BF16, False),                   # a chain: causal in the tree
    ([5, 0, 3], [70, 12, 3], 8, 1, 64, 16, F16, True),
    ([26, 26], [126, 2026], 16, 2, 64, 64, F16, True),
    ([64, 13, 64], [64, 1013, 2064], 8, 8, 128, 32, BF16, True),
    ([64], [5000], 64, 8, 128, 16, BF16, True),
    ([33, 1, 64], [160, 161, 162], 8, 1, 128, 1024, BF16, True),
    ([70, 3], [170, 90], 4, 2, 128, 16, BF16, False),                 # larger than max_tree says
    ([300], [500], 8, 2, 64, 16, F16, False),
]


@pytest.mark.parametrize("news,lens,h,hk,d,block,dtype,masked", TREES)
def test_tree_matches_the_formula(cuda_device, att, news, lens, h, hk, d, block, dtype, masked):
    k, v, table = _paged(31, lens, hk, d, block, dtype)
    q = _randn(32, sum(news), h, d, dtype=dtype)
    mask = _masks(33, news) if masked else None
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, mag, tiny = ref.tree(q, k, v, table, lens, news, mask)
    for max_tree in {min(64, max(news)), 1, 64}:
        out = att.tree_attention(q, k, v, table, lens_t, ref.cumulative(news, cuda_device), max_tree=max_tree,
                                 tree_mask=mask)
        ref.check(out, want, mag, tiny, dtype, f"{news} {lens} max_tree {max_tree}")
    _status(cuda_device)


def test_tree_many_requests(cuda_device, att):
    """More requests than threads of a CTA, many of them empty, lengths from 0 to some hundreds."""
    rng = random.Random(4)
    lens = [rng.choice([0, 1, rng.randrange(1, 40), rng.randrange(1, 700)]) for _ in range(700)]
    news = [min(m, rng.choice([0, 1, 1, 1, 2])) for m in lens]
    k, v, table = _paged(41, lens, 2, 64, 16, F16)
    q = _randn(42, sum(news), 4, 64, dtype=F16)
    out = att.tree_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                             ref.cumulative(news, cuda_device), max_tree=2)
    ref.check(out, *ref.tree(q, k, v, table, lens, news, None), F16, "many")


def test_tree_rows_that_see_nothing(cuda_device, att):
    """No context and an empty mask: zeros; the rows beside them are not disturbed."""
    news, lens, h, hk, d = [6, 4], [6, 40], 4, 2, 128
    k, v, table = _paged(51, lens, hk, d, 16, BF16)
    q = _randn(52, 10, h, d)
    mask = torch.tensor([1, 0, 5, 0, 16, 63, 0, 2, 0, 15], dtype=torch.int64, device="cuda")
    out = att.tree_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                             ref.cumulative(news, cuda_device), max_tree=6, tree_mask=mask)
    ref.check(out, *ref.tree(q, k, v, table, lens, news, mask), BF16, "masks")
    assert (out[1] == 0).all() and (out[3] == 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_tree_masked_places_do_not_matter(cuda_device, att, bad):
    news, lens, h, hk, d = [16], [90], 8, 2, 128
    k, v, table = _paged(61, lens, hk, d, 16, BF16)
    q = _randn(62, 16, h, d)
    mask = _masks(63, news)
    want, mag, tiny = ref.tree(q, k, v, table, lens, news, mask)
    hidden = [i for i in range(16) if not (int(mask[i]) >> 9) & 1]                # rows that do not see token 9
    at = lens[0] - 16 + 9
    page = int(table[0, at // 16])
    k[page, :, at % 16], v[page, :, at % 16] = bad, bad
    out = att.tree_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                             ref.cumulative(news, cuda_device), max_tree=16, tree_mask=mask)
    assert len(hidden) > 4
    ref.check(out[hidden], want[hidden], mag[hidden], tiny[hidden], BF16, f"{bad}")


def test_tree_tables_are_not_trusted(cuda_device, att):
    """Blocks outside the cache are not seen, lengths are clipped to the table."""
    lens, h, hk, d, block = [64, 100], 4, 2, 128, 16
    k, v, table = _paged(71, lens, hk, d, block, BF16)
    q = _randn(72, 2, h, d)
    want = torch.zeros(2, h, d, dtype=torch.float64, device="cuda")
    mag, tiny = want.clone(), want.clone()
    broken = table.clone()
    broken[0, 1], broken[0, 2] = -1, k.shape[0]
    seen0 = torch.ones(1, 64, dtype=torch.bool, device="cuda")
    seen0[:, 16:48] = False
    lens_t = torch.tensor([64, 1 << 30], dtype=torch.int32, device="cuda")
    narrow = broken[:, :6].contiguous()                                           # 96 tokens at most
    seen1 = torch.ones(1, 96, dtype=torch.bool, device="cuda")
    for head in range(h):
        for b, seen, m in ((0, seen0, 64), (1, seen1, 96)):
            got = ref.attend_all(q[b:b + 1, head], ref.gather(k, table[b], head // 2, m),
                                 ref.gather(v, table[b], head // 2, m), seen, d ** -0.5)
            for t, g in zip((want, mag, tiny), got):
                t[b, head] = g[0]
    out = att.tree_attention(q, k, v, narrow, lens_t, ref.cumulative([1, 1], cuda_device), max_tree=1)
    ref.check(out, want, mag, tiny, BF16, "tables")


def test_tree_cache_beyond_32_bits(cuda_device, att):
    """Blocks whose elements lie past 2^31, in a strided cache (k and v interleaved block by block)."""
    hk, d, block, blocks = 8, 128, 16, 70000
    both = torch.empty(blocks, 2, hk, block, d, dtype=BF16, device="cuda")        # 4.6 GB
    k, v = both[:, 0], both[:, 1]
    ids = [blocks - 1, 3, blocks - 2, blocks - 40, 65537]
    for i in ids:
        k[i], v[i] = _randn(81 + i, hk, block, d), _randn(82 + i, hk, block, d)
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    q = _randn(83, 1, 32, d)
    out = att.tree_attention(q, k, v, table, torch.tensor([75], dtype=torch.int32, device="cuda"),
                             ref.cumulative([1], cuda_device), max_tree=1)
    ref.check(out, *ref.tree(q, k, v, table, [75], [1], None), BF16, "far blocks")
    # and the cache write reaches them
    n = 6
    slots = torch.tensor([i * block + 5 for i in ids] + [-1], device="cuda")
    kk, vv = _randn(84, n, hk, d), _randn(85, n, hk, d)
    freq = torch.full((8,), 0.1, device="cuda")
    _, turned = att.rope_cache(_randn(86, n, 32, d), kk, vv, torch.zeros(n, dtype=torch.int32, device="cuda"), slots, freq,
                               k, v, return_k=True)
    for t, i in enumerate(ids):
        assert torch.equal(k[i, :, 5], turned[t]) and torch.equal(v[i, :, 5], vv[t])


def test_tree_repeats_and_streams(cuda_device, att):
    """Split work is joined in a fixed order: the same bits every time, on any stream, and from a graph."""
    news, lens, h, hk, d = [1, 7, 20], [9000, 40, 3000], 32, 8, 128
    k, v, table = _paged(91, lens, hk, d, 16, BF16)
    q = _randn(92, sum(news), h, d)
    lens_t, cu = torch.tensor(lens, dtype=torch.int32, device="cuda"), ref.cumulative(news, cuda_device)

    def call(out=None):
        return att.tree_attention(q, k, v, table, lens_t, cu, max_tree=20, out=out)
    first = call()
    ref.check(first, *ref.tree(q, k, v, table, lens, news, None), BF16, "first")
    for _ in range(20):
        assert torch.equal(call(), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(first)
    with torch.cuda.graph(graph, stream=side):
        call(out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    # the graph reads the lengths when it runs
    lens_t[0] = 20
    graph.replay()
    torch.cuda.synchronize()
    ref.check(out, *ref.tree(q, k, v, table, [20, 40, 3000], news, None), BF16, "new lengths")


# --------------------------------------------------------------------- rope
ROPES = [
    # tokens, heads, kv heads, head_dim, rotary_dim, interleaved, dtype
    (1, 4, 1, 128, 128, False, BF16),
    (1, 32, 8, 64, 64, True, F16),
    (7, 5, 5, 64, 32, False, F16),
    (33, 28, 4, 128, 64, True, BF16),
    (700, 8, 2, 128, 128, False, BF16),
    (257, 3, 1, 80, 20, True, F16),       # no whole vectors
    (19, 2, 2, 33, 6, False, BF16),       # odd heads
    (64, 4, 2, 256, 256, True, BF16),
    (5000, 4, 2, 128, 32, False, F16),
]


@pytest.mark.parametrize("n,h,hk,d,rot,interleaved,dtype", ROPES)
def test_rope_matches_the_formula(cuda_device, att, n, h, hk, d, rot, interleaved, dtype):
    qkv = _randn(n + d, n, h + 2 * hk, d, dtype=dtype)
    q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    g = torch.Generator(device="cuda").manual_seed(n)
    positions = torch.randint(0, 1 << 20, (n,), generator=g, device="cuda", dtype=torch.int32)
    positions[0] = 0
    freq, _ = att.rope_frequencies(d, rotary_dim=rot, base=500000.0)
    block, scale = 16, 1.25
    blocks = -(-n // block) + 1
    slots = torch.randperm(blocks * block, generator=g, device="cuda")[:n]
    if n > 2:
        slots[1], slots[2] = -1, blocks * block                                   # written nowhere
    caches = [torch.full((blocks, hk, block, d), 3.0, dtype=dtype, device="cuda") for _ in range(2)]
    q_out, k_out = att.rope_cache(q, k, v, positions, slots, freq, *caches, interleaved=interleaved, scale=scale,
                                  return_k=True)
    for got, x in ((q_out, q), (k_out, k)):
        want, mag = ref.rope(x, positions, freq, interleaved, scale)
        # one rounding to the type, and fp32 arithmetic on cosines good to 2^-21
        bound = ref.UNIT[dtype] * want.abs() + 1e-6 * mag + 2.0 ** -25
        assert ((got.double() - want).abs() <= bound).all()
        assert torch.equal(got[..., rot:], x[..., rot:])
    want_k, want_v = (torch.full((blocks * block, hk, d), 3.0, dtype=dtype, device="cuda") for _ in range(2))
    keep = (slots >= 0) & (slots < blocks * block)
    want_k[slots[keep]], want_v[slots[keep]] = k_out[keep], v[keep]
    for cache, want in zip(caches, (want_k, want_v)):
        assert torch.equal(cache.transpose(1, 2).reshape(blocks * block, hk, d), want)
    # without a cache, and without the keys
    q2, k2 = att.rope(q, k, positions, freq, interleaved=interleaved, scale=scale)
    assert torch.equal(q2, q_out) and torch.equal(k2, k_out)
    q3, k3 = att.rope_cache(q, k, v, positions, slots, freq, *caches, interleaved=interleaved, scale=scale)
    assert torch.equal(q3, q_out) and k3 is None


def test_rope_is_a_rotation(cuda_device, att):
    """Scores depend on the distance alone, and positions of 2^20 are as exact as small ones."""
    q, k = _randn(3, 2, 1, 128, dtype=F16), _randn(4, 2, 1, 128, dtype=F16)
    q[1], k[1] = q[0], k[0]
    freq, _ = att.rope_frequencies(128)
    far = 1 << 20
    qr, _ = att.rope(q, k, torch.tensor([11, far + 11], dtype=torch.int32, device="cuda"), freq)
    _, kr = att.rope(q, k, torch.tensor([3, far + 3], dtype=torch.int32, device="cuda"), freq)
    s = (qr.double() * kr.double()).sum((1, 2))
    mag = (qr.double().abs() * kr.double().abs()).sum().item()
    assert abs(s[0] - s[1]).item() <= 4 * 2.0 ** -11 * mag / 16


def test_rope_unaligned_rows_and_strided_caches(cuda_device, att):
    n, h, hk, d, block = 37, 4, 2, 64, 8
    base = _randn(5, n, (h + 2 * hk) * d + 1)[:, 1:].view(n, h + 2 * hk, d)
    q, k, v = base[:, :h], base[:, h:h + hk], base[:, h + hk:]
    both = torch.zeros(n, 2, hk, block, d, dtype=BF16, device="cuda")
    positions = torch.arange(n, dtype=torch.int32, device="cuda")
    slots = torch.arange(n, device="cuda") * block + 3
    freq, _ = att.rope_frequencies(d)
    got = att.rope_cache(q, k, v, positions, slots, freq, both[:, 0], both[:, 1], return_k=True)
    want = att.rope(q.contiguous(), k.contiguous(), positions, freq)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(both[:, 0, :, 3], want[1]) and torch.equal(both[:, 1, :, 3], v)
    both[:, :, :, 3] = 0
    assert (both == 0).all()


# -------------------------------------------------------------------- pages
@pytest.mark.parametrize("batch,block,high,new,short", [
    (1, 16, 0, 1, False), (1, 16, 100, 0, False), (3, 16, 70, 40, False), (8, 64, 4000, 1, False),
    (255, 16, 300, 9, False), (1024, 16, 500, 3, False), (1025, 32, 200, 70, False), (2500, 8, 60, 20, False),
    (40, 16, 100, 90, True), (1300, 16, 100, 90, True), (5, 24, 100, 90, False)])
def test_page_step_matches_the_plain_form(cuda_device, att, batch, block, high, new, short):
    rng = random.Random(batch + high)
    held = [rng.randrange(0, high + 1) for _ in range(batch)]
    added = [rng.choice([0, 1, rng.randrange(0, new + 1)]) if new else 0 for _ in range(batch)]
    width = max(-(-(h + n) // block) for h, n in zip(held, added)) or 1
    if short:
        width = max(1, width - 2)                                                 # some requests outgrow the table
    ids = list(range(50000))
    rng.shuffle(ids)
    table = []
    for h in held:
        have = min(-(-h // block), width)
        table.append([ids.pop() for _ in range(have)] + [-7] * (width - have))
    lacked = sum(min(-(-(h + n) // block), width) - min(-(-h // block), width) for h, n in zip(held, added))
    count = lacked // 2 if short else lacked + 3
    free = ids[:count + 5]
    table_t = torch.tensor(table, dtype=torch.int32, device="cuda")
    args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (held, added, free, [count])]
    total = sum(added)
    for extra in (0, 37):
        got = att.page_step(table_t, *args, block, total + extra)
        want = ref.pages(table, held, added, free, count, block)
        assert table_t.tolist() == want[0]
        assert got.slots.tolist() == want[1] + [-1] * extra
        assert got.positions.tolist() == want[2] + [0] * extra
        assert got.cu_seqlens.tolist() == want[3]
        assert got.seq_lens.tolist() == want[4]
        assert got.free_count.tolist() == [want[5]]
        assert got.missing.tolist() == [want[6]]
    assert [a.tolist() for a in args] == [held, added, free, [count]]


def test_page_step_in_a_strided_table(cuda_device, att):
    wide = torch.full((3, 20), -9, dtype=torch.int32, device="cuda")
    table = wide[:, 4:10]
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 0, 0], [33, 1, 16], list(range(10, 20)), [9])]
    got = att.page_step(table, *ints, 16, 50)
    assert table.tolist() == [[18, 17, 16, -9, -9, -9], [15, -9, -9, -9, -9, -9], [14, -9, -9, -9, -9, -9]]
    assert got.free_count.tolist() == [4] and got.missing.tolist() == [0]
    table[:] = -9
    assert (wide == -9).all()


# ------------------------------------------------------------- all together
def test_steps_through_the_cache_match_one_prompt(cuda_device, att):
    """A prompt, then single tokens, then a drafted chain, through page_step, rope_cache and the attentions, give what
    one prompt over all tokens gives."""
    b, h, hk, d, block = 3, 8, 2, 128, 16
    steps = [[37, 1, 90], [1, 1, 1], [1, 0, 1], [5, 5, 5]]
    totals = [sum(s[i] for s in steps) for i in range(b)]
    x = [_randn(200 + i, totals[i], h + 2 * hk, d) for i in range(b)]
    freq, scale = att.rope_frequencies(d, base=500000.0, scaling=dict(
        rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192))
    kc, vc = att.kv_cache(40, hk, block, d)
    table = torch.full((b, 12), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    free, count = torch.arange(40, dtype=torch.int32, device="cuda"), torch.tensor([40], dtype=torch.int32, device="cuda")
    outs = [[] for _ in range(b)]
    done = [0] * b
    for step, news in enumerate(steps):
        cur = torch.cat([x[i][done[i]:done[i] + news[i]] for i in range(b)])
        ps = att.page_step(table, lens, torch.tensor(news, dtype=torch.int32, device="cuda"), free, count, block, sum(news))
        q, k = att.rope_cache(cur[:, :h], cur[:, h:h + hk], cur[:, h + hk:], ps.positions, ps.slots, freq, kc, vc,
                              scale=scale, return_k=True)
        if step == 0:
            o = att.prompt_attention(q, k, cur[:, h + hk:], ps.cu_seqlens)
        else:
            o = att.tree_attention(q, kc, vc, table, ps.seq_lens, ps.cu_seqlens, max_tree=max(news))
        lens, count = ps.seq_lens, ps.free_count
        at = 0
        for i in range(b):
            outs[i].append(o[at:at + news[i]])
            at += news[i]
            done[i] += news[i]
    assert count.tolist() == [40 - sum(-(-t // block) for t in totals)]
    for i in range(b):
        whole = x[i]
        q, k = att.rope(whole[:, :h], whole[:, h:h + hk], torch.arange(totals[i], dtype=torch.int32, device="cuda"), freq,
                        scale=scale)
        want, mag, tiny = ref.prompt(q, k, whole[:, h + hk:], [totals[i]], [totals[i]])
        ref.check(torch.cat(outs[i]), want, mag, tiny, BF16, f"request {i}")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk,h,hk,d,dtype", [
    ([127, 50, 1949], [127, 0, 1949], 12, 4, 128, F16),                          # no keys between two long walks
    ([60, 1, 40, 7, 900], [0, 0, 0, 0, 5000], 8, 2, 64, BF16),
    ([300] + [2] * 40 + [500], [900] + [600] * 40 + [500], 4, 1, 128, BF16),     # second row tiles of nobody, one after another
    ([900] + [2] * 20 + [2000], [2500] + [1400] * 20 + [2000], 4, 1, 128, BF16),
])
def test_prompt_units_without_rows_or_keys(cuda_device, att, lq, lk, h, hk, d, dtype, causal):
    """Units that have nothing for one or both row tiles, between units that have; the same every time."""
    q, k, v = _qkv(sum(lk) + d, sum(lq), sum(lk), h, hk, d, dtype)
    cq, ck = ref.cumulative(lq, cuda_device), ref.cumulative(lk, cuda_device)
    want = ref.prompt(q, k, v, lq, lk, causal)
    far = [_behind(t, 1500 * len(lq)) for t in (k, v)]
    outs = [att.prompt_attention(q, k, v, cq, ck, causal=causal) for _ in range(8)]
    more = [att.prompt_attention(q, *far, cq, ck, causal=causal) for _ in range(8)]
    _status(cuda_device)
    for got in (outs, more):
        ref.check(got[0], *want, dtype, f"{lq} {lk}")
        assert all(torch.equal(o, got[0]) for o in got)


# ----------------------------------------------------------------- refusals
def test_python_refusals(cuda_device, att):
    q, k = _randn(1, 6, 4, 128), _randn(2, 6, 2, 128)
    cu = ref.cumulative([6], cuda_device)
    kc, vc = att.kv_cache(4, 2, 16, 128)
    table, lens = torch.zeros(1, 4, dtype=torch.int32, device="cuda"), torch.tensor([6], dtype=torch.int32, device="cuda")
    pos, slots = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.arange(6, device="cuda")
    freq, _ = att.rope_frequencies(128)

    def prompt(q=q, k=k, v=k, cu_q=cu, cu_k=None, **kw):
        return att.prompt_attention(q, k, v, cu_q, cu_k, **kw)

    def tree(q=q, kc=kc, vc=vc, table=table, lens=lens, cu=cu, max_tree=6, **kw):
        return att.tree_attention(q, kc, vc, table, lens, cu, max_tree=max_tree, **kw)

    def turn(q=q, k=k, v=k, pos=pos, slots=slots, freq=freq, kc=kc, vc=vc):
        return att.rope_cache(q, k, v, pos, slots, freq, kc, vc)

    prompt(), tree(), turn()
    for call, error in [
            (lambda: prompt(q=q.float()), TypeError), (lambda: prompt(k=k.half()), TypeError),
            (lambda: prompt(q=q[:, :3]), ValueError), (lambda: prompt(q=q[..., :96], k=k[..., :96], v=k[..., :96]), ValueError),
            (lambda: prompt(v=k[:5]), ValueError), (lambda: prompt(q=q[:5]), ValueError), (lambda: prompt(q=q[0]), ValueError),
            (lambda: prompt(cu_q=cu.long()), TypeError), (lambda: prompt(cu_q=cu[:1]), ValueError),
            (lambda: prompt(cu_k=ref.cumulative([3, 3], cuda_device)), ValueError), (lambda: prompt(cu_q=cu.cpu()), ValueError),
            (lambda: prompt(scale=float("nan")), ValueError), (lambda: prompt(out=torch.empty_like(k)), ValueError),
            (lambda: prompt(out=torch.empty_like(q).half()), TypeError), (lambda: prompt(out=q), ValueError),
            (lambda: tree(out=q), ValueError),
            (lambda: tree(kc=kc[:, :, :12], vc=vc[:, :, :12]), ValueError), (lambda: tree(kc=kc.half()), TypeError),
            (lambda: tree(vc=vc[:3]), ValueError), (lambda: tree(max_tree=0), ValueError), (lambda: tree(max_tree=1.5), ValueError),
            (lambda: tree(lens=lens.long()), TypeError), (lambda: tree(table=table[0]), ValueError),
            (lambda: tree(table=table.long()), TypeError), (lambda: tree(tree_mask=slots[:5]), ValueError),
            (lambda: tree(tree_mask=slots.int()), TypeError), (lambda: tree(q=q[:, :3]), ValueError),
            (lambda: turn(pos=pos.long()), TypeError), (lambda: turn(slots=slots.int()), TypeError),
            (lambda: turn(slots=slots[:4]), ValueError), (lambda: turn(freq=freq.double()), TypeError),
            (lambda: turn(freq=torch.ones(65, device="cuda")), ValueError), (lambda: turn(k=k[:4], v=k[:4]), ValueError),
            (lambda: turn(v=q), ValueError), (lambda: turn(vc=None), TypeError)]:
        with pytest.raises(error):
            call()


def test_empty_calls(cuda_device, att):
    none = torch.empty(0, 4, 128, dtype=BF16, device="cuda")
    zero = ref.cumulative([0], cuda_device)
    assert att.prompt_attention(none, none[:, :2], none[:, :2], zero).shape == (0, 4, 128)
    q = _randn(1, 3, 4, 128)
    assert (att.prompt_attention(q, none[:, :2], none[:, :2], ref.cumulative([3], cuda_device), zero) == 0).all()
    kc, vc = att.kv_cache(2, 2, 16, 128)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert att.tree_attention(none, kc, vc, table, lens, zero, max_tree=1).shape == (0, 4, 128)
    freq, _ = att.rope_frequencies(128)
    a, b = att.rope(none, none[:, :2], torch.empty(0, dtype=torch.int32, device="cuda"), freq)
    assert a.shape == (0, 4, 128) and b.shape == (0, 2, 128)
