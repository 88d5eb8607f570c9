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


def test_out_apart_from_every_input(cuda_device, att):
    """One key/value head per query head: out could be k or v by its shape."""
    n, h, d = 70, 4, 64
    q, k, v = (_randn(3 + i, n, h, d) for i in range(3))
    cu = ref.cumulative([n], cuda_device)
    both = torch.cat([v, v])
    for out in (q, k, v):
        with pytest.raises(ValueError, match="overlap"):
            att.prompt_attention(q, k, v, cu, out=out)
    with pytest.raises(ValueError, match="overlap"):
        att.prompt_attention(q, k, both[:n], cu, out=both[n // 2:n // 2 + n])
    half = both[:, :2]
    with pytest.raises(ValueError, match="overlap"):
        att.prompt_attention(q[:, :2], both[:n, 1:3], half[:n], cu, out=both[n:, :2].as_strided((n, 2, d), half.stride(), d))
    want = att.prompt_attention(q, k, v, cu)
    qkv = torch.empty(n, 4 * h, d, dtype=BF16, device="cuda")          # q, k, v and the output side by side
    qkv[:, :h], qkv[:, h:2 * h], qkv[:, 2 * h:3 * h] = q, k, v
    out = qkv[:, 3 * h:]
    assert att.prompt_attention(qkv[:, :h], qkv[:, h:2 * h], qkv[:, 2 * h:3 * h], cu, out=out) is out
    assert torch.equal(out, want)


def test_tree_out_apart_from_the_cache(cuda_device, att):
    lens, hk, d, block = [40], 2, 64, 16
    k, v, table = _paged(7, lens, hk, d, block, BF16)
    q = _randn(8, 1, 2, d)
    args = table, torch.tensor(lens, dtype=torch.int32, device="cuda"), ref.cumulative([1], cuda_device)
    want = att.tree_attention(q, k, v, *args, max_tree=1)
    for cache in (k, v):
        place = cache[1, :, 3:4].transpose(0, 1)                        # [1, heads, d]: one token's place in a block
        assert place.shape == q.shape
        with pytest.raises(ValueError, match="overlap"):
            att.tree_attention(q, k, v, *args, max_tree=1, out=place)
    wide = torch.zeros(3, 2, d, dtype=BF16, device="cuda")
    att.tree_attention(q, k, v, *args, max_tree=1, out=wide[1:2])
    assert torch.equal(wide[1:2], want) and not wide[0].any() and not wide[2].any()


@pytest.mark.parametrize("batch,width", [(1, 3), (3, 3), (9, 20), (30, 3)])
def test_units_just_longer_than_those_left_whole(cuda_device, att, batch, width):
    """Three steps a unit, with few and with many units: cuts everywhere in them."""
    news, lens = [33 + i % 32 for i in range(batch)], [257 + (i * 37) % 128 for i in range(batch)]
    k, v, table = _paged(11, lens, 2, 64, 128, BF16)
    table = torch.nn.functional.pad(table, (0, max(0, width - table.shape[1])), value=-1).contiguous()
    q = _randn(12, sum(news), 8, 64)
    args = table, torch.tensor(lens, dtype=torch.int32, device="cuda"), ref.cumulative(news, cuda_device)
    outs = [att.tree_attention(q, k, v, *args, max_tree=64) for _ in range(3)]
    ref.check(outs[0], *ref.tree(q, k, v, table, lens, news, None), BF16, f"{batch}")
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_a_chain_of_hundreds_behind_a_long_context(cuda_device, att):
    """A prompt's next chunk over the cache."""
    news, lens = [512, 300, 1], [4512, 9000, 700]
    k, v, table = _paged(13, lens, 2, 128, 16, BF16)
    q = _randn(14, sum(news), 8, 128)
    args = table, torch.tensor(lens, dtype=torch.int32, device="cuda"), ref.cumulative(news, cuda_device)
    want = ref.tree(q, k, v, table, lens, news, None)
    for most in (512, 1):
        ref.check(att.tree_attention(q, k, v, *args, max_tree=most), *want, BF16, f"max_tree {most}")
