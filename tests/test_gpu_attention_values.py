"""GPU tests of attention over values that are not finite: what a row sees reaches it, what it does not see reaches
nothing, in whole units and in units that several workers share.  Rows without such a value are held to the bounds of
attention_ref.py; where a row sees an infinity or a NaN in v, that element is what the formula gives."""
from __future__ import annotations

import math

import pytest
import torch

import attention_ref as ref
from test_gpu_attention import _masks, _paged, _qkv, _randn, _status, att  # noqa: F401  (att: a fixture)

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
INF, NAN = math.inf, math.nan


def _check(out, want, seen, bad, elements, dtype, what):
    """`want`: the reference for finite values; seen [rows]: whether a row sees the bad value, in `elements` of its head."""
    out = out.clone()
    part = out[seen][..., elements]
    assert (part.isnan() if math.isnan(bad) else part == bad).all(), f"{what}: a row sees {bad} and has another value there"
    out[..., elements] = torch.where(seen[:, None, None], want[0][..., elements].to(dtype), out[..., elements])
    ref.check(out, *want, dtype, what)


@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("length,news,h,hk,d,block,dtype", [
    (40, 1, 4, 2, 128, 16, BF16), (9000, 1, 4, 1, 128, 16, BF16), (9000, 5, 8, 1, 64, 32, F16), (7001, 40, 8, 1, 128, 16, BF16),
    (30001, 1, 16, 2, 64, 64, F16)])
def test_a_value_that_rows_see_reaches_them(cuda_device, att, length, news, h, hk, d, block, dtype, bad):
    """One bad element of v, at the first, some middle and the last key that all rows see."""
    k, v, table = _paged(101, [length], hk, d, block, dtype)
    q = _randn(102, news, h, d, dtype=dtype)
    lens, cu = torch.tensor([length], dtype=torch.int32, device="cuda"), ref.cumulative([news], cuda_device)
    seen = torch.ones(news, dtype=torch.bool, device="cuda")
    want = ref.tree(q, k, v, table, [length], [news], None)
    for at in (0, length // 3, length - news):
        spoiled = v.clone()
        spoiled[table[0, at // block], :, at % block, 3] = bad
        out = att.tree_attention(q, k, spoiled, table, lens, cu, max_tree=news)
        _check(out, want, seen, bad, [3], dtype, f"{bad} at {at}")
    _status(cuda_device)


def _us(call):
    """The shortest of three runs on the device."""
    times = []
    for _ in range(3):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        call()
        end.record()
        end.synchronize()
        times.append(begin.elapsed_time(end) * 1e3)
    return min(times)


def _spoiled(t, at, element, bad):
    t = t.clone()
    t[at, :, element] = bad
    return t


@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("n,h,hk,d,dtype", [(50, 4, 2, 128, BF16), (333, 2, 1, 64, F16), (700, 2, 2, 128, BF16), (3001, 2, 1, 128, BF16)])
def test_a_prompt_value_reaches_the_rows_from_its_own_on(cuda_device, att, n, h, hk, d, dtype, bad):
    q, k, v = _qkv(111, n, n, h, hk, d, dtype)
    cu, rows = ref.cumulative([n], cuda_device), torch.arange(n, device="cuda")
    want = ref.prompt(q, k, v, [n], [n])
    for at in (0, n // 2, n - 2):
        out = att.prompt_attention(q, k, _spoiled(v, at, 5, bad), cu)
        _check(out, want, rows >= at, bad, [5], dtype, f"{bad} at {at}")
    # the same element of two tokens: rows between them see the first and lie in tiles that hold the second
    first, second = n // 3, n // 3 + 7
    out = att.prompt_attention(q, k, _spoiled(_spoiled(v, first, 5, bad), second, 5, bad), cu)
    _check(out, want, rows >= first, bad, [5], dtype, f"{bad} twice")
    # another element of a later token: rows that do not see it keep what they have
    out = att.prompt_attention(q, k, _spoiled(_spoiled(v, first, 5, bad), second, 9, bad), cu)
    part = out[rows >= second][..., 9]
    assert (part.isnan() if math.isnan(bad) else part == bad).all()
    out[..., 9] = torch.where((rows >= second)[:, None], want[0][..., 9].to(dtype), out[..., 9])
    _check(out, want, rows >= first, bad, [5], dtype, f"{bad} in two elements")
    _status(cuda_device)


@pytest.mark.parametrize("bad", [INF, NAN])
def test_a_tree_token_value_reaches_the_rows_that_see_it(cuda_device, att, bad):
    """Rows that see token 9 have its value, the others are as if it were finite; a value of the context reaches all."""
    news, lens, h, hk, d = [40], [3040], 8, 1, 128
    k, v, table = _paged(121, lens, hk, d, 16, BF16)
    q, mask = _randn(122, 40, h, d), _masks(123, news)
    want = ref.tree(q, k, v, table, lens, news, mask)
    seen = (mask >> 9) & 1 == 1
    assert 2 < seen.sum() < 38
    lens_t, cu = torch.tensor(lens, dtype=torch.int32, device="cuda"), ref.cumulative(news, cuda_device)
    for at in ([3009], [100, 3009]):
        spoiled = v.clone()
        for t in at:
            spoiled[table[0, t // 16], :, t % 16, 77 if t == 3009 else 33] = bad
        out = att.tree_attention(q, k, spoiled, table, lens_t, cu, max_tree=40, tree_mask=mask)
        if len(at) == 2:
            assert (out[..., 33].isnan() if math.isnan(bad) else out[..., 33] == bad).all()
            out[..., 33] = want[0][..., 33].to(BF16)
        _check(out, want, seen, bad, [77], BF16, f"{bad} at {at}")
    _status(cuda_device)


# A value that rows see costs them a look at the keys of their masked steps, some hundred of them and some microseconds a
# tile; done over key by key, each row would cost its whole walk, hundreds of times the call.  Four times lies between.
@pytest.mark.parametrize("what", ["key", "value", "query"])
@pytest.mark.parametrize("bad", [INF, NAN])
def test_a_long_prompt_that_sees_a_bad_value_is_not_done_over(cuda_device, att, what, bad):
    n, h, hk, d = 8192, 32, 8, 128
    x, cu = _randn(131, n, h + 2 * hk, d), ref.cumulative([n], cuda_device)
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    att.prompt_attention(q, k, v, cu)
    usual = _us(lambda: att.prompt_attention(q, k, v, cu))
    {"key": k, "value": v, "query": q}[what][0] = bad
    out = att.prompt_attention(q, k, v, cu)
    _status(cuda_device)
    if what == "value":
        assert (out.isnan() if math.isnan(bad) else out == bad).all()
    elif what == "key":
        assert out.isnan().all()                     # infinities of both signs in every score
    else:
        assert out[0].isnan().all() and torch.isfinite(out[1:]).all()
    assert _us(lambda: att.prompt_attention(q, k, v, cu)) < 4 * usual


def test_long_contexts_that_see_a_bad_value_are_not_done_over(cuda_device, att):
    lens, h, hk, d = [20000] * 16, 32, 8, 128
    blocks = torch.randperm(16 * 1250, device="cuda").to(torch.int32).view(16, 1250)
    k, v = _randn(141, 16 * 1250, hk, 16, d), _randn(142, 16 * 1250, hk, 16, d)
    q = _randn(143, 16 * 26, h, d)
    args = q, k, v, blocks, torch.tensor(lens, dtype=torch.int32, device="cuda"), ref.cumulative([26] * 16, cuda_device)
    want = att.tree_attention(*args, max_tree=26)
    usual = _us(lambda: att.tree_attention(*args, max_tree=26))
    v[blocks[:, 7].long(), :, 3, 11] = NAN
    out = att.tree_attention(*args, max_tree=26)
    _status(cuda_device)
    assert out[..., 11].isnan().all()
    out[..., 11] = want[..., 11]
    assert torch.equal(out, want)
    assert _us(lambda: att.tree_attention(*args, max_tree=26)) < 4 * usual
