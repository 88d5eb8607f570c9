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
