"""GPU tests of the decoder stack (attention over the paged cache beside the
SVD MLP block) against a plain fp64 decoder.

Tolerance: a layer rounds its activations to bf16 (unit roundoff u = 2^-8) some
eight times on the way (norm, q/k/v, rotary, probabilities, attention, output
projection and residual, the MLP's own intermediates and output), each an
independent relative error of about u / sqrt(3) of a term whose size is at most
the residual stream's: with two layers below 16 u / sqrt(3) = 0.036 even if they
all added up in step, and about 0.01 as a root of squares.  2e-2 of the norm lies
between the two."""
from __future__ import annotations

import math

import pytest
import torch

import svdmlp_oracle as orc
from helpers import to_dev

pytestmark = pytest.mark.gpu
HIDDEN, FF, RANK, HEADS, KV, DIM, LAYERS = 256, 512, 104, 4, 2, 64, 2


def _weights(seed):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, scale):
        return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).cuda()
    _, f = orc.make_inputs(seed, 1, HIDDEN, FF, RANK)
    return dict(wq=normal(HIDDEN, HEADS * DIM, scale=HIDDEN ** -0.5), wk=normal(HIDDEN, KV * DIM, scale=HIDDEN ** -0.5),
                wv=normal(HIDDEN, KV * DIM, scale=HIDDEN ** -0.5), wo=normal(HEADS * DIM, HIDDEN, scale=(HEADS * DIM) ** -0.5),
                n1=(1 + normal(HIDDEN, scale=0.02)), n2=(1 + normal(HIDDEN, scale=0.02)),
                factors=[to_dev(a, torch.device("cuda", 0)) for a in f])


def _norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.double()


def _plain(x, weights, inv_freq, positions, seen):
    """The decoder in fp64 over one sequence: x [n, H], seen [n, n]."""
    x = x.double()
    cos, sin = (positions.double()[:, None] * inv_freq.double()).cos(), (positions.double()[:, None] * inv_freq.double()).sin()

    def rope(t):
        a, b = t[..., :DIM // 2], t[..., DIM // 2:]
        return torch.cat((a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]), -1)
    for w in weights:
        y = _norm(x, w["n1"])
        q, k, v = (rope((y @ w["wq"].double()).unflatten(1, (HEADS, DIM))), rope((y @ w["wk"].double()).unflatten(1, (KV, DIM))),
                   (y @ w["wv"].double()).unflatten(1, (KV, DIM)))
        out = []
        for h in range(HEADS):
            s = (q[:, h] @ k[:, h * KV // HEADS].T / math.sqrt(DIM)).masked_fill(~seen, -math.inf)
            out.append(torch.softmax(s, 1) @ v[:, h * KV // HEADS])
        x = x + torch.cat(out, 1) @ w["wo"].double()
        y = _norm(x, w["n2"])
        ug, vg, uu, vu, ud, vd = (f.double() for f in w["factors"])
        gate = y @ ug @ vg
        x = x + (gate * torch.sigmoid(gate) * (y @ uu @ vu)) @ ud @ vd
    return x


@pytest.fixture(scope="module")
def model():
    from svdflash_b200.kernels import attention
    from svdflash_b200.models import DecoderLayer, SvdMlpBlock
    inv_freq, _ = attention.rope_frequencies(DIM)
    weights = [_weights(700 + i) for i in range(LAYERS)]
    layers = [DecoderLayer(w["wq"], w["wk"], w["wv"], w["wo"], w["n1"], SvdMlpBlock(*w["factors"], w["n2"]), heads=HEADS,
                           kv_heads=KV, inv_freq=inv_freq) for w in weights]
    return layers, weights, inv_freq


def _close(got, want, what):
    rel = (got.double() - want).norm() / want.norm()
    assert torch.isfinite(got.float()).all() and rel <= 2e-2, f"{what}: relative error {rel:.3e}"


def _causal(n):
    return torch.ones(n, n, dtype=torch.bool, device="cuda").tril()


def test_prefill_then_steps_match_the_plain_decoder(cuda_device, model):
    from svdflash_b200.models import PagedDecoder
    layers, weights, inv_freq = model
    lens, total = [33, 1, 150], [39, 7, 156]
    g = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(t, HIDDEN, generator=g, device="cuda").to(torch.bfloat16) for t in total]
    want = [_plain(x, weights, inv_freq, torch.arange(x.shape[0], device="cuda"), _causal(x.shape[0])) for x in xs]
    dec = PagedDecoder(layers, 3, 40, 200)
    outs = [[o] for o in dec.prefill(torch.cat([x[:n] for x, n in zip(xs, lens)]), lens).split(lens)]
    done = list(lens)
    for news in ([1, 1, 1], [1, 1, 1], [3, 3, 3], [1, 1, 1]):     # single tokens and a chain of three
        y = dec.step(torch.cat([x[n:n + k] for x, n, k in zip(xs, done, news)]), news)
        for o, part in zip(outs, y.split(news)):
            o.append(part)
        done = [a + b for a, b in zip(done, news)]
    dec.check()
    assert dec.seq_lens.tolist() == total
    for b in range(3):
        _close(torch.cat(outs[b]), want[b], f"request {b}")


def test_rejected_tokens_are_taken_back(cuda_device, model):
    """Drafted chains that are cut short leave no trace: neither in the results nor in the free list."""
    from svdflash_b200.models import PagedDecoder
    layers, weights, inv_freq = model
    g = torch.Generator(device="cuda").manual_seed(2)
    x = [torch.randn(60, HIDDEN, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
    junk = torch.randn(2 * 20, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
    dec = PagedDecoder(layers, 2, 12, 96)
    dec.prefill(torch.cat([x[0][:30], x[1][:15]]), [30, 15])
    before = dec.free_count.item()
    for _ in range(5):                                            # more in all than the cache holds
        dec.step(junk, [20, 20])
        dec.keep(torch.tensor([30, 15], dtype=torch.int32, device="cuda"))
        assert dec.free_count.item() == before
    dec.step(junk[:9], [6, 3])
    dec.keep(torch.tensor([31, 99], dtype=torch.int32, device="cuda"))   # at most what it holds
    assert dec.seq_lens.tolist() == [31, 18]
    dec.keep(torch.tensor([30, 15], dtype=torch.int32, device="cuda"))
    y = dec.step(torch.cat([x[0][30:60], x[1][15:60]]), [30, 45])
    dec.check()
    held = [int(b) for row, n in zip(dec.block_table.tolist(), (4, 4)) for b in row[:n]]
    free = dec.free_blocks[:dec.free_count.item()].tolist()
    assert sorted(held + free) == list(range(12))
    for b, (lo, part) in enumerate(zip((30, 15), y.split([30, 45]))):
        want = _plain(x[b], weights, inv_freq, torch.arange(60, device="cuda"), _causal(60))
        _close(part, want[lo:], f"request {b}")


def test_a_tree_matches_its_paths(cuda_device, model):
    from svdflash_b200.models import PagedDecoder
    layers, weights, inv_freq = model
    g = torch.Generator(device="cuda").manual_seed(3)
    n, parents = 40, [-1, 0, 0, 1, 2, 4]
    x = torch.randn(n + len(parents), HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
    seen = _causal(n + len(parents))
    rows = []
    for i, up in enumerate(parents):
        rows.append((rows[up] if up >= 0 else 0) | 1 << i)
        seen[n + i, n:] = torch.tensor([(rows[i] >> j) & 1 == 1 for j in range(len(parents))], device="cuda")
    dec = PagedDecoder(layers, 1, 8, 128)
    dec.prefill(x[:n], [n])
    y = dec.step(x[n:], [len(parents)], tree_mask=torch.tensor(rows, dtype=torch.int64, device="cuda"))
    dec.check()
    _close(y, _plain(x, weights, inv_freq, torch.arange(n + len(parents), device="cuda"), seen)[n:], "tree")


def test_a_cache_that_is_too_small_is_reported(cuda_device, model):
    from svdflash_b200.models import PagedDecoder
    layers, _, _ = model
    dec = PagedDecoder(layers, 1, 2, 96)
    dec.prefill(torch.zeros(40, HIDDEN, dtype=torch.bfloat16, device="cuda"), [40])
    with pytest.raises(RuntimeError, match="blocks too few"):
        dec.check()
    with pytest.raises(ValueError, match="sum to"):
        dec.step(torch.zeros(3, HIDDEN, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="at least one layer"):
        PagedDecoder([], 1, 2, 96)
