"""GPU tests of what a decoder stack does from step to step: trees of drafted tokens against their own paths, lengths,
captured steps, misuse.  The plain decoder, the weights and the tolerance are those of test_gpu_decoder.py."""
from __future__ import annotations

import pytest
import torch

import test_gpu_decoder as plain
from test_gpu_decoder import HIDDEN, model  # noqa: F401  (the module's decoder, as a fixture)

pytestmark = pytest.mark.gpu


def _hidden(seed, n):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)


def _alone(x, weights, inv_freq):
    """The plain decoder over one sequence by itself."""
    n = x.shape[0]
    return plain._plain(x, weights, inv_freq, torch.arange(n, device="cuda"), plain._causal(n))


def test_every_tree_token_is_its_own_path(cuda_device, model):
    """A token's hidden state is what its path from the root gives when it is run alone, behind the same context."""
    from svdflash_b200.models import PagedDecoder
    layers, weights, inv_freq = model
    contexts = [40, 17]
    parents = [[-1, 0, 0, 1, 2, 4, 2, -1], [-1, -1, 0, 0, 2]]   # two roots each: drafts of the next token itself
    xs = [_hidden(30 + b, c + len(p)) for b, (c, p) in enumerate(zip(contexts, parents))]
    masks, paths = [], []
    for p in parents:
        rows = []
        for i, up in enumerate(p):
            rows.append((rows[up] if up >= 0 else 0) | 1 << i)
        masks += rows
        paths.append([[j for j in range(len(p)) if row >> j & 1] for row in rows])
    dec = PagedDecoder(layers, 2, 16, 128)
    dec.prefill(torch.cat([x[:c] for x, c in zip(xs, contexts)]), contexts)
    news = [len(p) for p in parents]
    y = dec.step(torch.cat([x[c:] for x, c in zip(xs, contexts)]), news,
                 tree_mask=torch.tensor(masks, dtype=torch.int64, device="cuda"))
    dec.check()
    for b, part in enumerate(y.split(news)):
        c = contexts[b]
        for i, path in enumerate(paths[b]):
            sequence = torch.cat((xs[b][:c], xs[b][c:][path]))
            plain._close(part[i], _alone(sequence, weights, inv_freq)[-1], f"request {b}, token {i}")
    # the accepted path, fed again behind the context, gives the same
    path = paths[0][5]
    dec.keep(torch.tensor(contexts, dtype=torch.int32, device="cuda"))
    again = dec.step(xs[0][contexts[0]:][path], [len(path), 0])
    plain._close(again, y[path].double(), "the path as a chain")
