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


@pytest.mark.parametrize("news", [[1, 1, 1], [3, 1, 2], [2, 2, 0]])
def test_replays_of_a_captured_step_go_on(cuda_device, model, news):
    """Twenty replays, into new blocks, against the plain decoder and against eager steps, with tokens taken back
    between them."""
    from svdflash_b200.models import PagedDecoder
    layers, weights, inv_freq = model
    lens, replays = [33, 1, 150], 20
    xs = [_hidden(50 + b, n + k * (replays + 1)) for b, (n, k) in enumerate(zip(lens, news))]

    def tokens(step):
        return torch.cat([x[n + k * step:n + k * (step + 1)] for x, n, k in zip(xs, lens, news)])
    decs = [PagedDecoder(layers, 3, 40, 256) for _ in range(2)]
    outs = [[o] for o in decs[0].prefill(torch.cat([x[:n] for x, n in zip(xs, lens)]), lens).split(lens)]
    decs[1].prefill(torch.cat([x[:n] for x, n in zip(xs, lens)]), lens)
    feed = tokens(0)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = decs[0].step(feed, news)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            last = decs[0].step(feed, news)
    decs[1].step(feed, news)
    for o, part in zip(outs, first.split(news)):
        o.append(part)
    junk = _hidden(60, sum(news))
    for i in range(1, replays + 1):
        if i % 7 == 0:                                  # a draft that is taken back
            held = decs[0].seq_lens.clone()
            feed.copy_(junk)
            graph.replay()
            decs[0].keep(held)
        feed.copy_(tokens(i))
        graph.replay()
        for o, part in zip(outs, last.clone().split(news)):
            o.append(part)
        decs[1].step(tokens(i), news)
    decs[0].check()
    total = [n + k * (replays + 1) for n, k in zip(lens, news)]
    assert decs[0].seq_lens.tolist() == decs[1].seq_lens.tolist() == total
    assert decs[0].free_count.tolist() == decs[1].free_count.tolist() == [40 - sum(-(-t // 16) for t in total)]
    assert (decs[0].block_table >= 0).sum().item() == sum(-(-t // 16) for t in total)
    for b in range(3):
        plain._close(torch.cat(outs[b]), _alone(xs[b], weights, inv_freq), f"request {b}")


@pytest.mark.parametrize("how", ["prefill", "step", "chain"])
def test_a_request_that_outgrows_its_table_is_reported(cuda_device, model, how):
    from svdflash_b200.models import PagedDecoder
    layers, _, _ = model
    dec = PagedDecoder(layers, 2, 12, 33)                # three blocks of 16: 48 tokens a request
    x = _hidden(70, 100)
    dec.prefill(x[:48 + 5], [48, 5])
    dec.check()                                          # full, and no more
    if how == "prefill":
        dec = PagedDecoder(layers, 2, 12, 33)
        dec.prefill(x[:49 + 5], [49, 5])
    elif how == "step":
        dec.step(x[:2])
    else:
        dec.step(x[:9], [9, 0])
        dec.keep(torch.tensor([40, 5], dtype=torch.int32, device="cuda"))   # what was dropped stays reported
    with pytest.raises(RuntimeError, match="outgrew its table of 48"):
        dec.check()


def test_prefill_of_a_request_that_holds_tokens_is_reported(cuda_device, model):
    from svdflash_b200.models import PagedDecoder
    layers, weights, inv_freq = model
    x = _hidden(80, 60)
    dec = PagedDecoder(layers, 2, 12, 64)
    dec.prefill(x[:20], [20, 0])
    y = dec.prefill(x[20:50], [0, 30])                   # one request after another
    dec.check()
    plain._close(y, _alone(x[20:50], weights, inv_freq), "the second request")
    dec.keep(torch.zeros(2, dtype=torch.int32, device="cuda"))
    y = dec.prefill(x[:50], [40, 10])                    # new requests in the places of old ones
    dec.check()
    plain._close(y[:40], _alone(x[:40], weights, inv_freq), "a new request")
    z = dec.step(x[40:50], [10, 0])                      # a prompt's second chunk
    dec.check()
    plain._close(z, _alone(x[:50], weights, inv_freq)[40:], "the second chunk")
    dec.prefill(x[50:60], [0, 10])
    with pytest.raises(RuntimeError, match="held 10 tokens"):
        dec.check()


def test_a_masked_tree_of_more_than_64_tokens_is_refused(cuda_device, model):
    """A row's mask has no bits for the tokens behind the 64th: they would not even see themselves."""
    from svdflash_b200.models import PagedDecoder
    layers, _, _ = model
    dec = PagedDecoder(layers, 1, 12, 160)
    dec.prefill(_hidden(90, 10), [10])
    mask = torch.ones(70, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="at most 64"):
        dec.step(_hidden(91, 70), [70], tree_mask=mask)
    assert dec.seq_lens.tolist() == [10]
    dec.step(_hidden(91, 64), [64], tree_mask=mask[:64])
    dec.step(_hidden(91, 70), [70])                      # a chain has no such end
    dec.check()


def test_a_captured_tree_step_goes_on(cuda_device, model):
    """Depths come from the mask at every replay: the mask's contents may change between them."""
    from svdflash_b200.models import PagedDecoder
    layers, _, _ = model
    decs = [PagedDecoder(layers, 2, 30, 128) for _ in range(2)]
    x = _hidden(95, 60)
    for dec in decs:
        dec.prefill(x[:30], [20, 10])
    masks = [torch.tensor(m, dtype=torch.int64, device="cuda") for m in
             ([1, 3, 5, 9, 1, 2, 6], [1, 2, 5, 13, 1, 3, 7], [1, 3, 7, 15, 1, 3, 5])]
    feed, mask, news = x[30:37].clone(), masks[0].clone(), [4, 3]
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = decs[0].step(feed, news, tree_mask=mask)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            y = decs[0].step(feed, news, tree_mask=mask)
    assert torch.equal(first, decs[1].step(feed, news, tree_mask=masks[0]))
    kept = torch.tensor([21, 11], dtype=torch.int32, device="cuda")   # each draft is taken back to one token
    for i, m in enumerate(masks):
        for dec in decs:
            dec.keep(kept + i)
        feed.copy_(x[37 + 7 * i:44 + 7 * i])
        mask.copy_(m)
        graph.replay()
        assert torch.equal(y, decs[1].step(feed, news, tree_mask=m))
    decs[0].check()
    assert decs[0].seq_lens.tolist() == decs[1].seq_lens.tolist() == [27, 16]
