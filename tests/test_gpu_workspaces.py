"""GPU tests of the pooled workspaces: captured steps beside calls that need more, captures on streams without a
workspace."""
from __future__ import annotations

import threading

import pytest
import torch

import attention_ref as ref
from test_gpu_attention import _paged, _randn, att  # noqa: F401  (att: a fixture)
from test_gpu_decoder import model  # noqa: F401  (a fixture)
from test_gpu_decoder_steps import _hidden

pytestmark = pytest.mark.gpu


def _call(att):
    """A divided unit: its partials go through the workspace."""
    news, lens = [1, 20], [9000, 3000]
    k, v, table = _paged(1, lens, 2, 128, 16, torch.bfloat16)
    q, out = _randn(2, 21, 8, 128), torch.empty(21, 8, 128, dtype=torch.bfloat16, device="cuda")
    args = q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), ref.cumulative(news, q.device)
    return lambda: att.tree_attention(*args, max_tree=20, out=out)


def test_a_graph_keeps_the_workspace_that_it_writes(cuda_device, att):
    from svdflash_b200.kernels import ops
    call, stream, graph = _call(att), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    want = call().clone()
    with torch.cuda.stream(stream):
        call()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
        held = ops.workspace_for(cuda_device, 1)
        ops.workspace_for(cuda_device, held.nbytes + (64 << 20))       # a larger call on the same stream
        size = held.nbytes
        del held
        filled = [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(4)]
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert all((t == 0x5A).all() for t in filled)
    ops.check_device_status(cuda_device)


def test_a_capture_that_needs_more_than_its_stream_has(cuda_device, att):
    from svdflash_b200.kernels import ops
    call, graph = _call(att), torch.cuda.CUDAGraph()
    want = call().clone()
    for warm in (0, 1 << 20):                                          # no workspace at all, and a small one
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            if warm:
                ops.workspace_for(cuda_device, warm)
                torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                out = call()
                again = att.rope(out, out[:, :2].contiguous(), torch.zeros(21, dtype=torch.int32, device="cuda"),
                                 torch.ones(64, device="cuda"))
                call()
            ops.check_device_status(cuda_device)                       # nothing has set it up yet
            for _ in range(3):
                out.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want) and torch.equal(again[0], want)
            ops.check_device_status(cuda_device)
            assert torch.equal(call(), want)                           # and calls have their own


def test_a_decoding_step_captured_without_a_warm_stream(cuda_device, model):
    """Its GEMMs need less than its attention: the workspace grows inside the capture."""
    from svdflash_b200.models import PagedDecoder
    layers, _, _ = model
    decs = [PagedDecoder(layers, 1, 16, 128) for _ in range(2)]
    x = _hidden(5, 40)
    for dec in decs:
        dec.prefill(x[:30], [30])
    decs[1].step(x[30:31])
    feed, stream, graph = x[31:32].clone(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        y = decs[0].step(feed)
    outs = []
    for i in range(30, 40):
        feed.copy_(x[i:i + 1])
        graph.replay()
        outs.append(y.clone())
    want = [decs[1].step(x[i:i + 1]) for i in range(31, 40)]
    decs[0].check()
    assert decs[0].seq_lens.tolist() == decs[1].seq_lens.tolist() == [40]
    assert torch.equal(torch.cat(outs[1:]), torch.cat(want))


def test_threads_on_one_stream(cuda_device, att):
    """Divided units of two shapes from several threads at once: each thread's launches meet in its own workspace."""
    from svdflash_b200.kernels import ops
    calls, wants, wrong = [], [], []
    for news, lens in ([[1], [9000]], [[20], [3000]], [[1, 1], [5000, 70]], [[40], [4000]]):
        k, v, table = _paged(len(news) + lens[0], lens, 2, 128, 16, torch.bfloat16)
        q = _randn(3, sum(news), 8, 128)
        args = q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), ref.cumulative(news, cuda_device)
        calls.append(lambda args=args, most=max(news): att.tree_attention(*args, max_tree=most))
        wants.append(calls[-1]())
    torch.cuda.synchronize()
    start = threading.Barrier(len(calls))

    def work(call, want):
        start.wait()
        outs = [call() for _ in range(200)]
        torch.cuda.synchronize()
        wrong.append(sum(not torch.equal(o, want) for o in outs))
    threads = [threading.Thread(target=work, args=pair) for pair in zip(calls, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [0] * len(calls)
    ops.check_device_status(cuda_device)
