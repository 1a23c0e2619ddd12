"""The kernels of the cache, attention and log-probability calls are loaded with a context's first
such call, which may be one that a graph captures."""
import threading

import pytest
import torch

import dflash_qmm
from gpu_util import announce

pytestmark = pytest.mark.gpu


def inputs():
    gen = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.randn(6, 9001, device="cuda", generator=gen)
    rows = torch.randn(2, 90, 128, device="cuda", generator=gen).bfloat16()
    q = torch.randn(2, 3, 256, device="cuda", generator=gen).bfloat16()
    return logits, rows, q


def work(ctx, logits, rows, q, cache, ws):
    top = ctx.token_logprobs(logits, top_k=4, ws=ws[:1 << 20])
    ctx.cache_append(cache, rows, rows)
    y = ctx.cache_attention(q, cache, ws=ws[1 << 20:])
    return (*top[1:], *y)


def test_first_calls_in_a_captured_graph():
    logits, rows, q = inputs()
    ws = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")
    cache = dflash_qmm.KVCache(2, 2, 90, 64)
    eager = dflash_qmm.Context(0)
    want = [a.clone() for a in work(eager, logits, rows, q, cache, ws)]
    torch.cuda.synchronize()
    ctx = dflash_qmm.Context(0)
    graph = torch.cuda.CUDAGraph()
    announce("first calls captured")
    with torch.cuda.graph(graph):
        got = work(ctx, logits, rows, q, cache, ws)
    for _ in range(3):
        for a in got:
            a.fill_(7)
        for a in cache.k + cache.v:
            a.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        again = work(eager, logits, rows, q, cache, ws)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want))
    for c in (ctx, eager):
        c.close()


def test_first_call_in_the_context_s_own_graph():
    logits, _, _ = inputs()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    ctx = dflash_qmm.Context(0)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    announce("first call in a graph of the context")
    ctx.graph_begin(stream)
    _, entropy, ids, _ = ctx.token_logprobs(logits, top_k=4, ws=ws, stream=stream)
    graph = ctx.graph_end(stream)
    want = ctx.token_logprobs(logits, top_k=4)
    for _ in range(3):
        entropy.fill_(7)
        ids.fill_(7)
        torch.cuda.synchronize()
        graph.launch(stream)
        stream.synchronize()
        assert torch.equal(entropy, want[1]) and torch.equal(ids, want[2])
    graph.close()
    ctx.close()


def test_first_calls_of_several_threads():
    logits, _, _ = inputs()
    ctx = dflash_qmm.Context(0)
    announce("first calls of threads")
    outs = [None] * 6

    def call(i):
        outs[i] = ctx.token_logprobs(logits, top_k=4)
    threads = [threading.Thread(target=call, args=(i,)) for i in range(len(outs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(o[2], outs[0][2]) and torch.equal(o[1], outs[0][1]) for o in outs)
    ctx.close()
