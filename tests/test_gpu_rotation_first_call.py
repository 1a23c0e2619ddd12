"""The rotation's and the sampled accept's kernels are loaded with a context's first call of each,
which may be one that a graph captures, or one of several threads'."""
import threading

import pytest
import torch

import dflash_qmm
from gpu_util import announce

pytestmark = pytest.mark.gpu


def inputs():
    gen = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(2, 9, 4, 128, device="cuda", generator=gen).bfloat16()
    logits = torch.randn(3, 4, 9001, device="cuda", generator=gen)
    drafts = torch.randint(0, 9001, (3, 3), device="cuda", generator=gen).to(torch.int32)
    return q, logits, drafts, torch.rand(3, 4, device="cuda", generator=gen)


def work(ctx, rope, q, logits, drafts, u, ws):
    return (ctx.rope(rope, q), ctx.qk_norm_rope(rope, q),
            *ctx.sample_accept(logits, u, drafts, draft_logits=logits[:, :-1], ws=ws))


def test_first_calls_in_a_captured_graph():
    rope = dflash_qmm.Rope(128)
    ws = torch.empty(8 << 20, dtype=torch.uint8, device="cuda")
    args = (rope, *inputs(), ws)
    eager = dflash_qmm.Context(0)
    want = [a.clone() for a in work(eager, *args)]
    torch.cuda.synchronize()
    ctx = dflash_qmm.Context(0)
    graph = torch.cuda.CUDAGraph()
    announce("first rotation and accept captured")
    with torch.cuda.graph(graph):
        got = work(ctx, *args)
    for _ in range(3):
        for a in got:
            a.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(work(eager, *args), want))
    for c in (ctx, eager):
        c.close()


def test_first_calls_of_several_threads():
    rope = dflash_qmm.Rope(128)
    args = (rope, *inputs(), None)
    ctx = dflash_qmm.Context(0)
    announce("first rotations and accepts of threads")
    outs = [None] * 6

    def call(i):
        outs[i] = work(ctx, *args)
    threads = [threading.Thread(target=call, args=(i,)) for i in range(len(outs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, outs[0]))
    ctx.close()
