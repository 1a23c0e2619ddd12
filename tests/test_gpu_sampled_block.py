"""The rotation with its norms and the sampled accept inside whole verify passes
(examples/verify_block.py): drafts kept by their probabilities against the passes' own logits, and
the example's command."""
import os
import sys

import numpy as np
import pytest
import torch

from rotation_util import accept, check_rotated, rotated

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXAMPLES = os.path.join(ROOT, "dflash-swift_amd", "examples")
sys.path.insert(0, EXAMPLES)

SHAPE = (512, 8, 2, 64, 1024, 2000)
SEQUENCES, PROMPT = 3, 21


@pytest.fixture(scope="module")
def model(ctx):
    from verify_block import Decoder
    m = Decoder(ctx, 2, *SHAPE, SEQUENCES, PROMPT, 32, seed=5)
    gen = torch.Generator().manual_seed(6)
    tokens = torch.randint(0, SHAPE[-1], (PROMPT,), generator=gen, dtype=torch.int32).cuda()
    m.block = torch.randint(0, SHAPE[-1], (SEQUENCES, 5), generator=gen, dtype=torch.int32).cuda()
    m.numbers = torch.rand(SEQUENCES, 5, generator=gen).cuda()
    m.read_prompt(tokens)
    return m


def starts(n):
    return torch.full((SEQUENCES,), n, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("temperature", (0.0, 0.7, 1.3))
def test_drafts_are_kept_as_the_logits_say(model, temperature):
    # drafts near the likeliest tokens, so that some are kept
    seen = model.verify(model.block, starts(0))["top_tokens"]
    block = model.block.clone()
    block[:, 1] = seen[:, 0, 0]
    seen = model.verify(block, starts(0))["top_tokens"]
    block[:, 2] = seen[:, 1, 1]
    tokens, kept, chances, logits = model.sample(block, starts(0), model.numbers, temperature)
    t = np.full(SEQUENCES, temperature)
    want = accept(logits.double().cpu().numpy(), model.numbers.cpu().numpy().astype(np.float64),
                  block[:, 1:].cpu().numpy(), None, None, t, t)
    assert want[3] > 1e-9
    assert tokens.cpu().tolist() == want[0].tolist() and kept.cpu().tolist() == want[1].tolist()
    assert np.abs(chances.cpu().numpy() - want[2]).max() <= 2.0 ** -17
    if temperature == 0:
        greedy = model.verify(block, starts(0))
        assert torch.equal(greedy["accepted"], kept)
        at = kept.long()[:, None]
        assert torch.equal(tokens.gather(1, at), greedy["tokens"].gather(1, at))


def test_a_block_of_one_row_draws(model):
    tokens, kept, chances, logits = model.sample(model.block[:, :1].contiguous(), starts(0),
                                                 model.numbers[:, :1].contiguous(), 0.9)
    assert kept.tolist() == [0] * SEQUENCES and chances.shape == (SEQUENCES, 0)
    t = np.full(SEQUENCES, 0.9)
    want = accept(logits.double().cpu().numpy(), model.numbers[:, :1].cpu().numpy().astype(float),
                  None, None, None, t, t)
    assert want[3] > 1e-9 and tokens.cpu().tolist() == want[0].tolist()


def test_a_fused_projections_heads_in_a_graph(ctx, model):
    """The rotation in place beside an append and the attention, captured and replayed."""
    import dflash_qmm
    gen = torch.Generator(device="cuda").manual_seed(8)
    fused = torch.randn(2, 3, (8 + 2 * 2) * 64, device="cuda", generator=gen).bfloat16()
    source = fused.clone()
    weight = torch.randn(64, device="cuda", generator=gen).bfloat16()
    cache = dflash_qmm.KVCache(2, 2, 40, 64)
    ws = torch.empty(8 << 20, dtype=torch.uint8, device="cuda")
    begin = torch.zeros(2, dtype=torch.int32, device="cuda")

    def work():
        fused.copy_(source)
        q, k, v = fused.split((512, 128, 128), -1)
        heads = k.unflatten(-1, (2, 64))
        q, _ = ctx.qk_norm_rope(model.rope, q.unflatten(-1, (8, 64)), heads, weight, weight,
                                starts=begin, k_out=heads)
        ctx.cache_append(cache, k, v, starts=begin)
        return q, ctx.cache_attention(q.flatten(2), cache, lengths=begin + 3, max_length=40,
                                      ws=ws)[0]
    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for n in range(3):
        begin.fill_(5 * n)
        source.copy_(source.roll(1, 0))
        graph.replay()
        torch.cuda.synchronize()
        mine = [a.clone() for a in got]
        assert all(torch.equal(a, b) for a, b in zip(mine, work()))
        q = source[..., :512].unflatten(-1, (8, 64)).cpu()
        pos = (begin[:, None] + torch.arange(3, device="cuda")).cpu()
        want, size = rotated(q, pos, model.rope.frequencies, weight=weight.cpu(), eps=1e-6)
        check_rotated(mine[0], want, size, torch.bfloat16, True)


@pytest.mark.parametrize("more", ([], ["--temperature", "0.8"]))
def test_the_command_runs(more, monkeypatch, capsys):
    import verify_block
    monkeypatch.setattr(sys, "argv", ["verify_block.py", "--small", "--passes", "2", *more])
    verify_block.main()
    assert capsys.readouterr().out.count("pass ") == 2
