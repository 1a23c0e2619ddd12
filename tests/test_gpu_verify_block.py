"""The operators of a verify pass run together (examples/verify_block.py): a prompt that all
sequences share, blocks of drafts over quantised caches, the projections in between, and the
scores of the logits.

There is no fixed result to compare a random model with, so the passes are held against each
other: a block's rows against the same tokens decoded one at a time, and the shared prompt against
the same prompt in each sequence's own cache.  Both routes quantise the same rows to the same
codes up to bf16 roundings of the layers before, and are compared by the projections' own bar for
bf16 outputs, max|d| <= 0.02 max(max|ref|, 1), per layer of two.
"""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "dflash-swift_amd", "examples"))

SHAPE = (512, 8, 2, 64, 1024, 2000)
LAYERS, SEQUENCES, PROMPT = 2, 3, 37


@pytest.fixture(scope="module")
def model(ctx):
    import torch
    from verify_block import Decoder
    m = Decoder(ctx, LAYERS, *SHAPE, SEQUENCES, PROMPT, PROMPT + 16, seed=3)
    gen = torch.Generator().manual_seed(4)
    m.tokens = torch.randint(0, SHAPE[-1], (PROMPT,), generator=gen, dtype=torch.int32).cuda()
    m.block = torch.randint(0, SHAPE[-1], (SEQUENCES, 5), generator=gen, dtype=torch.int32).cuda()
    m.read_prompt(m.tokens)
    return m


def close(a, b):
    d = (a.double() - b.double()).abs().max().item()
    return d <= LAYERS * 0.02 * max(b.abs().max().item(), 1.0)


def starts(n):
    import torch
    return torch.full((SEQUENCES,), n, dtype=torch.int32, device="cuda")


def test_a_block_is_its_tokens_one_at_a_time(model):
    import torch
    whole = model.verify(model.block, starts(0))["logits"]
    assert torch.isfinite(whole).all()
    each = torch.cat([model.verify(model.block[:, j:j + 1].contiguous(), starts(j))["logits"]
                      for j in range(model.block.shape[1])], 1)
    assert close(whole, each)


def test_a_shared_prompt_is_the_same_prompt_in_every_sequence(model):
    import torch
    shared = model.verify(model.block, starts(0))["logits"]
    tokens = model.tokens[None].expand(SEQUENCES, -1)
    for at in range(0, PROMPT, 16):
        part = tokens[:, at:at + 16].contiguous()
        n = part.shape[1]
        model.forward(part, "own", starts(at), starts(at + n), 0, PROMPT + 16)
    alone = model.forward(model.block, "own", starts(PROMPT), starts(PROMPT + 5), 0, PROMPT + 16)
    assert torch.isfinite(alone).all()
    assert close(shared, alone)


def test_drafts_are_scored_and_taken_as_the_logits_say(model):
    import torch
    got = model.verify(model.block, starts(0), top_k=3)
    p = got["logits"].double().log_softmax(-1)
    drafts = model.block[:, 1:].long()
    want = p[:, :-1].gather(-1, drafts[..., None])[..., 0]
    # fp32 sums of 2000 exponentials: well within 1e-5 of the scores' size
    assert (got["draft_logprobs"][:, :-1].double() - want).abs().max() <= 1e-5 * p.abs().max()
    assert torch.isnan(got["draft_logprobs"][:, -1]).all()
    best = got["logits"].float().max(-1).values
    taken = got["logits"].float().gather(-1, got["tokens"].long()[..., None])[..., 0]
    assert torch.equal(best, taken)
    # the model's own tokens as drafts are all accepted, up to the first that is not
    block = torch.cat((model.block[:, :1], got["tokens"][:, :1], model.block[:, 2:]), 1)
    again = model.verify(block, starts(0))
    for b in range(SEQUENCES):
        want = 0
        while want < 4 and again["tokens"][b, want] == block[b, want + 1]:
            want += 1
        assert again["accepted"][b] == want
