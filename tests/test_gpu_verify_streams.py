"""The cache, attention and log-probability calls on a stream that is not torch's current one."""
import pytest
import torch

import dflash_qmm
from gpu_util import announce

pytestmark = pytest.mark.gpu


def test_outputs_that_are_dropped_are_not_the_current_streams_next(ctx):
    """Outputs of a call on a busy stream, dropped before it runs: what the current stream then
    allocates and fills keeps its values, and the outputs that were kept are right."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(4, 8, 8 * 128, device="cuda", generator=gen).bfloat16()
    own = dflash_qmm.KVCache(4, 2, 700, 128)
    rows = torch.randn(4, 700, 256, device="cuda", generator=gen).bfloat16()
    ctx.cache_append(own, rows, rows)
    logits = torch.randn(64, 5000, device="cuda", generator=gen)
    want = ctx.cache_attention(q, own)
    want_top = ctx.token_logprobs(logits, top_k=8)
    want_rows = ctx.cache_read(own, 700)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    announce("calls on a busy stream")
    for handle in (side, side.cuda_stream):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        y, _ = ctx.cache_attention(q, own, stream=handle)
        _, _, ids, _ = ctx.token_logprobs(logits, top_k=8, stream=handle)
        k, _ = ctx.cache_read(own, 700, stream=handle)
        mine = [torch.full_like(a, 7) for a in (*want, *want_top[1:], *want_rows) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(bool((a == 7).all()) for a in mine)
        assert torch.equal(y, want[0]) and torch.equal(ids, want_top[2])
        assert torch.equal(k, want_rows[0])
