"""Log probabilities of given tokens, entropy and top alternatives (dfq_token_logprobs), against
log_softmax in 64 bits.

Alternatives are compared exactly.  The largest logit is exact; x - m is one rounding of an exact
difference, an exponential a few units of 2^-23 and of 2^-24 |x - m| (at most 2^-24 * 104 where it
is not zero), and sums of positive terms in fp32 by at most V threads' chains of a few hundred keep
2^-16 relative at the worst; so a log probability is within 2^-16 + 2^-23 |lp|, and the entropy
within that much of (1 + entropy).
"""
import math

import pytest
import torch

from gpu_util import announce
from kv_util import logprobs

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def check(got, want, top):
    lp, entropy, ids, best = [None if g is None else g.cpu() for g in got]

    def near(a, b, extra):
        a = a.double()
        assert torch.equal(a.isnan(), b.isnan())
        same = a == b                                  # infinities
        off = torch.where(same | b.isnan(), torch.zeros_like(b), (a - b).abs())
        tol = 2.0 ** -16 * extra + 2.0 ** -23 * torch.where(b.isfinite(), b.abs(),
                                                            torch.zeros_like(b))
        assert (off <= tol).all(), float((off / tol).max())

    near(lp, want[0], torch.ones_like(want[0]))
    near(entropy, want[1], 1 + want[1].abs().nan_to_num(0.0))  # where NaN is due, it is compared above
    if top:
        assert torch.equal(ids.long(), want[2])
        near(best, want[3], torch.ones_like(want[3]))
    else:
        assert ids is None and best is None


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("M,V,top", [(1, 1, 1), (1, 2, 5), (3, 7, 32), (2, 255, 4), (5, 256, 0),
                                     (4, 257, 32), (1, 4099, 20), (17, 1000, 5), (2, 33001, 32),
                                     (1, 151936, 5), (300, 513, 1)])
def test_shapes(ctx, M, V, top, dt):
    gen = torch.Generator().manual_seed(M * 7 + V)
    x = (3 * torch.randn(M, V, generator=gen)).to(DT[dt])
    tokens = torch.randint(0, V, (M,), generator=gen).to(torch.int32)
    announce(f"logprobs M={M} V={V} top={top} {dt}")
    got = ctx.token_logprobs(x.cuda(), tokens.cuda(), top_k=top)
    torch.cuda.synchronize()
    check(got, logprobs(x, tokens, top), top)


ODD_V = [40, 5000]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("V", ODD_V)
def test_odd_rows(ctx, dt, V):
    """Ties, one number, banned tokens, masks of the type's lowest value, infinities and NaN."""
    gen = torch.Generator().manual_seed(V)
    low = torch.finfo(DT[dt]).min
    rows = [
        torch.zeros(V),                                            # all equal
        torch.full((V,), -math.inf),                               # nothing
        torch.full((V,), low),                                     # all at the lowest value
        torch.full((V,), math.nan),
        torch.randint(0, 3, (V,), generator=gen).float(),          # many ties
        torch.arange(V).float() / 64,                              # rising
        -torch.arange(V).float() / 64,                             # falling
        torch.where(torch.arange(V) % 3 == 0, torch.randn(V, generator=gen),
                    torch.tensor(-math.inf)),                      # banned tokens
        torch.where(torch.arange(V) % 5 == 1, torch.randn(V, generator=gen), torch.tensor(low)),
        torch.full((V,), -math.inf).index_fill(0, torch.tensor([V - 1]), 2.5),  # one number
        torch.randn(V, generator=gen).index_fill(0, torch.tensor([V // 2]), math.nan),
        torch.randn(V, generator=gen).index_fill(0, torch.tensor([3]), math.inf),
        torch.randn(V, generator=gen).index_fill(0, torch.tensor([3, V - 2]), math.inf),
        torch.randn(V, generator=gen) - 30000.0,
        torch.where(torch.arange(V) % 2 == 0, torch.tensor(0.0), torch.tensor(-0.0)),
        torch.full((V,), math.nan).index_fill(0, torch.tensor([1, 9]), -4.0),
        1e4 * torch.randn(V, generator=gen),
    ]
    x = torch.stack(rows).to(DT[dt])
    tokens = torch.tensor([0, 1, 2, 3, V - 1, V - 1, 0, 1, 2, V - 1, 5, 3, 4, 5, -1, V, 2 ** 31 - 1],
                          dtype=torch.int32)
    for top in (1, 9, 32):
        announce(f"logprobs odd V={V} top={top} {dt}")
        got = ctx.token_logprobs(x.cuda(), tokens.cuda(), top_k=top)
        torch.cuda.synchronize()
        check(got, logprobs(x, tokens, top), top)


@pytest.mark.parametrize("dt", list(DT))
def test_sorted_long_rows(ctx, dt):
    """Rising, falling and constant rows of a real vocabulary: the alternatives in one place, or
    every element ahead of all before it."""
    V = 40000
    up = torch.linspace(-20, 20, V)
    x = torch.stack([up, -up, torch.ones(V), up.roll(V // 3)]).to(DT[dt])
    tokens = torch.tensor([V - 1, 0, 5, 17], dtype=torch.int32)
    announce(f"logprobs sorted {dt}")
    got = ctx.token_logprobs(x.cuda(), tokens.cuda(), top_k=32)
    torch.cuda.synchronize()
    check(got, logprobs(x, tokens, 32), 32)


def test_strided_rows_and_streams(ctx):
    gen = torch.Generator().manual_seed(1)
    wide = torch.randn(6, 1300, generator=gen).to(torch.bfloat16)
    dev = wide.cuda()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    announce("logprobs strided")
    tokens = torch.arange(6, dtype=torch.int32)
    dtok = tokens.cuda()
    torch.cuda.synchronize()
    got = ctx.token_logprobs(dev[:, 3:1204], dtok, top_k=7, stream=stream)
    again = ctx.token_logprobs(dev[:, 3:1204], dtok, top_k=7, stream=stream)
    stream.synchronize()
    check(got, logprobs(wide[:, 3:1204], tokens, 7), 7)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_same_tokens_as_the_greedy_accept(ctx):
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(8, 30000, generator=gen).to(torch.bfloat16).cuda()
    tokens, _ = ctx.argmax_accept(x)
    announce("logprobs of the accepted tokens")
    lp, _, ids, top = ctx.token_logprobs(x, tokens, top_k=1)
    torch.cuda.synchronize()
    assert torch.equal(ids[:, 0], tokens) and torch.equal(top[:, 0], lp)


def test_captured_call(ctx):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(4, 20000, generator=gen).to(torch.float16)
    dev, tokens = x.cuda(), torch.tensor([1, 2, 3, 4], dtype=torch.int32).cuda()
    ws = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.graph_begin(stream)
    got = ctx.token_logprobs(dev, tokens, top_k=6, ws=ws, stream=stream)
    graph = ctx.graph_end(stream)
    for step in range(3):
        x = torch.randn(4, 20000, generator=gen).to(torch.float16)
        dev.copy_(x)
        torch.cuda.synchronize()
        announce(f"logprobs graph {step}")
        graph.launch(stream)
        stream.synchronize()
        check(got, logprobs(x, tokens.cpu(), 6), 6)


def test_refusals(ctx):
    x = torch.zeros(3, 50, dtype=torch.bfloat16, device="cuda")
    f = torch.zeros(3 * 64, device="cuda")
    i = torch.zeros(3 * 64, dtype=torch.int32, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

    def call(**kw):
        a = dict(handle=ctx.handle, logits=x.data_ptr(), stride=50, M=3, V=50, dt=0,
                 tokens=i.data_ptr(), top=2, lp=f.data_ptr(), entropy=f.data_ptr(),
                 ids=i.data_ptr(), best=f.data_ptr(), ws=ws.data_ptr(), wsb=ws.numel())
        a.update(kw)
        return ctx.lib.dfq_token_logprobs(*a.values(), None)

    assert call(handle=None) == 1 and call(logits=None) == 1 and call(M=0) == 1 and call(V=0) == 1
    assert call(stride=49) == 1 and call(dt=3) == 2 and call(top=33) == 2 and call(top=-1) == 2
    assert call(V=1 << 30, stride=1 << 30) == 2
    assert call(lp=None) == 1 and call(ids=None) == 1 and call(best=None) == 1
    assert call(tokens=None, entropy=None, top=0) == 1
    assert call(logits=x.data_ptr() + 1) == 1 and call(entropy=f.data_ptr() + 2) == 1
    with pytest.raises(ValueError):
        ctx.token_logprobs(x.t())
    with pytest.raises(ValueError):
        ctx.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(dflash_qmm_error()):
        ctx.token_logprobs(x, top_k=33)


def dflash_qmm_error():
    import dflash_qmm
    return dflash_qmm.DfqError


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("M,V,top", [(700, 9001, 20), (1300, 2503, 32), (6, 100003, 32)])
def test_many_rows_and_long_joins(ctx, M, V, top, dt):
    """More rows than workgroups are there at once (each row one workgroup's), and few long rows
    with more alternatives in their parts than one piece of the join holds."""
    gen = torch.Generator().manual_seed(M + V)
    few = (3 * torch.randn(2, V, generator=gen)).to(DT[dt])
    tokens = torch.randint(0, V, (2,), generator=gen).to(torch.int32)
    announce(f"logprobs M={M} V={V} top={top} {dt}")
    got = ctx.token_logprobs(few.repeat(M // 2, 1).cuda(), tokens.repeat(M // 2).cuda(), top_k=top)
    torch.cuda.synchronize()
    want = [w.repeat(M // 2, *[1] * (w.dim() - 1)) for w in logprobs(few, tokens, top)]
    check(got, want, top)
