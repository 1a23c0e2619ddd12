"""Rotations of so many heads that a lane turns several of them: against the 64-bit plain form, against
calls in which it turns one, into fresh outputs and in place over fused rows."""
import pytest
import torch

import dflash_qmm
from gpu_util import announce
from rotation_util import DTYPES, check_rotated, rotated

pytestmark = pytest.mark.gpu

# heads, rotated channels, heads of queries and of keys, heads a lane: counts that the latter does not
# divide, fewer heads than that, lanes of a head that hold nothing (80), 1 to 32 lanes a head
CASES = [(128, 128, 7, 3, 2), (128, 64, 17, 1, 3), (128, 128, 17, 3, 16), (80, 32, 7, 1, 4),
         (256, 64, 16, 2, 3), (512, 512, 5, 2, 6), (512, 128, 17, 3, 16), (64, 64, 7, 3, 16),
         (16, 16, 7, 3, 2), (48, 48, 9, 2, 5)]


def lanes_of(dim):
    n = 1
    while 16 * n < dim:
        n *= 2
    return n


def heads_a_lane(cus, tokens, heads, dim):
    return min(max(tokens * heads * lanes_of(dim) // 64 // (8 * cus), 1), 16)


@pytest.mark.parametrize("normed", (False, True))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("dim,rotary,q_heads,k_heads,each", CASES)
def test_lanes_of_several_heads(ctx, dim, rotary, q_heads, k_heads, each, name, interleaved, normed):
    announce(f"rope {dim} {rotary} {q_heads} {k_heads} {each} {name} {interleaved} {normed}")
    gen = torch.Generator(device="cuda").manual_seed(41)
    dt, heads, cus = DTYPES[name], q_heads + k_heads, ctx.num_cus
    batch = 3
    rows = -(-8 * cus * each * 64 // lanes_of(dim) // heads // batch) + 5
    tokens = batch * rows
    assert heads_a_lane(cus, tokens, heads, dim) == each
    rope = dflash_qmm.Rope(rotary, base=1e6, interleaved=interleaved)
    fused = torch.randn(batch, rows, (heads + k_heads) * dim, device="cuda", generator=gen).to(dt)
    positions = torch.randint(0, 200000, (batch, rows), device="cuda", generator=gen,
                              dtype=torch.int32)
    weights = [(1 + 0.3 * torch.randn(dim, device="cuda", generator=gen)).to(dt) for _ in range(2)]

    def cut(x):
        q, k, v = x.split((q_heads * dim, k_heads * dim, k_heads * dim), -1)
        return q.unflatten(-1, (q_heads, dim)), k.unflatten(-1, (k_heads, dim)), v

    def call(q, k, positions, **out):
        if normed:
            return ctx.qk_norm_rope(rope, q, k, *weights, positions=positions, **out)
        return ctx.rope(rope, q, k, positions=positions, **out)

    q, k, v = cut(fused)
    got = call(q, k, positions)
    # all tokens, as calls in which a lane has one head make them
    flat = [x.reshape(1, tokens, *x.shape[2:]) for x in (q, k)]
    step = 16 * cus * 64 // lanes_of(dim) // heads - 1
    assert heads_a_lane(cus, step, heads, dim) == 1
    for at in range(0, tokens, step):
        part = [x[:, at:at + step] for x in flat]
        one = call(*part, positions.view(1, -1)[:, at:at + step].contiguous())
        for x, y in zip(got, one):
            assert torch.equal(x.reshape(1, tokens, *x.shape[2:])[:, at:at + step], y), at
    # some tokens of every third of the call, as the plain form has them
    some = torch.randint(0, tokens, (12,), generator=torch.Generator().manual_seed(2))
    some[0], some[1] = 0, tokens - 1
    pos = positions.view(-1).cpu()[some].view(1, -1)
    for x, y, w in zip((q, k), got, weights):
        x, y = (a.reshape(tokens, *a.shape[2:])[some.cuda()][None].cpu() for a in (x, y))
        want, size = rotated(x, pos, rope.frequencies, interleaved=interleaved,
                             weight=w.cpu() if normed else None, eps=1e-6 if normed else None)
        check_rotated(y, want, size, dt, normed)
    # in place over the fused rows, whose last part stays
    again = fused.clone()
    aq, ak, av = cut(again)
    call(aq, ak, positions, q_out=aq, k_out=ak)
    assert torch.equal(aq, got[0]) and torch.equal(ak, got[1]) and torch.equal(av, v)
