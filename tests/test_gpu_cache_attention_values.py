"""Attention over quantised values of very different size (dfq_cache_attention), against the formula
in 64 bits, each channel by what that channel itself holds.

Tolerances.  With p the softmax weights of a row and, in one channel, v the values and w = |s| top +
|b| their groups' extent (top the largest code): the output is rounded to its dtype (2^-9 or 2^-12 of
itself, taken twice); a weight may be rounded to 11 bits before it meets a value, code and bias alike
(2^-12 p |v| a token, taken twice); sums over codes and over biases may keep as few as 20 bits of their
own size, which is that of the groups' extent (2^-20 p w, taken four times); and a score summed in fp32
is off by at most (head_dim + 8) 2^-24 scale Z, Z the largest sum of |q| (|s c| + |b|), which every
weight shares (2 p |v| of it).
"""
import math

import pytest
import torch

import dflash_qmm
from gpu_util import announce
from kv_util import DTYPES, pack, quantise, unpack, values

pytestmark = pytest.mark.gpu


def arrays_of(x, bits, gs):
    """CPU arrays [slots][heads][tokens][..] of a cache that holds rows x [slots, heads, tokens,
    dim] of its dtype."""
    codes, scale, bias = quantise(x, bits, gs)
    return pack(codes, bits), scale, bias


class One:
    """A block of `rows` queries [rows, heads, dim] of one sequence over its cache, chain mask."""

    def __init__(self, q, k, v, bits, gs, scale=None):
        self.q, self.k, self.v, self.bits, self.gs = q, k, v, bits, gs
        self.dim = q.shape[-1]
        self.scale = self.dim ** -0.5 if scale is None else scale

    def run(self, ctx):
        cache = dflash_qmm.KVCache.from_arrays([a.cuda() for a in self.k],
                                               [a.cuda() for a in self.v], self.bits, self.gs)
        y, lse = ctx.cache_attention(self.q.flatten(1)[None].cuda(), cache, scale=self.scale)
        torch.cuda.synchronize()
        return y[0].view(self.q.shape).double().cpu(), lse[0].double().cpu()

    def expected(self):
        """(y, lse, tolerance of y, of lse) in 64 bits."""
        rows, heads, dim = self.q.shape
        ulp = 2.0 ** -8 if self.q.dtype == torch.bfloat16 else 2.0 ** -11
        y = torch.zeros(rows, heads, dim, dtype=torch.float64)
        lse = torch.zeros(rows, heads, dtype=torch.float64)
        y_tol, lse_tol = torch.zeros_like(y), torch.zeros_like(lse)
        for h in range(heads):
            k, v = (values([a[0, h] for a in part], self.bits, self.gs)
                    for part in (self.k, self.v))
            spread = lambda a: a.double().abs().repeat_interleave(self.gs, -1)  # noqa: E731
            size = unpack(self.k[0][0, h], self.bits).double() * spread(self.k[1][0, h]) + \
                spread(self.k[2][0, h])
            extent = ((1 << self.bits) - 1) * spread(self.v[1][0, h]) + spread(self.v[2][0, h])
            for m in range(rows):
                n = k.shape[0] - rows + m + 1
                q = self.q[m, h].double()
                z = (k[:n] @ q) * self.scale
                score = (dim + 8) * 2.0 ** -24 * self.scale * (size[:n] @ q.abs()).max()
                p = torch.softmax(z, 0)
                y[m, h], lse[m, h] = p @ v[:n], torch.logsumexp(z, 0)
                y_tol[m, h] = ulp * y[m, h].abs() + \
                    (2.0 ** -11 + 2 * score) * (p @ v[:n].abs()) + 2.0 ** -18 * (p @ extent[:n])
                lse_tol[m, h] = score + 2.0 ** -20 * (1 + lse[m, h].abs())
        return y, lse, y_tol, lse_tol

    def check(self, y, lse):
        want_y, want_lse, y_tol, lse_tol = self.expected()
        off = ((lse - want_lse).abs() / lse_tol)
        assert (off <= 1).all(), float(off.max())
        off = (y - want_y).abs() / y_tol.clamp_min(1e-300)
        assert (off <= 1).all(), float(off.max())


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("bits,gs,dim", [(4, 64, 128), (8, 64, 128), (4, 32, 64), (8, 128, 256)])
@pytest.mark.parametrize("offset", [4.0, 16.0, -16.0])
def test_an_outlying_channel_spoils_no_other(ctx, offset, bits, gs, dim, dt):
    """One channel of V lies far from its group's others, as V of trained models has them: theirs
    all lie at one end of the codes, whose part and the middle's cancel in them."""
    heads, rows, n = 2, 4, 200
    q = (1.5 * normal(1, rows, heads, dim)).to(DTYPES[dt])
    k = normal(2, 1, heads, n, dim).to(DTYPES[dt])
    v = 0.3 * normal(3, 1, heads, n, dim)
    v[..., 5] += offset
    c = One(q, arrays_of(k, bits, gs), arrays_of(v.to(DTYPES[dt]), bits, gs), bits, gs)
    announce(f"attention outlying channel {offset} bits={bits} gs={gs} dim={dim} {dt}")
    c.check(*c.run(ctx))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("bits,gs,dim", [(4, 64, 128), (8, 32, 256)])
def test_groups_far_from_zero(ctx, bits, gs, dim, dt):
    """V whose groups lie near zero, at 3, 40 and (bf16 holds two numbers there) 200 times their half
    range from it, and on one value, by token and group in turn."""
    heads, rows, n = 2, 5, 300
    q = (1.5 * normal(4, rows, heads, dim)).to(DTYPES[dt])
    k = normal(5, 1, heads, n, dim).to(DTYPES[dt])
    v = normal(6, 1, heads, n, dim).clamp(-1, 1).unflatten(-1, (-1, gs))
    at = torch.tensor([0.0, 3.0, -40.0, 200.0, 5.0])
    kind = torch.arange(n)[:, None] * 3 + torch.arange(dim // gs)
    v = torch.where((kind % 5 == 4)[..., None], 0.0, v) + at[kind % 5][..., None]
    c = One(q, arrays_of(k, bits, gs), arrays_of(v.flatten(-2).to(DTYPES[dt]), bits, gs), bits, gs)
    announce(f"attention far groups bits={bits} gs={gs} dim={dim} {dt}")
    c.check(*c.run(ctx))


def aimed(q, scores, scale):
    """K rows [tokens, dim] whose products with the one query q are `scores`."""
    f = q.double()
    return torch.tensor(scores).double()[:, None] * f / (scale * (f @ f))


def one_query(seed, dim, dt, scores):
    """A single row and head, and K rows with about these scores."""
    q = normal(seed, 1, 1, dim).to(DTYPES[dt])
    return q, aimed(q[0, 0], scores, dim ** -0.5)[None, None].to(DTYPES[dt])


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("power", [28, 34, 60])
@pytest.mark.parametrize("at", [3, 290])
def test_a_token_of_no_weight_and_huge_values(ctx, at, power, bits):
    """One token that the row sees has values 2^power times the others' and a weight 2^-power - 40
    of theirs: nothing of it reaches the outputs."""
    n, dim, gs = 400, 128, 64
    scores = normal(7, n)
    scores[at] = -(power + 40) * math.log(2.0)
    q, k = one_query(8, dim, "bf16", scores.tolist())
    v = normal(9, 1, 1, n, dim)
    v[0, 0, at] *= 2.0 ** power
    c = One(q, arrays_of(k, bits, gs), arrays_of(v.bfloat16(), bits, gs), bits, gs)
    announce(f"attention huge token at {at} 2^{power} bits={bits}")
    c.check(*c.run(ctx))


@pytest.mark.parametrize("size", [1e-24, 1e-12, 1e12, 1e30])
def test_small_and_large_values(ctx, size):
    q = (1.5 * normal(15, 4, 2, 128)).bfloat16()
    k = normal(16, 1, 2, 300, 128).bfloat16()
    v = (size * normal(17, 1, 2, 300, 128)).bfloat16()
    c = One(q, arrays_of(k, 4, 64), arrays_of(v, 4, 64), 4, 64)
    announce(f"attention values of size {size}")
    c.check(*c.run(ctx))


@pytest.mark.parametrize("value", [1e-30, 5.0, 1e25, -3e38])
@pytest.mark.parametrize("tokens", [1, 300])
def test_values_all_the_same(ctx, tokens, value):
    """Groups of equal elements have no scale, only a bias."""
    q = normal(13, 1, 2, 128).bfloat16()
    k = normal(14, 1, 2, tokens, 128).bfloat16()
    v = torch.full((1, 2, tokens, 128), value, dtype=torch.bfloat16)
    c = One(q, arrays_of(k, 4, 64), arrays_of(v, 4, 64), 4, 64)
    announce(f"attention equal values {value} tokens={tokens}")
    c.check(*c.run(ctx))


@pytest.mark.parametrize("scale", [1e-30, 1e-38])
def test_no_scores_and_hidden_tokens(ctx, scale):
    """Queries of zero and a tiny scale: every score is 0, and the draft chain's mask still holds."""
    q = torch.zeros(6, 2, 128, dtype=torch.bfloat16)
    k = normal(18, 1, 2, 50, 128).bfloat16()
    v = normal(19, 1, 2, 50, 128).bfloat16()
    c = One(q, arrays_of(k, 4, 64), arrays_of(v, 4, 64), 4, 64, scale=scale)
    announce(f"attention no scores scale={scale}")
    c.check(*c.run(ctx))


def test_scores_far_below_zero(ctx):
    """A row whose scores all lie below -1e30 has a softmax as any other."""
    n, dim = 70, 64
    scores = [-1e33 * (2 + i % 7) for i in range(n)]
    scores[41] = -5e32
    q, k = one_query(20, dim, "bf16", scores)
    v = normal(21, 1, 1, n, dim).bfloat16()
    c = One(q, arrays_of(k, 8, 64), arrays_of(v, 8, 64), 8, 64)
    announce("attention scores far below zero")
    y, lse = c.run(ctx)
    want_y, want_lse, _, _ = c.expected()
    assert ((lse - want_lse) / want_lse).abs().max() < 1e-4
    assert ((y - want_y).abs() <= 2.0 ** -8 * want_y.abs() + 2.0 ** -18 * v.abs().max()).all()


@pytest.mark.parametrize("bits,dt", [(4, "bf16"), (8, "f16")])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e8, 1e9, 1e12])
def test_large_scores(ctx, size, bits, dt):
    """Scores of either sign far past what fp32 holds in whole numbers: the largest alone counts,
    and lies apart from the others by more than any sum's rounding."""
    n, dim = 500, 128
    scores = (size * normal(22, n)).clamp(-2 * size, 2 * size)
    scores[77], scores[401] = 3 * size, 4 * size
    q, k = one_query(23, dim, "bf16" if size > 1e3 else dt, scores.tolist())
    dt = "bf16" if size > 1e3 else dt
    v = normal(24, 1, 1, n, dim).to(DTYPES[dt])
    c = One(q, arrays_of(k, bits, 64), arrays_of(v, bits, 64), bits, 64)
    announce(f"attention large scores {size} bits={bits} {dt}")
    y, lse = c.run(ctx)
    want_y, want_lse, _, _ = c.expected()
    ulp = 2.0 ** -8 if dt == "bf16" else 2.0 ** -11
    assert ((lse - want_lse) / want_lse).abs().max() < 1e-4
    assert ((y - want_y).abs() <= ulp * want_y.abs() + 2.0 ** -18 * v.abs().max()).all()


@pytest.mark.parametrize("dim,gs", [(64, 32), (128, 64), (256, 32)])
@pytest.mark.parametrize("power", [-50, -28, 28, 50])
def test_groups_of_very_different_size(ctx, power, dim, gs):
    """The values of every other group are 2^power times their neighbours'."""
    heads, rows, n, bits = 2, 4, 333, 4
    q = (1.5 * normal(10, rows, heads, dim)).bfloat16()
    k = normal(11, 1, heads, n, dim).bfloat16()
    v = normal(12, 1, heads, n, dim).unflatten(-1, (-1, gs))
    v[..., 1::2, :] *= 2.0 ** power
    c = One(q, arrays_of(k, bits, gs), arrays_of(v.flatten(-2).bfloat16(), bits, gs), bits, gs)
    announce(f"attention groups apart by 2^{power} dim={dim} gs={gs}")
    c.check(*c.run(ctx))
