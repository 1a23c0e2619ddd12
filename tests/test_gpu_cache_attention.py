"""Attention of a verify block over a shared prefix and the sequences' own quantised caches
(dfq_cache_attention), against the formula in 64 bits on the values that the caches stand for.

Tolerances.  With A the largest |v| that a row sees and Z the largest sum of |q| (|s c| + |b|)
over its tokens: an output is rounded to its dtype (2^-9 or 2^-12 of itself at most, taken twice),
each probability may be rounded to 11 bits before it meets the codes, so that a token's share is
off by 2^-11 of it, and codes span at most twice A (2^-10 A in all); and a score summed in fp32 is
off by at most (head_dim + 8) 2^-24 scale Z, which is also the bound on lse.  exp and log add a few
2^-23 of the score and of lse.
"""
import math

import pytest
import torch

import dflash_qmm
from gpu_util import announce
from kv_util import DTYPES, FORMATS, attention, random_arrays

pytestmark = pytest.mark.gpu


class Case:
    """A random call: CPU arrays, their device copies and its arguments."""

    def __init__(self, seed, dim=128, bits=4, gs=64, dt="bf16", batch=1, rows=1, heads=2, group=1,
                 prefix=0, capacity=0, lengths=None, tree=False, spread=1.0, q_spread=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.dim, self.bits, self.gs, self.dtype = dim, bits, gs, DTYPES[dt]
        self.batch, self.rows, self.heads, self.group = batch, rows, heads, group
        make = lambda slots, cap: [random_arrays(gen, slots, heads, cap, dim, bits, gs,  # noqa
                                                 self.dtype, spread) for _ in range(2)]
        self.prefix = make(1, prefix) if prefix else None
        self.prefix_length = prefix
        self.own = make(batch, capacity) if capacity else None
        self.lengths = None
        if lengths is not None:
            self.lengths = torch.tensor(lengths, dtype=torch.int32)
        self.q = (torch.randn(batch, rows, heads * group, dim, generator=gen) * q_spread
                  ).to(self.dtype)
        self.tree = None
        if tree:
            self.tree = torch.randint(0, 1 << rows, (batch, rows), generator=gen).to(torch.int32)
        self.max_length = capacity
        self.scale = dim ** -0.5

    def device(self):
        side = lambda a: None if a is None else dflash_qmm.KVCache.from_arrays(  # noqa
            *[[x.cuda() for x in part] for part in a], self.bits, self.gs)
        self.d_prefix, self.d_own = side(self.prefix), side(self.own)
        self.d_q = self.q.flatten(2).cuda()
        self.d_lengths = None if self.lengths is None else self.lengths.cuda()
        self.d_tree = None if self.tree is None else self.tree.cuda()
        return self

    def run(self, ctx, **kw):
        args = dict(lengths=self.d_lengths, max_length=self.max_length, prefix=self.d_prefix,
                    prefix_length=self.prefix_length, tree=self.d_tree, scale=self.scale)
        args.update(kw)
        return ctx.cache_attention(args.pop("q", self.d_q), self.d_own, **args)

    def expected(self):
        lengths = self.lengths
        if lengths is None:
            lengths = torch.full((self.batch,), self.max_length)
        lengths = lengths.clamp(0, self.max_length)
        return attention(self.q, self.prefix, self.prefix_length, self.own, lengths, self.tree,
                         self.scale, self.bits, self.gs, self.heads)

    def check(self, y, lse, want=None):
        want_y, want_lse, worst = self.expected() if want is None else want
        y, lse = y.double().cpu().view(want_y.shape), lse.double().cpu()
        ulp = 2.0 ** -8 if self.dtype == torch.bfloat16 else 2.0 ** -11
        score = (self.dim + 8) * 2.0 ** -24 * self.scale * worst[..., 1]
        seen = torch.isfinite(want_lse)
        assert torch.equal(lse == -math.inf, want_lse == -math.inf)
        assert not y[~seen].any()
        tol = ulp * want_y.abs() + ((2.0 ** -10 + 4 * score) * worst[..., 0] + 2.0 ** -23)[..., None]
        off = (y - want_y).abs()
        assert (off[seen] <= tol[seen]).all(), float((off / tol)[seen].max())
        off = (lse - want_lse).abs()[seen]
        tol = (score + 2.0 ** -20 * (1 + want_lse.abs()))[seen]
        assert (off <= tol).all(), float((off / tol).max())


def run_case(ctx, name, **kw):
    c = Case(sum(map(ord, name)), **kw).device()
    announce(f"attention {name} {kw}")
    y, lse = c.run(ctx)
    torch.cuda.synchronize()
    c.check(y, lse)
    return c, y, lse


@pytest.mark.parametrize("dim,bits,gs,dt", FORMATS)
def test_every_format(ctx, dim, bits, gs, dt):
    run_case(ctx, f"{dim}_{bits}_{gs}_{dt}", dim=dim, bits=bits, gs=gs, dt=dt, batch=2, rows=3,
             heads=2, group=3, prefix=45, capacity=83, lengths=[83, 38])


# (batch, rows, heads, group, prefix, capacity, lengths, tree)
SHAPES = [
    (1, 1, 1, 1, 0, 1, None, False),            # one token in all
    (1, 1, 2, 5, 0, 257, None, False),          # one decoded token
    (1, 8, 2, 5, 0, 700, None, False),          # a verify block
    (3, 16, 1, 8, 0, 130, [16, 130, 77], False),
    (2, 4, 2, 2, 31, 64, [64, 33], False),      # pages that end inside a tile
    (2, 4, 2, 2, 32, 32, [4, 32], False),
    (2, 4, 2, 2, 33, 31, [31, 5], True),
    (4, 5, 1, 7, 1, 9, [5, 9, 6, 8], True),     # a prefix of one token
    (2, 3, 2, 1, 100, 0, None, False),          # a prefix alone
    (20, 7, 1, 6, 515, 40, [7 + i for i in range(20)], True),  # 840 rows share a prefix
    (9, 1, 3, 12, 1025, 3, [1, 2, 3] * 3, False),
    (2, 16, 1, 1, 4100, 50, [16, 50], True),
    (1, 2, 1, 16, 0, 5000, None, False),        # a long own cache
    (33, 16, 1, 8, 64, 20, [16 + i % 5 for i in range(33)], False),
]


@pytest.mark.parametrize("i", range(len(SHAPES)))
@pytest.mark.parametrize("dt,bits", [("bf16", 4), ("f16", 8)])
def test_shapes(ctx, i, dt, bits):
    batch, rows, heads, group, prefix, cap, lengths, tree = SHAPES[i]
    run_case(ctx, f"shape{i}_{dt}", dt=dt, bits=bits, batch=batch, rows=rows, heads=heads,
             group=group, prefix=prefix, capacity=cap, lengths=lengths, tree=tree)


@pytest.mark.parametrize("prefix", [0, 40])
def test_rows_that_see_little_or_nothing(ctx, prefix):
    """Lengths of 0, below the block's rows (its first rows are not there) and out of range, and
    draft rows whose mask is empty."""
    c = Case(11, rows=6, batch=6, heads=2, group=2, prefix=prefix, capacity=50,
             lengths=[0, 1, 5, 6, -3, 4000], tree=True)
    c.tree[3] = 0
    c.tree[5] = 0
    c.tree[2, 4] = 0
    c.device()
    announce(f"attention empty rows prefix={prefix}")
    y, lse = c.run(ctx)
    torch.cuda.synchronize()
    c.check(y, lse)
    if not prefix:
        assert (lse[0] == -math.inf).all() and not y[0].any()


@pytest.mark.parametrize("bits", [4, 8])
def test_what_hidden_tokens_hold_takes_no_part(ctx, bits):
    """NaN, infinities and the type's extremes past the lengths and in draft rows that the others
    do not see change no output, bit for bit."""
    kw = dict(bits=bits, batch=3, rows=5, heads=2, group=3, prefix=33, capacity=90,
              lengths=[90, 40, 65])
    base = Case(21, **kw)
    base.tree = torch.tensor([[1 << m | 1 for m in range(5)]] * 3, dtype=torch.int32)
    base.tree[:, 0] = 1
    base.tree[:, 4] = 1 << 1                     # row 4 sees row 1; nobody sees rows 2, 3, 4
    base.tree[:, 2:4] = 1
    want = base.device().run(ctx)
    torch.cuda.synchronize()
    base.check(*want)
    for odd in (math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).max,
                torch.finfo(torch.bfloat16).min):
        for part in base.own:
            for a in part[1:]:
                for b, n in enumerate([90, 40, 65]):
                    a[b, :, n:] = odd
                    a[b, :, n - 3:n] = odd
        announce(f"attention hidden {odd}")
        got = base.device().run(ctx)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), odd


def test_non_finite_values_reach_the_rows_that_see_them(ctx):
    """A NaN group in V spoils that group's channels of the rows that see it, and no others; one
    in K spoils the whole row."""
    c = Case(5, dim=128, gs=64, rows=4, batch=1, heads=1, group=2, capacity=60, lengths=[60])
    c.own[1][1][0, 0, 58, 1] = math.nan          # block row 2's V, upper 64 channels
    c.device()
    announce("attention NaN in V")
    y, lse = c.run(ctx)
    y = y.view(4, 2, 128)
    assert torch.isfinite(lse).all()
    assert y[2:, :, 64:].isnan().all() and torch.isfinite(y[2:, :, :64]).all()
    assert torch.isfinite(y[:2]).all()
    c.own[0][2][0, 0, 59, 0] = math.nan          # block row 3's K
    c.device()
    announce("attention NaN in K")
    y, lse = c.run(ctx)
    y = y.view(4, 2, 128)
    assert lse[0, 3].isnan().all() and y[3].isnan().all()
    assert torch.isfinite(lse[0, :3]).all() and torch.isfinite(y[:2]).all()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_peaked_flat_and_scaled_rows(ctx, dt):
    """Scores far apart and equal; queries and values of very different size within one row."""
    for seed, q_spread, spread in ((1, 30.0, 1.0), (2, 0.0, 1.0), (3, 1e-3, 50.0), (4, 1.0, 1e-3)):
        c = Case(seed, dt=dt, batch=2, rows=3, heads=2, group=2, prefix=300, capacity=200,
                 lengths=[200, 111], q_spread=q_spread, spread=spread)
        c.q[:, :, :, ::7] *= 2.0 ** -6
        c.device()
        announce(f"attention spread {dt} q={q_spread} kv={spread}")
        y, lse = c.run(ctx)
        torch.cuda.synchronize()
        c.check(y, lse)


def test_values_of_very_different_size_by_token(ctx):
    """The V scales of a sequence rise and fall by 2^12 from token to token."""
    c = Case(17, batch=1, rows=2, heads=2, group=3, prefix=260, capacity=300, lengths=[300])
    for arrays in (c.prefix[1], c.own[1]):
        for a in arrays[1:]:
            n = a.shape[2]
            a *= (2.0 ** ((torch.arange(n) * 5) % 13 - 6.0)).to(a.dtype)[None, None, :, None]
    c.device()
    announce("attention uneven V")
    y, lse = c.run(ctx)
    torch.cuda.synchronize()
    c.check(y, lse)


def test_strided_queries_streams_and_same_bits(ctx):
    c = Case(8, dim=64, gs=32, batch=3, rows=5, heads=2, group=4, prefix=70, capacity=95,
             lengths=[95, 50, 60]).device()
    want = c.run(ctx)
    again = c.run(ctx)
    torch.cuda.synchronize()
    c.check(*want)
    assert torch.equal(want[0], again[0]) and torch.equal(want[1], again[1])
    wide = torch.randn(3, 5, 3 + 8 * 64 + 6).to(torch.bfloat16).cuda()
    wide[:, :, 3:3 + 512] = c.d_q
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    announce("attention strided q on a stream")
    got = c.run(ctx, q=wide[:, :, 3:3 + 512], stream=stream)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_lengths_default_to_max_length(ctx):
    c = Case(9, batch=2, rows=2, heads=1, group=2, capacity=64)
    c.max_length = 41
    c.device()
    y, lse = c.run(ctx)
    torch.cuda.synchronize()
    c.check(y, lse)


def test_captured_call_follows_the_lengths(ctx):
    """One captured graph, replayed as the device's lengths change, with eager work between."""
    c = Case(10, batch=2, rows=4, heads=2, group=5, prefix=90, capacity=400,
             lengths=[30, 400]).device()
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    y = torch.empty_like(c.d_q)
    lse = torch.empty(2, 4, 10, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.graph_begin(stream)
    c.run(ctx, out=y, lse=lse, ws=ws, stream=stream)
    graph = ctx.graph_end(stream)
    for lengths in ([30, 400], [4, 5], [0, 399], [211, 64]):
        c.lengths = torch.tensor(lengths, dtype=torch.int32)
        c.d_lengths.copy_(c.lengths)
        torch.cuda.synchronize()
        announce(f"attention graph {lengths}")
        graph.launch(stream)
        stream.synchronize()
        c.check(y, lse)
        eager = c.run(ctx)
        torch.cuda.synchronize()
        assert torch.equal(eager[0], y) and torch.equal(eager[1], lse)


def test_offsets_past_32_bits(ctx):
    """The last slot of caches over 4 GiB."""
    slots, heads, cap, dim = 36, 8, 60000, 256
    arrays = [(torch.zeros(slots, heads, cap, 64, dtype=torch.int32, device="cuda"),
               torch.zeros(slots, heads, cap, 8, dtype=torch.bfloat16, device="cuda"),
               torch.zeros(slots, heads, cap, 8, dtype=torch.bfloat16, device="cuda"))
              for _ in range(2)]
    big = dflash_qmm.KVCache.from_arrays(*arrays, 8, 32)
    small = Case(12, dim=dim, bits=8, gs=32, batch=1, rows=2, heads=8, group=1, capacity=70,
                 lengths=[70])
    for part, full in zip(small.own, arrays):
        for a, f in zip(part, full):
            f[-1, :, cap - 70:] = a[0].cuda()
    # the tokens before them score far below: their bias is large and negative along q
    for m in range(2):
        small.q[0, m] = small.q[0, m].abs()
    arrays[0][2][-1, :, :cap - 70] = -60.0
    small.device()
    q = small.d_q.repeat(slots, 1, 1)
    announce("attention past 4 GiB")
    lengths = torch.zeros(slots, dtype=torch.int32)
    lengths[-1] = cap
    y, lse = ctx.cache_attention(q, big, lengths=lengths.cuda(), max_length=cap)
    torch.cuda.synchronize()
    small.check(y[-1:], lse[-1:])
    assert not y[:-1].any() and (lse[:-1] == -math.inf).all()


def test_refusals(ctx):
    c = Case(13, dim=64, gs=32, batch=2, rows=3, heads=2, group=2, prefix=20, capacity=30,
             lengths=[30, 7]).device()
    y = torch.empty_like(c.d_q)
    lse = torch.empty(2, 3, 4, device="cuda")
    ws = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")

    def call(**kw):
        a = dict(handle=ctx.handle, prefix=c.d_prefix.desc, prefix_length=20, cache=c.d_own.desc,
                 lengths=c.d_lengths.data_ptr(), max_length=30, tree=None, q=c.d_q.data_ptr(),
                 stride=256, y=y.data_ptr(), lse=lse.data_ptr(), batch=2, rows=3, heads=4,
                 scale=0.125, ws=ws.data_ptr(), wsb=ws.numel())
        a.update(kw)
        return ctx.lib.dfq_cache_attention(*a.values(), None)

    assert call() == 0 and call(lse=None) == 0
    assert call(handle=None) == 1 and call(q=None) == 1 and call(y=None) == 1
    assert call(prefix=None) == 1                       # a length without its cache
    assert call(cache=None) == 1 and call(cache=None, max_length=0) == 1
    assert call(cache=None, max_length=0, lengths=None, tree=ws.data_ptr()) == 1
    assert call(cache=None, max_length=0, lengths=None) == 0
    assert call(prefix_length=21) == 1 and call(prefix_length=-1) == 1
    assert call(max_length=31) == 1 and call(max_length=-1) == 1
    assert call(rows=17) == 2 and call(rows=0) == 1 and call(batch=3) == 1 and call(batch=0) == 1
    assert call(heads=3) == 1 and call(heads=0) == 1 and call(stride=255) == 1
    assert call(scale=0.0) == 1 and call(scale=-1.0) == 1
    assert call(scale=math.nan) == 1 and call(scale=math.inf) == 1
    assert call(q=c.d_q.data_ptr() + 1) == 1 and call(y=y.data_ptr() + 2) == 1
    assert call(lse=lse.data_ptr() + 2) == 1 and call(lengths=c.d_lengths.data_ptr() + 1) == 1
    for field, value in (("bits", 8), ("group_size", 64), ("heads", 1), ("dtype", 1),
                         ("head_dim", 128)):
        other = dflash_qmm.KVCache.from_arrays(c.d_prefix.k, c.d_prefix.v, 4, 32)
        setattr(other._desc, field, value)
        assert call(prefix=other.desc) == 1, field
    with pytest.raises(ValueError):
        c.run(ctx, q=c.d_q.half())
    with pytest.raises(ValueError):
        c.run(ctx, lengths=c.d_lengths.long())
    with pytest.raises(ValueError):
        c.run(ctx, tree=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        ctx.cache_attention(c.d_q)


@pytest.mark.parametrize("dim,bits,gs,dt", FORMATS)
def test_large_scores_keep_fp32(ctx, dim, bits, gs, dt):
    """With one token a row's lse is its score z.  Its products have random signs, so that the
    partial sums are some Z / sqrt(dim) (Z their sizes' sum) and each of the dim / 32 + 2 dim / gs
    additions of a matrix step or a group rounds by 2^-25 of that at most: 2^-25 Z for the errors'
    root mean square.  Eight roundings of z follow (to log2 and back, the offset off and on), and
    one of a logarithm below 2^4 (2^-21).  Large queries leave that last one small beside sums of
    fewer than 24 bits."""
    c = Case(37, dim, bits, gs, dt, batch=16, rows=1, heads=4, group=4, capacity=1,
             q_spread=64.0).device()
    announce(f"large scores dim={dim} bits={bits} gs={gs} {dt}")
    _, lse = c.run(ctx)
    _, want, worst = c.expected()
    off = (lse.double().cpu() - want).square().mean().sqrt()
    size = c.scale * worst[..., 1].mean() + 8 * want.square().mean().sqrt()
    assert off <= 2.0 ** -25 * size + 2.0 ** -21


@pytest.mark.parametrize("dim,bits,gs,dt", FORMATS)
@pytest.mark.parametrize("capacity", [83, 1571])
def test_own_caches_in_every_format(ctx, capacity, dim, bits, gs, dt):
    """Few tokens (one range, whose workgroups write the outputs) and many (several, joined)."""
    run_case(ctx, f"own{capacity}_{dim}_{bits}_{gs}_{dt}", dim=dim, bits=bits, gs=gs, dt=dt,
             batch=2, rows=5, heads=2, group=4, capacity=capacity, lengths=[capacity, 38])
