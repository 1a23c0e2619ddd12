"""The rotary positions and the head norms with them against 64-bit plain forms: head widths,
rotated widths, pairs, positions, strides, outputs in place, and calls that refuse."""
import itertools
import math

import pytest
import torch

import dflash_qmm
from gpu_util import announce
from rotation_util import DTYPES, check_rotated, rotated

pytestmark = pytest.mark.gpu


def run(ctx, rope, q, k, norms=None, inverse=False, offset=0, seed=0, **where):
    """One call against the plain forms."""
    if norms is None:
        got = ctx.rope(rope, q, k, inverse=inverse, **where)
        weights = (None, None)
    else:
        weights = norms
        got = ctx.qk_norm_rope(rope, q, k, *weights, eps=1e-6, weight_offset=offset, **where)
    torch.cuda.synchronize()
    batch, rows = q.shape[:2]
    if "positions" in where:
        pos = where["positions"].cpu().long()
    else:
        pos = torch.arange(rows).expand(batch, -1) + where.get("start", 0)
        if where.get("starts") is not None:
            pos = pos + where["starts"].cpu().long()[:, None]
    if k is None:
        got = (got,)
    for x, y, w in zip((q, k), got, weights):
        assert y.dtype == x.dtype and y.shape == x.shape
        want, size = rotated(x.cpu(), pos, rope.frequencies, rope.amplitude, rope.interleaved,
                             inverse, None if w is None else w.cpu(), offset,
                             None if norms is None else 1e-6)
        check_rotated(y, want, size, x.dtype, norms is not None)
    return got


def heads(gen, batch, rows, n, dim, dtype):
    x = torch.randn(batch, rows, n, dim, device="cuda", generator=gen)
    return (x * torch.exp(torch.randn(dim, device="cuda", generator=gen))).to(dtype)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# every way to hold a head: chunks of 16 channels over 1 .. 32 lanes with idle ones among them, and
# what has to go pair by pair
WIDTHS = [(2, 2), (6, 4), (16, 16), (32, 16), (48, 48), (64, 64), (64, 20), (80, 32), (80, 40),
          (96, 24), (112, 112), (128, 128), (128, 64), (192, 128), (256, 64), (256, 256),
          (300, 298), (512, 512), (512, 128)]


@pytest.mark.parametrize("dim,rotary", WIDTHS)
@pytest.mark.parametrize("name", sorted(DTYPES))
def test_widths(ctx, dim, rotary, name):
    announce(f"rope dim {dim} rotary {rotary} {name}")
    gen = generator(dim + rotary)
    for interleaved, normed in itertools.product((False, True), (False, True)):
        rope = dflash_qmm.Rope(rotary, base=1e4, interleaved=interleaved)
        q, k = (heads(gen, 2, 3, n, dim, DTYPES[name]) for n in (5, 2))
        starts = torch.tensor([0, 70001], dtype=torch.int32, device="cuda")
        norms = None
        if normed:
            norms = [torch.randn(dim, device="cuda", generator=gen).to(DTYPES[name])
                     for _ in range(2)]
        run(ctx, rope, q, k, norms, starts=starts)


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("interleaved", (False, True))
def test_positions(ctx, name, interleaved):
    announce(f"rope positions {name} {interleaved}")
    gen = generator(5)
    rope = dflash_qmm.Rope(32, base=1e6, interleaved=interleaved)
    far = [0, 1, -1, 2, 1000000, -1000000, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1]
    pos = torch.tensor([far], dtype=torch.int32, device="cuda")
    q, k = (heads(gen, 1, len(far), n, 64, DTYPES[name]) for n in (3, 1))
    for inverse in (False, True):
        run(ctx, rope, q, k, inverse=inverse, positions=pos)
    # start and starts are added without wrapping
    starts = torch.tensor([2 ** 31 - 3], dtype=torch.int32, device="cuda")
    run(ctx, rope, q, k, start=2 ** 31 - 1, starts=starts)
    run(ctx, rope, q, k, start=-2 ** 31 + 1, starts=-starts)
    run(ctx, rope, q, k, start=17)
    run(ctx, rope, q, k)


def test_turning_back_is_the_inverse(ctx):
    """R^T R x = x to the fp32 arithmetic's bound, twice."""
    gen = generator(6)
    rope = dflash_qmm.Rope(128, base=1e6)
    q = heads(gen, 3, 40, 6, 128, torch.float32)
    there = ctx.rope(rope, q, start=123456)
    back = ctx.rope(rope, there, start=123456, inverse=True)
    size = q.abs() + torch.cat((q[..., 64:], q[..., :64]), -1).abs()
    assert bool(((back - q).abs() <= 2.0 * size * 2.0 ** -20).all())


@pytest.mark.parametrize("scaling", [
    {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
    {"type": "bands", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_length": 8192},
    {"type": "yarn", "factor": 4.0, "original_length": 32768}])
def test_scaled(ctx, scaling):
    gen = generator(7)
    rope = dflash_qmm.Rope(64, base=5e5, scaling=scaling)
    q, k = (heads(gen, 2, 5, n, 128, torch.bfloat16) for n in (4, 4))
    run(ctx, rope, q, k, start=99999)
    given = dflash_qmm.Rope(64, frequencies=rope.frequencies, amplitude=rope.amplitude)
    assert torch.equal(given.turns, rope.turns)
    free = dflash_qmm.Rope(64, frequencies=[(-1) ** i * 3.0 * i for i in range(32)], amplitude=-0.5)
    run(ctx, free, q, k, start=12345)


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("dim,rotary", [(128, 128), (64, 20)])
def test_slices_of_fused_rows(ctx, name, dim, rotary):
    """Heads cut from fused rows at odd element offsets, whose neighbours stay as they were, into
    outputs in place and into slices of another tensor."""
    announce(f"rope slices {name} {dim}")
    gen = generator(8)
    dt = DTYPES[name]
    batch, rows, hq, hk = 2, 7, 6, 2
    rope = dflash_qmm.Rope(rotary, interleaved=rotary == 20)
    norms = [torch.randn(dim, device="cuda", generator=gen) for _ in range(2)]
    for offset, normed in itertools.product((0, 1, 3), (False, True)):
        fused = torch.randn(batch, rows, (hq + 2 * hk) * dim + 5, device="cuda",
                            generator=gen).to(dt)
        before = fused.clone()
        q = fused[..., offset:offset + hq * dim].unflatten(-1, (hq, dim))
        k = fused[..., offset + hq * dim:offset + (hq + hk) * dim].unflatten(-1, (hk, dim))
        want = run(ctx, rope, q, k, norms if normed else None)
        call = (lambda **kw: ctx.qk_norm_rope(rope, q, k, *norms, **kw)) if normed else \
            (lambda **kw: ctx.rope(rope, q, k, **kw))
        other = torch.full_like(fused, 7)
        call(q_out=other[..., 1:1 + hq * dim].unflatten(-1, (hq, dim)),
             k_out=other[..., 1 + hq * dim:1 + (hq + hk) * dim].unflatten(-1, (hk, dim)))
        call(q_out=q, k_out=k)
        torch.cuda.synchronize()
        for a, b in zip((q, k), want):
            assert torch.equal(a, b)
        wide = (hq + hk) * dim
        assert torch.equal(other[..., 1:1 + wide], fused[..., offset:offset + wide])
        assert bool((other[..., :1] == 7).all()) and bool((other[..., 1 + wide:] == 7).all())
        assert torch.equal(fused[..., :offset], before[..., :offset])
        assert torch.equal(fused[..., offset + wide:], before[..., offset + wide:])


def test_other_orders(ctx):
    """Heads in front of rows, and inputs that all sequences share (a stride of 0)."""
    gen = generator(9)
    rope = dflash_qmm.Rope(64)
    x = torch.randn(3, 4, 9, 64, device="cuda", generator=gen).bfloat16()   # [batch, heads, rows]
    starts = torch.tensor([5, 0, 9], dtype=torch.int32, device="cuda")
    q = x.transpose(1, 2)
    want = run(ctx, rope, q, None, starts=starts)[0]
    out = torch.empty_like(x)
    ctx.rope(rope, q, starts=starts, q_out=out.transpose(1, 2))
    assert torch.equal(out.transpose(1, 2), want)
    shared = x[:1].transpose(1, 2).expand(3, -1, -1, -1)
    run(ctx, rope, shared, shared[:, :, 1:3], starts=starts)


@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("dim,rotary", [(256, 64), (64, 20), (32, 12)])
def test_what_is_behind_the_rotated_channels_stays(ctx, dim, rotary, interleaved):
    gen = generator(10)
    rope = dflash_qmm.Rope(rotary, interleaved=interleaved, amplitude=2.0)
    q = heads(gen, 2, 5, 3, dim, torch.bfloat16)
    q[..., rotary::3] = math.inf
    q[..., rotary + 1::3] = math.nan
    got = ctx.rope(rope, q, start=3)
    assert torch.equal(got[..., rotary:].view(torch.int16), q[..., rotary:].view(torch.int16))
    assert bool(torch.isfinite(got[..., :rotary]).all())


def test_values_without_size(ctx):
    """Heads of zeros, of the least and the largest numbers, and with an infinity in them."""
    gen = generator(11)
    rope = dflash_qmm.Rope(128)
    for name, dt in DTYPES.items():
        f = torch.finfo(dt)
        q = heads(gen, 1, 6, 2, 128, dt)
        q[:, 0] = 0
        q[:, 1] = f.smallest_normal * f.eps * 3
        q[:, 2] *= 1e-4 / q[:, 2].float().abs().amax().item()
        w = torch.randn(128, device="cuda", generator=gen).to(dt)
        run(ctx, rope, q, None, (w, None), start=2)
        if dt != torch.float16:
            # sums of squares past fp32 come out as 0
            q[:, 3] = 1e30
            assert not ctx.qk_norm_rope(rope, q, None, w)[:, 3].any()
        q[:, 4, 0, 9] = math.inf
        q[:, 4, 1, 9] = math.nan
        y = ctx.qk_norm_rope(rope, q, None, w)
        assert bool(torch.isnan(y[:, 4, 1]).all())
        assert bool(torch.isfinite(y[:, 5]).all())


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("dim,rotary", [(128, 128), (256, 64), (6, 4)])
def test_norms(ctx, name, dim, rotary):
    """Weights in either dtype, at any address, as distances from 1, and left out."""
    announce(f"norms {name} {dim}")
    gen = generator(12)
    dt = DTYPES[name]
    rope = dflash_qmm.Rope(rotary)
    q, k = (heads(gen, 3, 5, n, dim, dt) for n in (8, 2))
    for kind in (dt, torch.float32):
        weights = [torch.randn(dim + 1, device="cuda", generator=gen).to(kind)[1:]
                   for _ in range(2)]
        for offset in (0.0, 1.0):
            run(ctx, rope, q, k, weights, offset=offset, start=7)
        run(ctx, rope, q, k, (weights[0], None), start=7)
        run(ctx, rope, q, None, (weights[0], None), start=7)
    run(ctx, rope, q, k, (None, None), start=7)
    # the norms alone, as the plain form with a rotation by nothing has them (bits may differ from
    # those of a rotation by nothing here, whose lanes hold other channels and sum them in another
    # order)
    got = ctx.qk_norm_rope(None, q, k, *weights)
    for x, y, w in zip((q, k), got, weights):
        want, size = rotated(x.cpu(), torch.zeros(3, 5, dtype=torch.long), [0.0] * (rotary // 2),
                             weight=w.cpu(), eps=1e-6)
        check_rotated(y, want, size, dt, True)


@pytest.mark.parametrize("batch,rows", [(1, 1), (1, 1000), (300, 1), (7, 33)])
def test_counts(ctx, batch, rows):
    """From one token to many: every head of every token is the single token's."""
    gen = generator(13)
    rope = dflash_qmm.Rope(128, base=1e6)
    q, k = (heads(gen, batch, rows, n, 128, torch.bfloat16) for n in (5, 1))
    w = [torch.randn(128, device="cuda", generator=gen).bfloat16() for _ in range(2)]
    pos = torch.randint(0, 100000, (batch, rows), generator=torch.Generator().manual_seed(1),
                        dtype=torch.int32).cuda()
    for call in (lambda q, k, p: ctx.rope(rope, q, k, positions=p),
                 lambda q, k, p: ctx.qk_norm_rope(rope, q, k, *w, positions=p)):
        got = call(q, k, pos)
        for b, m in {(0, 0), (batch - 1, rows - 1), (batch // 2, rows // 2)}:
            one = call(q[b:b + 1, m:m + 1], k[b:b + 1, m:m + 1], pos[b:b + 1, m:m + 1].contiguous())
            assert all(torch.equal(x[b, m], y[0, 0]) for x, y in zip(got, one))


def test_offsets_past_32_bits(ctx):
    """Sequences, rows and heads that lie more than 2^31 elements apart."""
    size = 2 ** 31 + 4096
    big = torch.empty(size, dtype=torch.bfloat16, device="cuda")
    rope = dflash_qmm.Rope(128)
    gen = generator(14)
    x = torch.randn(2, 1, 1, 128, device="cuda", generator=gen).bfloat16()
    want = ctx.rope(rope, x, start=11)
    far = 2 ** 31 + 64
    for shape, strides in (((2, 1, 1, 128), (far, 128, 128, 1)),
                           ((1, 2, 1, 128), (far, far, 128, 1)),
                           ((1, 1, 2, 128), (far, far, far, 1))):
        view = big.as_strided(shape, strides)
        view.copy_(x.view(shape))
        pos = torch.full(shape[:2], 11, dtype=torch.int32, device="cuda")
        announce(f"rope far {shape}")
        assert torch.equal(ctx.rope(rope, view, positions=pos).view(-1), want.view(-1))
        ctx.rope(rope, view, positions=pos, q_out=view)
        assert torch.equal(view.reshape(-1), want.view(-1))
    del big


def test_captured_and_replayed(ctx):
    gen = generator(15)
    rope = dflash_qmm.Rope(128)
    q, k = (heads(gen, 4, 8, n, 128, torch.bfloat16) for n in (8, 2))
    w = [torch.randn(128, device="cuda", generator=gen).bfloat16() for _ in range(2)]
    starts = torch.zeros(4, dtype=torch.int32, device="cuda")

    def both():
        return (*ctx.rope(rope, q, k, starts=starts),
                *ctx.qk_norm_rope(rope, q, k, *w, starts=starts))
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for n in range(3):
        starts.fill_(1000 * n)
        q.copy_(q.roll(1, 0))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, both()))


def test_another_stream(ctx):
    """Outputs of a call on a busy stream, dropped before it runs, are not the current one's."""
    gen = generator(16)
    rope = dflash_qmm.Rope(128)
    q, k = (heads(gen, 4, 64, n, 128, torch.bfloat16) for n in (8, 2))
    want = ctx.rope(rope, q, k)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    y, _ = ctx.rope(rope, q, k, stream=side)
    mine = [torch.full_like(a, 7) for a in want for _ in range(3)]
    torch.cuda.synchronize()
    assert all(bool((a == 7).all()) for a in mine) and torch.equal(y, want[0])
