"""The quantised key/value cache: rows quantised as they are written (dfq_cache_append) and read
back (dfq_cache_read), against the format's definition.

Codes, scales and biases are compared bit for bit: the definition is a fixed sequence of fp32
operations, each rounded once.  Values read back are scale * code + bias, whose product is exact
in fp32: one rounding to fp32 and one to a 16-bit dtype, compared bit for bit too.
"""
import math

import pytest
import torch

import dflash_qmm
from gpu_util import announce
from kv_util import DTYPES, FORMATS, pack, quantise, unpack

pytestmark = pytest.mark.gpu


def rows_of(gen, batch, rows, width, dtype):
    x = torch.randn(batch, rows, width, generator=gen) * 2.0
    return (x + torch.randn(width, generator=gen)).to(dtype)


def same(got, want):
    """Bit for bit, NaN equal to NaN."""
    return bool(((got == want) | (got.isnan() & want.isnan())).all()) if got.is_floating_point() \
        else torch.equal(got, want)


def check_written(cache, k, v, starts, rows):
    """Every position of every slot: the written ones by the definition, the others untouched."""
    for name, x, arrays in (("k", k, cache.k), ("v", v, cache.v)):
        batch = x.shape[0]
        x = x.view(batch, rows, cache.heads, cache.head_dim).transpose(1, 2)
        codes, scale, bias = quantise(x, cache.bits, cache.group_size)
        want = [torch.full_like(a, 77).cpu() for a in arrays]
        for b in range(batch):
            for m in range(rows):
                pos = starts[b] + m
                if 0 <= pos < cache.capacity:
                    for w, part in zip(want, (pack(codes, cache.bits), scale, bias)):
                        w[b, :, pos] = part[b, :, m]
        for w, a, part in zip(want, arrays, ("codes", "scales", "biases")):
            assert same(a.cpu(), w), (name, part)


def filled_cache(*args, **kw):
    cache = dflash_qmm.KVCache(*args, **kw)
    for a in (*cache.k, *cache.v):
        a.fill_(77)
    return cache


@pytest.mark.parametrize("dim,bits,gs,dt", FORMATS)
def test_append_and_read_every_format(ctx, dim, bits, gs, dt):
    gen = torch.Generator().manual_seed(dim + bits + gs)
    dtype, heads, batch, rows, cap = DTYPES[dt], 3, 2, 37, 53
    announce(f"append d={dim} b={bits} g={gs} {dt}")
    cache = filled_cache(3, heads, cap, dim, bits, gs, dtype)
    k, v = (rows_of(gen, batch, rows, heads * dim, dtype) for _ in range(2))
    starts = torch.tensor([4, 11], dtype=torch.int32)
    ctx.cache_append(cache, k.cuda(), v.cuda(), start=1, starts=starts.cuda())
    torch.cuda.synchronize()
    check_written(cache, k, v, [5, 12], rows)
    for out in (dtype, torch.float32):
        got = ctx.cache_read(cache, rows, start=1, starts=starts.cuda(), dtype=out)
        torch.cuda.synchronize()
        for x, y in zip((k, v), got):
            x = x.view(batch, rows, heads, dim)
            codes, scale, bias = quantise(x, bits, gs)
            c = codes.float().unflatten(-1, (-1, gs))
            want = (c * scale.float()[..., None] + bias.float()[..., None]).flatten(-2).to(out)
            assert same(y.cpu(), want)


@pytest.mark.parametrize("batch,rows", [(1, 1), (5, 1), (1, 16), (2, 17), (1, 300)])
def test_rows_cut_from_a_fused_output(ctx, batch, rows):
    """K and V as slices of a wider row, at an odd element offset, on a stream of their own."""
    gen = torch.Generator().manual_seed(batch * 1000 + rows)
    heads, dim = 2, 128
    fused = rows_of(gen, batch, rows, 1 + 3 * heads * dim + 5, torch.bfloat16)
    announce(f"append fused batch={batch} rows={rows}")
    cache = filled_cache(batch, heads, rows + 3, dim, 4, 64, torch.bfloat16)
    dev = fused.cuda()
    torch.cuda.synchronize()
    k, v = (dev[:, :, a:a + heads * dim] for a in (1, 1 + 2 * heads * dim))
    stream = torch.cuda.Stream()
    ctx.cache_append(cache, k, v, start=2, stream=stream)
    got = ctx.cache_read(cache, rows, start=2, stream=stream)
    stream.synchronize()
    check_written(cache, k.cpu().contiguous(), v.cpu().contiguous(), [2] * batch, rows)
    assert got[0].shape == (batch, rows, heads, dim)


def test_positions_outside_the_cache(ctx):
    """Rows before 0 and past the capacity are not written, and read as zero."""
    gen = torch.Generator().manual_seed(3)
    heads, dim, rows, cap = 2, 64, 9, 12
    cache = filled_cache(3, heads, cap, dim, 8, 32, torch.float16)
    k, v = (rows_of(gen, 3, rows, heads * dim, torch.float16) for _ in range(2))
    starts = torch.tensor([-4, 7, 2147483647], dtype=torch.int32)
    announce("append outside the cache")
    ctx.cache_append(cache, k.cuda(), v.cuda(), starts=starts.cuda())
    got = ctx.cache_read(cache, rows, starts=starts.cuda())
    torch.cuda.synchronize()
    check_written(cache, k, v, starts.tolist(), rows)
    for b, first in enumerate(starts.tolist()):
        for m in range(rows):
            if not 0 <= first + m < cap:
                assert not got[0][b, m].any() and not got[1][b, m].any()
            else:
                assert got[0][b, m].any()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_groups_of_equal_extreme_and_odd_elements(ctx, dt):
    dtype = DTYPES[dt]
    big = 65504.0 if dt == "f16" else 3.3e38
    x = torch.zeros(1, 9, 64, dtype=dtype)
    x[0, 0] = 1.5                                    # equal elements
    x[0, 1, ::2] = -0.0                              # zeros of both signs
    x[0, 2, 5] = math.nan
    x[0, 3, 40] = math.inf
    x[0, 4, 3] = -math.inf
    x[0, 5, 0], x[0, 5, 1] = big, -big               # a range past fp32 in bf16, not in fp16
    x[0, 6] = torch.arange(64).to(dtype) * 2.0 ** -24  # denormal scales in fp16
    x[0, 7, 9] = -big
    x[0, 8] = torch.linspace(-1, 1, 64).to(dtype)
    announce(f"append odd groups {dt}")
    for bits in (4, 8):
        cache = filled_cache(1, 1, 9, 64, bits, 32, dtype)
        ctx.cache_append(cache, x.cuda(), x.cuda())
        got = ctx.cache_read(cache, 9)[0].cpu()[0, :, 0]
        check_written(cache, x, x, [0], 9)
        for r, group in ((2, 0), (3, 1), (4, 0)):
            half = got[r, 32 * group:32 * group + 32]
            assert half.isnan().all() and not got[r, 32 - 32 * group:64 - 32 * group].isnan().any()
        assert (got[0] == 1.5).all() and not got[1].any()
        assert not unpack(cache.k[0].cpu()[0, 0, :1], bits).any()


def test_one_output_only(ctx):
    cache = filled_cache(1, 2, 40, 128, 4, 64, torch.bfloat16)
    gen = torch.Generator().manual_seed(5)
    k, v = (rows_of(gen, 1, 40, 256, torch.bfloat16) for _ in range(2))
    announce("read one of k and v")
    ctx.cache_append(cache, k.cuda(), v.cuda())
    both = ctx.cache_read(cache, 40)
    only = torch.zeros_like(both[1])
    assert ctx.lib.dfq_cache_read(ctx.handle, cache.desc, None, only.data_ptr(), 0, 1, 40, 0, None,
                                  dflash_qmm._stream(None)) == 0
    torch.cuda.synchronize()
    assert torch.equal(only, both[1])


def test_offsets_past_32_bits(ctx):
    """The last slot of a cache whose code arrays are over 4 GiB each."""
    heads, dim, cap, slots = 8, 256, 60000, 36
    cache = dflash_qmm.KVCache.from_arrays(
        *[(torch.empty(slots, heads, cap, 64, dtype=torch.int32, device="cuda"),
           torch.empty(slots, heads, cap, 8, dtype=torch.bfloat16, device="cuda"),
           torch.empty(slots, heads, cap, 8, dtype=torch.bfloat16, device="cuda"))
          for _ in range(2)], 8, 32)
    assert cache.k[0].numel() * 4 > 1 << 32
    gen = torch.Generator().manual_seed(9)
    k, v = (rows_of(gen, slots, 2, heads * dim, torch.bfloat16) for _ in range(2))
    announce("append past 4 GiB")
    ctx.cache_append(cache, k.cuda(), v.cuda(), start=cap - 2)
    got = ctx.cache_read(cache, 2, start=cap - 2, batch=slots, dtype=torch.float32)
    torch.cuda.synchronize()
    for x, y in zip((k, v), got):
        c, s, b = quantise(x.view(slots, 2, heads, dim), 8, 32)
        want = c.float().unflatten(-1, (-1, 32)) * s.float()[..., None] + b.float()[..., None]
        assert torch.equal(y.cpu(), want.flatten(-2))


def test_refusals(ctx):
    """Every argument the calls refuse, with nothing launched."""
    good = dflash_qmm.KVCache(2, 2, 16, 64, 4, 32, torch.bfloat16)
    x = torch.zeros(2, 3, 128, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, device="cuda")

    def append(cache=good, kk=x.data_ptr(), stride=128, batch=2, rows=3, handle=ctx.handle):
        return ctx.lib.dfq_cache_append(handle, cache.desc if cache else None, kk, x.data_ptr(),
                                        stride, batch, rows, 0, None, None)

    def read(cache=good, kk=k.data_ptr(), vv=k.data_ptr(), dt=0, batch=2, rows=3):
        return ctx.lib.dfq_cache_read(ctx.handle, cache.desc, kk, vv, dt, batch, rows, 0, None,
                                      None)

    assert append(handle=None) == 1 and append(cache=None) == 1
    assert append(kk=None) == 1 and append(kk=x.data_ptr() + 1) == 1
    assert append(stride=127) == 1 and append(batch=0) == 1 and append(rows=0) == 1
    assert append(batch=3) == 1                      # more sequences than slots
    assert read(kk=None, vv=None) == 1 and read(kk=k.data_ptr() + 8) == 1
    assert read(dt=1) == 2 and read(batch=3) == 1 and read(rows=-1) == 1
    for field, value, status in (("bits", 3, 2), ("head_dim", 96, 2), ("group_size", 48, 2),
                                 ("group_size", 128, 2), ("dtype", 2, 2), ("capacity", 0, 1),
                                 ("heads", 0, 1), ("k_codes", None, 1), ("v_scales", None, 1),
                                 ("k_codes", good.k[0].data_ptr() + 4, 1),
                                 ("v_biases", good.v[2].data_ptr() + 1, 1),
                                 ("capacity", 1 << 30, 2), ("slots", 1 << 20, 2)):
        bad = dflash_qmm.KVCache.from_arrays(good.k, good.v, 4, 32)
        setattr(bad._desc, field, value)
        assert append(cache=bad) == status and read(cache=bad) == status, (field, value)
    assert b"slots" in ctx.lib.dfq_last_error()
    with pytest.raises(ValueError):
        ctx.cache_append(good, x.float(), x.float())
    with pytest.raises(ValueError):
        ctx.cache_append(good, x[:, :, :64], x[:, :, :64])
    with pytest.raises(ValueError):
        ctx.cache_append(good, x, x, starts=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        ctx.cache_append(good, x[:, :, ::2].repeat(1, 1, 2).transpose(1, 2).transpose(1, 2),
                         x.transpose(0, 1).contiguous().transpose(0, 1))
