"""64-bit plain forms of the cache, attention and log-probability operators, and random caches."""
import math

import torch

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
FORMATS = [(d, b, g, t) for d in (64, 128, 256) for b in (4, 8) for g in (32, 64, 128) if g <= d
           for t in ("bf16", "f16")]


def quantise(x, bits, gs):
    """(codes [.., dim] int64, scales, biases [.., groups]) of rows x in their 16-bit dtype, by
    the format's definition: fp32 arithmetic, scale and bias rounded to the dtype."""
    f = x.float().unflatten(-1, (-1, gs))
    top = float((1 << bits) - 1)
    low, high = f.amin(-1), f.amax(-1)
    scale, bias = ((high - low) / top).to(x.dtype), low.to(x.dtype)
    bad = ~(torch.isfinite(scale) & torch.isfinite(bias) & torch.isfinite(f).all(-1))
    s, b = scale.float(), bias.float()
    s = torch.where(bad, torch.zeros_like(s), s)[..., None]
    codes = torch.where(s > 0, ((f - b[..., None]) / s).round().clamp(0, top),
                        torch.zeros_like(f))
    codes = torch.where(bad[..., None], torch.zeros_like(f), codes)
    nan = torch.tensor(math.nan, dtype=x.dtype)
    return (codes.flatten(-2).long(), torch.where(bad, nan, scale), torch.where(bad, nan, bias))


def pack(codes, bits):
    per = 32 // bits
    c = codes.unflatten(-1, (-1, per)) << (torch.arange(per) * bits)
    w = c.sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def unpack(words, bits):
    per = 32 // bits
    w = words.long() & 0xffffffff
    return ((w[..., None] >> (torch.arange(per) * bits)) & ((1 << bits) - 1)).flatten(-2)


def values(arrays, bits, gs):
    """The values (float64) that a cache's CPU arrays stand for."""
    codes = unpack(arrays[0], bits).double().unflatten(-1, (-1, gs))
    return (codes * arrays[1].double()[..., None] + arrays[2].double()[..., None]).flatten(-2)


def random_arrays(gen, slots, heads, capacity, dim, bits, gs, dtype, spread=1.0):
    """CPU (codes, scales, biases) of random rows; the codes, scales and biases themselves are
    random too, with scales of either sign as a cache written elsewhere may have them."""
    lead = (slots, heads, capacity)
    codes = torch.randint(0, 1 << bits, lead + (dim,), generator=gen)
    scales = torch.randn(lead + (dim // gs,), generator=gen) * spread / (1 << bits)
    biases = torch.randn(lead + (dim // gs,), generator=gen) * spread / 2
    return pack(codes, bits), scales.to(dtype), biases.to(dtype)


def attention(q, prefix, prefix_length, own, lengths, tree, scale, bits, gs, heads):
    """(y, lse, worst) in float64 for q [batch, rows, q_heads, dim]; prefix and own are pairs of
    CPU arrays (K, V) or None.  worst [batch, rows, q_heads, 2]: the largest |v| that a row sees
    and the largest sum of |q| |s c| + |q| |b| over its tokens."""
    batch, rows, q_heads, dim = q.shape
    y = torch.zeros(batch, rows, q_heads, dim, dtype=torch.float64)
    lse = torch.full((batch, rows, q_heads), -math.inf, dtype=torch.float64)
    worst = torch.zeros(batch, rows, q_heads, 2, dtype=torch.float64)

    def parts(arrays, slot, head, n):
        a = [x[slot, head, :n] for x in arrays]
        size = (unpack(a[0], bits).double().unflatten(-1, (-1, gs)) * a[1].double().abs()[..., None]
                + a[2].double().abs()[..., None]).flatten(-2)
        return values(a, bits, gs), size

    for b in range(batch):
        n = max(0, int(lengths[b])) if own is not None else 0
        for h in range(heads):
            ks, vs, sizes, pos = [], [], [], []
            if prefix is not None and prefix_length:
                k, size = parts(prefix[0], 0, h, prefix_length)
                ks.append(k), sizes.append(size)
                vs.append(parts(prefix[1], 0, h, prefix_length)[0])
                pos += [None] * prefix_length
            if n:
                k, size = parts(own[0], b, h, n)
                ks.append(k), sizes.append(size)
                vs.append(parts(own[1], b, h, n)[0])
                pos += list(range(n))
            if not pos:
                continue
            k, v, size = torch.cat(ks), torch.cat(vs), torch.cat(sizes)
            for m in range(rows):
                bits_m = int(tree[b, m]) if tree is not None else (2 << m) - 1
                see = [p is None or p < n - rows or (bits_m >> (p - (n - rows))) & 1 == 1
                       for p in pos]
                see = torch.tensor(see)
                if not see.any():
                    continue
                for j in range(h * (q_heads // heads), (h + 1) * (q_heads // heads)):
                    z = (k[see] @ q[b, m, j].double()) * scale
                    lse[b, m, j] = torch.logsumexp(z, 0)
                    y[b, m, j] = torch.softmax(z, 0) @ v[see]
                    worst[b, m, j, 0] = v[see].abs().max()
                    worst[b, m, j, 1] = (size[see] @ q[b, m, j].double().abs()).max()
    return y, lse, worst


def logprobs(x, tokens, k):
    """(logprobs, entropy, top tokens, top logprobs) of logits x in float64."""
    x = x.double()
    z = torch.log_softmax(x, -1)
    p = z.exp()
    entropy = -torch.where(p > 0, p * z, torch.where(z.isnan(), z, torch.zeros_like(z))).sum(-1)
    m, v = x.shape
    lp = torch.full((m,), math.nan, dtype=torch.float64)
    for i, t in enumerate(tokens.tolist()):
        if 0 <= t < v:
            lp[i] = z[i, t]
    ids = torch.full((m, k), -1, dtype=torch.int64)
    top = torch.full((m, k), math.nan, dtype=torch.float64)
    for i in range(m):
        real = [j for j in range(v) if not math.isnan(x[i, j])]
        best = sorted(real, key=lambda j: (-float(x[i, j]), j))[:k]
        for n, j in enumerate(best):
            ids[i, n], top[i, n] = j, z[i, j]
    return lp, entropy, ids, top
