"""64-bit plain forms of the rotary positions, the head norms and the sampled accept."""
import math

import numpy as np
import torch

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half_step(dtype):
    """A rounding's largest error relative to the value, and the largest among denormals."""
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def rotated(x, positions, frequencies, amplitude=1.0, interleaved=False, inverse=False, weight=None,
            offset=0.0, eps=None):
    """(values, sizes) in float64 of x [batch, rows, heads, dim] on the CPU: heads normed where eps
    is given, then turned to positions [batch, rows].  Sizes are |a| + |b| of each value's pair
    times the amplitude, that errors are counted in."""
    x = x.double()
    if eps is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        if weight is not None:
            x = x * (weight.double() + offset)
    n = len(frequencies)
    # whole arithmetic keeps far positions: the angle's place in its turn, to 2^-60 or so
    turn = [[[float(angle(int(p), f)) for f in frequencies] for p in row]
            for row in positions.tolist()]
    t = torch.tensor(turn, dtype=torch.float64).view(*positions.shape, 1, n)
    cos, sin = t.cos() * amplitude, t.sin() * amplitude
    if inverse:
        sin = -sin
    first = torch.arange(n) * 2 if interleaved else torch.arange(n)
    second = first + (1 if interleaved else n)
    y, size = x.clone(), x.abs()
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(amplitude)
    return y, size


def angle(position, frequency):
    """position * frequency within a turn, by exact fractions of a 200-bit 2 pi."""
    from fractions import Fraction
    # 2 pi to 64 decimal places
    turn = Fraction(62831853071795864769252867665590057683943387987502116419498891846,
                    10 ** 64)
    whole = position * Fraction(frequency) / turn
    return float((whole - math.floor(whole)) * turn)


def check_rotated(got, want, size, dtype, normed):
    """Each value within its rounding and the fp32 arithmetic's bound.

    Sine and cosine: the angle within an eighth of a turn (0.79) is rounded as a whole number, its
    factor and their product, 0.79 * 2^-23, and is 2^-32 turns short (1.5e-9); the sums' last terms
    round 3 times by 2^-24; amplitude, product and sum by 2^-24 each: under 2^-21 of |a| + |b|.
    The norm: up to 22 sums of squares, halved by the root, the root itself (2^-23), three
    products and the weight's sum: under 2^-20."""
    relative, least = half_step(dtype)
    bound = size * (2.0 ** -21 + (2.0 ** -20 if normed else 0.0))
    bound = bound + (want.abs() + bound) * relative + least + 2.0 ** -149
    off = (got.double().cpu() - want).abs()
    same = (got.double().cpu() == want) | (torch.isnan(want) & torch.isnan(got.double().cpu()))
    bad = ~((off <= bound) | same)
    assert not bad.any(), (int(bad.sum()), off[bad].max(), bound[bad][off[bad].argmax()])


def distribution(x, t):
    """Probabilities of a row of logits (float64 array) at temperature t, or None."""
    if not (0 <= t < math.inf):
        return None
    if t == 0:
        if np.isnan(x).all():
            return None
        p = np.zeros_like(x)
        p[np.nanargmax(x)] = 1.0
        return p
    top = x.max()
    if np.isnan(x).any() or not np.isfinite(top):
        return None
    with np.errstate(over="ignore", under="ignore"):
        e = np.exp((x - top) / t)
    return e / e.sum()


def accept(logits, uniforms, drafts, lengths, draft_logits, temperature, draft_temperature):
    """(tokens, accepted, chances, margin) by the definition, one sequence after the other; margin
    is how near the nearest decision lies to its border: of u q to p, relative to p, and of the
    running sums to u times the whole, relative to the whole."""
    b, m, v = logits.shape
    tokens = np.full((b, m), -1, dtype=np.int32)
    accepted = np.zeros(b, dtype=np.int32)
    chances = np.zeros((b, m - 1))
    margin = math.inf
    for i in range(b):
        t, td = float(temperature[i]), float(draft_temperature[i])
        n = m - 1 if lengths is None else min(max(int(lengths[i]), 0), m - 1)
        left, done = None, False
        for j in range(n + 1):
            p = distribution(logits[i, j], t)
            if j == n:
                if not done:
                    left, accepted[i], done = p, j, True
                break
            d = int(drafts[i, j])
            known = 0 <= d < v
            q = None
            if draft_logits is not None and td != 0:
                q = distribution(draft_logits[i, j], td)
            else:
                q = np.zeros(v)
                if known:
                    q[d] = 1.0
            ok = False
            if p is not None and q is not None and known:
                u = float(uniforms[i, j])
                chances[i, j] = min(1.0, p[d] / q[d]) if q[d] > 0 else float(p[d] > 0)
                ok = u * q[d] < p[d]
                if p[d] > 0 and t > 0:
                    margin = min(margin, abs(u * q[d] - p[d]) / p[d])
            if done:
                continue
            if ok:
                tokens[i, j] = d
                continue
            accepted[i], done = j, True
            if p is None or q is None:
                left = None
                continue
            left = np.maximum(p - q, 0.0)
            if not left.sum() > 0:
                left = p if draft_logits is not None and td != 0 else q
        if left is None:
            continue
        u = float(uniforms[i, m - 1])
        run = np.cumsum(left)
        at = int(np.searchsorted(run, u * run[-1], side="right"))
        if at >= v:
            at = int(np.nonzero(left)[0][-1])
        tokens[i, accepted[i]] = at
        if t > 0 and left[left > 0].size > 1:
            margin = min(margin, np.abs(run[left > 0][:-1] / run[-1] - u).min())
    return tokens, accepted, chances, margin
