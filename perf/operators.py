"""A verify pass's attention over a quantised key/value cache, and the scoring of its logits.

Four operators stand next to the quantised projections in a speculative decoder's verify pass:

* append: the block's new K and V rows are quantised as they are written to the cache (affine
  codes of 4 or 8 bits, one scale and bias per group of a head's channels);
* read: a span of the cache back as the values it stands for;
* attention: the block's queries against a prefix that all sequences share (held once) and each
  sequence's own cache, with the draft chain's or the draft tree's mask inside the block;
* logprobs: log probabilities of given tokens, the entropy and the top alternatives of each row
  of logits.

Shapes are those of the benchmark's model (5120 wide: 40 query heads over 8 K/V heads of 128, a
fused q|k|v row of 7168, a vocabulary of 151936) and generic ones with heads of 64 and 256.

Interface: own, listed(), draw(rng), prepare(case, seed), run(state), work(case),
exact(case, seed).
"""
import math
import os
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}

MOST_ROWS = 8192 * 8 * 128            # channels of the largest listed append
MOST_READ = 32768 * 8 * 128           # and of the largest listed read
MOST_SCORES = 16 * 8 * 40 * 16900 * 128   # query-key products of the largest listed attention
MOST_LOGITS = 2048 * 151936


def _cache_case(name, kind, **kw):
    c = {"kind": kind, "slots": 1, "rows": 1, "heads": 8, "dim": 128, "bits": 4, "gs": 64,
         "dtype": "bf16"}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def _logit_case(name, **kw):
    c = {"kind": "logprobs", "rows": 1, "vocab": 151936, "top": 1, "dtype": "bf16"}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the smallest append: one token of each of 8 sequences, 8-bit, and its values back
        _cache_case("append_step_8bit", "append", slots=8, rows=1, bits=8, start=1023,
                    capacity=2048),
        # a prompt of 8192 tokens into a 4-bit cache, the rows cut from the fused q|k|v output
        _cache_case("append_prompt", "append", rows=8192, start=37, capacity=8300),
        # ragged chunks of five prompts with wide heads, fp16, groups of 32
        _cache_case("append_ragged_f16", "append", slots=5, rows=333, heads=2, dim=256, bits=8,
                    gs=32, dtype="f16", start=101, capacity=1000),
        # a whole 32768-token cache back as bf16 values
        _cache_case("read_long", "read", rows=32768, start=0, capacity=32770),
        # odd spans of four caches with narrow heads back as fp16
        _cache_case("read_ragged_f16", "read", slots=4, rows=1537, dim=64, bits=8, gs=32,
                    dtype="f16", start=13, capacity=2000),
        # one decoded token of one sequence over a middling cache: latency
        _cache_case("attn_decode", "attention", rows=1, q_heads=40, prefix=0, length=4097),
        # a verify block of 8 rows over a long cache: the cache's bytes count
        _cache_case("attn_verify_long", "attention", rows=8, q_heads=40, prefix=0,
                    length=32776),
        # 16 sequences that share a 16384-token prompt verify a block of 8 each: the prefix is
        # one product for all 128 rows
        _cache_case("attn_shared_prefix", "attention", slots=16, rows=8, q_heads=40,
                    prefix=16384, length=512),
        # a draft tree of 7 rows for five sequences, wide heads, 8-bit fp16, odd sizes
        _cache_case("attn_tree_f16", "attention", slots=5, rows=7, q_heads=16, heads=2, dim=256,
                    bits=8, gs=32, dtype="f16", prefix=2049, length=301, tree=True),
        # the logits of a verify block of 8 with five alternatives each
        _logit_case("logprobs_verify", rows=8, top=5),
        # scoring a 2048-token prompt with 20 alternatives a token
        _logit_case("logprobs_prompt", rows=2048, top=20),
        # fp32 logits of an odd vocabulary, the best token only
        _logit_case("logprobs_f32", rows=33, vocab=32003, top=1, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "attention", "attention", "attention",
                       "attention", "logprobs", "logprobs"])
    if kind == "logprobs":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        vocab = _log(rng, 1000, 151936)
        rows = min(_log(rng, 1, 2048), MOST_LOGITS // (vocab * SIZE[dtype] // 2))
        return _logit_case(None, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]),
                           dtype=dtype)
    dim = rng.choice([64, 128, 128, 256])
    c = {"dim": dim, "bits": rng.choice([4, 4, 8]),
         "gs": rng.choice([g for g in (32, 64, 64, 128) if g <= dim]),
         "dtype": rng.choice(["bf16", "bf16", "f16"]), "heads": rng.choice([1, 2, 4, 8])}
    slots = _log(rng, 1, 16)
    if kind == "attention":
        c["q_heads"] = c["heads"] * rng.choice([1, 2, 3, 4, 5, 8])
        rows = rng.randint(1, 16)
        each = slots * rows * c["q_heads"] * dim
        most = max(2 * rows, MOST_SCORES // each)
        prefix = rng.choice([0, _log(rng, 1, 32768)])
        length = _log(rng, rows, 2048 if prefix else 32768)
        prefix = min(prefix, most // 2)
        length = max(rows, min(length, most // 2))
        return _cache_case(None, kind, slots=slots, rows=rows, prefix=prefix, length=length,
                           tree=rng.random() < 0.4, **c)
    most = (MOST_ROWS if kind == "append" else MOST_READ) // (slots * c["heads"] * dim)
    rows = max(1, min(_log(rng, 1, 32768), most))
    start = rng.choice([0, _log(rng, 1, 999)])
    return _cache_case(None, kind, slots=slots, rows=rows, start=start,
                       capacity=start + rows + rng.randint(2, 200), **c)


# ---- inputs -------------------------------------------------------------------------------

def _rows(gen, slots, rows, heads, dim, dtype, spread):
    """K or V rows: normal, with a mean of its own for each channel as K caches have them."""
    x = torch.randn(slots, rows, heads, dim, device="cuda", generator=gen)
    x += spread * torch.randn(heads, dim, device="cuda", generator=gen)
    return x.to(DT[dtype])


def _quantise(x, bits, gs):
    """Codes (fp32 whole numbers) [.., groups, gs], scales and biases [.., groups] of rows x."""
    top = float((1 << bits) - 1)
    f = x.float().unflatten(-1, (-1, gs))
    low, high = f.amin(-1), f.amax(-1)
    scale = ((high - low) / top).to(x.dtype)
    bias = low.to(x.dtype)
    s, b = scale.float()[..., None], bias.float()[..., None]
    codes = torch.where(s > 0, torch.round((f - b) / s).clamp(0, top), torch.zeros_like(f))
    return codes, scale, bias


def _pack(codes, bits):
    """Words of a row's codes, element 0 in the low bits."""
    per = 32 // bits
    c = codes.flatten(-2).to(torch.int64).unflatten(-1, (-1, per))
    at = torch.arange(per, device=c.device) * bits
    return (c << at).sum(-1).to(torch.int32)


def _cache_arrays(x, capacity, bits, gs):
    """The three arrays [slots][heads][capacity][..] of a cache holding rows x [slots][T][..]."""
    slots, _, heads, dim = x.shape
    codes, scale, bias = _quantise(x.transpose(1, 2), bits, gs)
    out = []
    for a in (_pack(codes, bits), scale, bias):
        t = torch.zeros(slots, heads, capacity, a.shape[-1], dtype=a.dtype, device="cuda")
        t[:, :, :a.shape[2]] = a
        out.append(t)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s = dict(case)
    dt = DT[case["dtype"]]
    if case["kind"] == "logprobs":
        m, v = case["rows"], case["vocab"]
        x = torch.empty(m, v, dtype=dt, device="cuda")
        for r in range(0, m, 256):
            n = min(256, m - r)
            x[r:r + n] = 2.5 * torch.randn(n, v, device="cuda", generator=gen)
        # some rows are nearly decided, as verify rows are
        boost = torch.randint(0, v, (m,), device="cuda", generator=gen)
        x[torch.arange(m, device="cuda"), boost] += 12 * torch.rand(
            m, device="cuda", generator=gen).to(dt)
        other = torch.randint(0, v, (m,), device="cuda", generator=gen)
        s["logits"] = x
        s["tokens"] = torch.where(other % 2 == 0, boost, other).to(torch.int32)
        return s
    b, m, h, d = case["slots"], case["rows"], case["heads"], case["dim"]
    if case["kind"] == "append":
        cap = case["capacity"]
        # the rows are cut from one fused output with the queries of a 5120-wide model in front
        fused = torch.zeros(b, m, (40 + 2 * h) * d, dtype=dt, device="cuda")
        k, v = fused[:, :, -2 * h * d:-h * d], fused[:, :, -h * d:]
        k.copy_(_rows(gen, b, m, h, d, case["dtype"], 1.0).flatten(2))
        v.copy_(_rows(gen, b, m, h, d, case["dtype"], 0.1).flatten(2))
        s["k"], s["v"] = k, v
        empty = torch.zeros(b, 0, h, d, dtype=dt, device="cuda")
        s["cache_k"] = _cache_arrays(empty, cap, case["bits"], case["gs"])
        s["cache_v"] = _cache_arrays(empty, cap, case["bits"], case["gs"])
        s["starts"] = _starts(case, gen)
        return s
    if case["kind"] == "read":
        cap = case["capacity"]
        for name, spread in (("cache_k", 1.0), ("cache_v", 0.1)):
            s[name] = _cache_arrays(_rows(gen, b, cap, h, d, case["dtype"], spread), cap,
                                    case["bits"], case["gs"])
        s["starts"] = _starts(case, gen)
        return s
    p, n = case["prefix"], case["length"]
    for name, slots, tokens in (("prefix", 1, p), ("cache", b, n)):
        if not tokens:
            continue
        for part, spread in (("_k", 1.0), ("_v", 0.1)):
            x = _rows(gen, slots, tokens, h, d, case["dtype"], spread)
            s[name + part] = _cache_arrays(x, tokens, case["bits"], case["gs"])
    q = 1.5 * torch.randn(b, m, case["q_heads"] * d, device="cuda", generator=gen)
    s["q"] = q.to(dt)
    # ragged sequences: from half the longest up, at least the block itself
    low = max(m, n // 2)
    lengths = torch.randint(low, n + 1, (b,), device="cuda", generator=gen)
    lengths[0] = n
    s["lengths"] = lengths.to(torch.int32)
    s["tree"] = None
    if case.get("tree"):
        # row j hangs on an earlier row: it sees that row's path and itself
        bits = torch.zeros(b, m, dtype=torch.int64)
        parent = torch.randint(0, 1 << 20, (b, m), device="cuda", generator=gen).cpu()
        for i in range(b):
            for j in range(m):
                up = int(bits[i, int(parent[i, j]) % j]) if j else 0
                bits[i, j] = up | (1 << j)
        s["tree"] = bits.to(torch.int32).cuda()
    return s


def _starts(case, gen):
    """Where each sequence's span starts: case["start"], one or two tokens later for some."""
    late = torch.randint(0, 3, (case["slots"],), device="cuda", generator=gen)
    return (case["start"] + late).to(torch.int32)


# ---- the plain forms ------------------------------------------------------------------------

def _values(arrays, bits, gs):
    """scale * code + bias of a cache's arrays [.., words], in fp32 [.., dim]."""
    words, scale, bias = arrays
    at = torch.arange(32 // bits, device=words.device, dtype=torch.int32) * bits
    codes = (words[..., None] >> at) & ((1 << bits) - 1)
    f = codes.flatten(-2).float().unflatten(-1, (-1, gs))
    return (f * scale.float()[..., None] + bias.float()[..., None]).flatten(-2)


def _span(s):
    """Index of each sequence's span: (slots, 1, 1), (1, heads, 1), (slots, 1, rows)."""
    dev = s["starts"].device
    slot = torch.arange(s["slots"], device=dev)[:, None, None]
    head = torch.arange(s["heads"], device=dev)[None, :, None]
    pos = s["starts"].long()[:, None, None] + torch.arange(s["rows"], device=dev)[None, None, :]
    return slot, head, pos


def _plain_read(s, arrays, at):
    f = _values([a[at] for a in arrays], s["bits"], s["gs"])
    return f.transpose(1, 2).to(arrays[1].dtype).contiguous()


def _plain_append(s):
    at = _span(s)
    out = {}
    for name in ("k", "v"):
        x = s[name].unflatten(-1, (s["heads"], s["dim"])).transpose(1, 2)
        codes, scale, bias = _quantise(x, s["bits"], s["gs"])
        arrays = s["cache_" + name]
        arrays[0][at] = _pack(codes, s["bits"])
        arrays[1][at] = scale
        arrays[2][at] = bias
        out[name] = _plain_read(s, arrays, at)
    return out


def _plain_attention(s):
    b, m, h, d = s["slots"], s["rows"], s["heads"], s["dim"]
    g, n = s["q_heads"] // h, s["length"]
    q = s["q"].float().view(b, m, h, g, d) / math.sqrt(d)
    own_k = _values(s["cache_k"], s["bits"], s["gs"])
    own_v = _values(s["cache_v"], s["bits"], s["gs"])
    each = q.permute(0, 2, 1, 3, 4).reshape(b * h, m * g, d)
    scores = torch.bmm(each, own_k.view(b * h, n, d).transpose(1, 2).contiguous())
    scores = scores.view(b, h, m, g, n)
    # row j of the block sits at lengths - rows + j
    first = (s["lengths"].long() - m)[:, None, None]
    pos = torch.arange(n, device=q.device)[None, None, :]
    row = torch.arange(m, device=q.device)[None, :, None]
    if s["tree"] is None:
        seen = pos <= first + row
    else:
        inside = (pos - first).clamp(0, m - 1)
        seen = (s["tree"].long()[:, :, None] >> inside) & 1 == 1
        seen = (pos < first) | ((pos < first + m) & seen)
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    if s["prefix"]:
        k = _values(s["prefix_k"], s["bits"], s["gs"])[0]
        v = _values(s["prefix_v"], s["bits"], s["gs"])[0]
        rows = q.permute(2, 0, 1, 3, 4).reshape(h, b * m * g, d)
        shared = torch.bmm(rows, k.transpose(1, 2).contiguous())
        shared = shared.view(h, b, m, g, -1).transpose(0, 1)
        scores = torch.cat((shared, scores), -1)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    e = e / total
    mine = e[..., s["prefix"]:].reshape(b * h, m * g, n)
    y = torch.bmm(mine, own_v.view(b * h, n, d)).view(b, h, m, g, d)
    if s["prefix"]:
        part = e[..., :s["prefix"]].transpose(0, 1).reshape(h, b * m * g, -1)
        y = y + torch.bmm(part, v).view(h, b, m, g, d).transpose(0, 1)
    y = y.permute(0, 2, 1, 3, 4).reshape(b, m, h * g * d).to(s["q"].dtype)
    lse = (top + torch.log(total))[..., 0].permute(0, 2, 1, 3).reshape(b, m, h * g)
    return {"y": y, "lse": lse}


def _plain_logprobs(s):
    x = s["logits"].float()
    m, v = x.shape
    top = x.amax(-1, keepdim=True)
    shifted = x - top
    e = torch.exp(shifted)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    given = torch.gather(shifted, 1, s["tokens"].long()[:, None])
    entropy = log_total - (e * shifted).sum(-1, keepdim=True) / total
    out = {"logprobs": (given - log_total)[:, 0], "entropy": entropy[:, 0]}
    if s["top"]:
        # order by value, ties to the lowest index: one whole number for the two
        i = x.view(torch.int32).long()
        i = torch.where(i < 0, -(i & 0x7fffffff), i)
        best = torch.topk(i * v + (v - 1 - torch.arange(v, device=x.device)), s["top"], -1)
        ids = v - 1 - torch.remainder(best.values, v)
        out["top_tokens"] = ids.to(torch.int32)
        out["top_logprobs"] = torch.gather(shifted, 1, ids) - log_total
    return out


# ---- the framework's operators --------------------------------------------------------------

_ctx = None


def _context():
    """A program keeps one context per GPU."""
    global _ctx
    if _ctx is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "dflash-swift_amd"))
        import dflash_qmm
        _ctx = dflash_qmm.Context(0)
    return _ctx


def _handle(s, name):
    """The cache object that a program keeps over its arrays."""
    key = name + "_handle"
    if key not in s:
        import dflash_qmm
        s[key] = dflash_qmm.KVCache.from_arrays(s[name + "_k"], s[name + "_v"], s["bits"],
                                                s["gs"])
    return s[key]


def _own(s):
    ctx = _context()
    if s["kind"] == "logprobs":
        lp, entropy, ids, top = ctx.token_logprobs(s["logits"], s["tokens"], top_k=s["top"])
        out = {"logprobs": lp, "entropy": entropy}
        if s["top"]:
            out["top_tokens"], out["top_logprobs"] = ids, top
        return out
    cache = _handle(s, "cache")
    if s["kind"] == "attention":
        prefix = _handle(s, "prefix") if s["prefix"] else None
        y, lse = ctx.cache_attention(s["q"], cache, lengths=s["lengths"],
                                     max_length=s["length"], prefix=prefix,
                                     prefix_length=s["prefix"], tree=s["tree"])
        return {"y": y, "lse": lse}
    if s["kind"] == "append":
        ctx.cache_append(cache, s["k"], s["v"], starts=s["starts"])
    k, v = ctx.cache_read(cache, s["rows"], starts=s["starts"])
    return {"k": k, "v": v}


def run(s):
    if own:
        return _own(s)
    if s["kind"] == "logprobs":
        return _plain_logprobs(s)
    if s["kind"] == "attention":
        return _plain_attention(s)
    if s["kind"] == "append":
        return _plain_append(s)
    at = _span(s)
    return {"k": _plain_read(s, s["cache_k"], at), "v": _plain_read(s, s["cache_v"], at)}


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        # a subtraction, an exponential, a comparison, two sums and a product a logit
        return {"bytes": n * SIZE[case["dtype"]] + case["rows"] * (12 + 8 * case["top"]),
                "flops": 6 * n}
    d = case["dim"]
    row = d * case["bits"] // 8 + 4 * d // case["gs"]   # one cached row of one head
    values = 2 * case["slots"] * case["rows"] * case["heads"]
    if case["kind"] == "read":
        return {"bytes": values * (row + 2 * d), "flops": 2 * values * d}
    if case["kind"] == "append":
        # the rows in, the cache's bytes out, the values back out
        return {"bytes": values * (2 * d + row + 2 * d), "flops": 8 * values * d}
    p, n, b = case["prefix"], case["length"], case["slots"]
    q = b * case["rows"] * case["q_heads"]
    tokens = p + b * (3 * n / 4 if b > 1 else n)   # ragged: three quarters of n on average
    return {"bytes": 2 * tokens * case["heads"] * row + q * (4 * d + 4),
            "flops": 4 * d * q * (p + tokens / b - p / b)}


# ---- the definition in 64 bits --------------------------------------------------------------

def _wide(arrays, bits, gs):
    """A cache's values in 64 bits, its codes taken byte by byte."""
    raw = arrays[0].contiguous().view(torch.uint8)
    if bits == 4:
        raw = torch.stack((raw % 16, torch.div(raw, 16, rounding_mode="floor")), -1).flatten(-2)
    spread = [a.double().repeat_interleave(gs, -1) for a in arrays[1:]]
    return torch.addcmul(spread[1], spread[0], raw.double())


def _exact_rows(x, bits, gs):
    """What rows x read back as, by the format's definition."""
    w = x.double().reshape(*x.shape[:-1], x.shape[-1] // gs, gs)
    b = w.min(-1, keepdim=True).values
    step = (w.max(-1, keepdim=True).values - b) / (2 ** bits - 1)
    step = step.to(x.dtype).double()
    steps = torch.div(w - b, torch.where(step == 0, torch.ones_like(step), step))
    steps = torch.where(step == 0, torch.zeros_like(w), steps.round().clip(0, 2 ** bits - 1))
    return (steps * step + b).reshape(x.shape)


def _exact_attention(s):
    b, m, h, d, n, p = (s[k] for k in ("slots", "rows", "heads", "dim", "length", "prefix"))
    g = s["q_heads"] // h
    y = torch.zeros(b, m, h, g, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(b, m, h, g, dtype=torch.float64, device="cuda")
    q = s["q"].double().reshape(b, m, h, g, d)
    tree = None if s["tree"] is None else s["tree"].tolist()
    lengths = s["lengths"].tolist()
    for i in range(h):
        k0 = v0 = torch.zeros(0, d, dtype=torch.float64, device="cuda")
        if p:
            k0 = _wide([a[0, i] for a in s["prefix_k"]], s["bits"], s["gs"])
            v0 = _wide([a[0, i] for a in s["prefix_v"]], s["bits"], s["gs"])
        for j in range(b):
            size = lengths[j]
            k1 = _wide([a[j, i, :size] for a in s["cache_k"]], s["bits"], s["gs"])
            v1 = _wide([a[j, i, :size] for a in s["cache_v"]], s["bits"], s["gs"])
            hidden = torch.zeros(m, size, dtype=torch.bool)
            for r in range(m):
                for t in range(m):
                    sees = t <= r if tree is None else tree[j][r] >> t & 1
                    hidden[r, size - m + t] = not sees
            z0 = q[j, :, i] @ k0.T if p else torch.zeros(m, g, 0, dtype=torch.float64,
                                                         device="cuda")
            z1 = (q[j, :, i] @ k1.T).masked_fill(hidden.cuda()[:, None, :], -math.inf)
            z = torch.cat((z0, z1), -1) * d ** -0.5
            lse[j, :, i] = torch.logsumexp(z, -1)
            w = torch.exp(z - lse[j, :, i][..., None])
            y[j, :, i] = w[..., :p] @ v0 + w[..., p:] @ v1
    return {"y": y.reshape(b, m, h * g * d), "lse": lse.reshape(b, m, h * g)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        shape = (s["slots"], s["rows"], s["heads"], s["dim"])
        return {n: _exact_rows(s[n].reshape(shape), s["bits"], s["gs"]) for n in ("k", "v")}
    if case["kind"] == "read":
        out = {}
        for n in ("k", "v"):
            spans = [[a[i, :, t:t + s["rows"]] for a in s["cache_" + n]]
                     for i, t in enumerate(s["starts"].tolist())]
            out[n] = torch.stack([_wide(a, s["bits"], s["gs"]).transpose(0, 1) for a in spans])
        return out
    if case["kind"] == "attention":
        return _exact_attention(s)
    rows = {"logprobs": [], "entropy": [], "top_tokens": [], "top_logprobs": []}
    for r in range(0, s["rows"], 128):
        z = torch.log_softmax(s["logits"][r:r + 128].double(), -1)
        rows["logprobs"].append(z.gather(1, s["tokens"][r:r + 128].long()[:, None])[:, 0])
        rows["entropy"].append(-(z.exp() * z).sum(-1))
        if s["top"]:
            best = torch.sort(s["logits"][r:r + 128].double(), dim=-1, descending=True,
                              stable=True)
            ids = best.indices[:, :s["top"]]
            rows["top_tokens"].append(ids.to(torch.int32))
            rows["top_logprobs"].append(z.gather(1, ids))
    return {n: torch.cat(v) for n, v in rows.items() if v}
