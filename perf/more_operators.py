"""What stands between a verify pass's projections and its attention, and behind its LM head.

Three operators of a speculative decoder's verify pass:

* rope: rotary positions of the block's queries and keys, cut from the fused q|k|v rows;
* norm_rope: the RMS norm of each head of queries and keys with the rotation in the same pass;
* accept: drafted tokens verified against the target's probabilities from given random numbers
  (with the chance that each draft had), and the token drawn behind them; without drafts, one
  token drawn from each row.

Shapes are those of the benchmark's model (5120 wide: 40 query heads over 8 K/V heads of 128, a
fused q|k|v row of 7168, a vocabulary of 151936) and generic ones.

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

MOST_BYTES = 8192 * 48 * 128 * 2     # q and k of the largest listed rotation
MOST_LOGITS = 64 * 15 * 151936       # target and draft logits of the largest listed verification

# the scaled forms of the frequencies, with the numbers that models are published with
SCALING = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "ntk": {"type": "ntk", "factor": 4.0},
    "bands": {"type": "bands", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
              "original_length": 8192},
    "yarn": {"type": "yarn", "factor": 4.0, "original_length": 32768, "beta_fast": 32.0,
             "beta_slow": 1.0},
}


def _rope_case(name, kind, **kw):
    c = {"kind": kind, "slots": 1, "rows": 1, "q_heads": 40, "heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "scaling": "none", "base": 1e6, "dtype": "bf16",
         "far": 32768, "tree": False, "inverse": False}
    if kind == "norm_rope":
        c["offset"] = 0.0
    c.update(kw)
    if name:
        c["name"] = name
    return c


def _accept_case(name, **kw):
    c = {"kind": "accept", "slots": 1, "rows": 8, "vocab": 151936, "drafted": True, "mixed": False,
         "dtype": "bf16"}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decoded token of each of 8 sequences: latency
        _rope_case("rope_step", "rope", slots=8),
        # a prompt of 8192 tokens far into a context stretched four times over
        _rope_case("rope_prompt_yarn", "rope", rows=8192, scaling="yarn", far=120000),
        # ragged chunks of five prompts, a quarter of wide heads rotated in neighbouring pairs
        _rope_case("rope_partial_f16", "rope", slots=5, rows=333, q_heads=16, heads=2, dim=256,
                   rotary=64, interleaved=True, scaling="bands", base=5e5, dtype="f16"),
        # keys and queries turned back to position 0, fp32, heads of 80, the largest positions
        _rope_case("rope_back_f32", "rope", rows=1537, q_heads=7, heads=7, dim=80, rotary=32,
                   base=1e4, dtype="f32", far=1000000, inverse=True),
        # the verify block of one sequence: latency, once a layer
        _rope_case("norm_rope_block", "norm_rope", rows=8),
        # the same prompt of 8192 tokens with its heads' norms
        _rope_case("norm_rope_prompt", "norm_rope", rows=8192),
        # draft trees of 16 rows for 33 sequences, wide heads with a quarter rotated, weights
        # held as their distance from 1
        _rope_case("norm_rope_tree_f16", "norm_rope", slots=33, rows=16, q_heads=16, heads=2,
                   dim=256, rotary=64, dtype="f16", base=1e7, offset=1.0, tree=True),
        # seven drafts of a greedy drafter (no draft probabilities): latency
        _accept_case("accept_block", drafted=False),
        # 16 sequences with seven sampled drafts each
        _accept_case("accept_drafted", slots=16),
        # 64 sequences: the logits' bytes count
        _accept_case("accept_many", slots=64),
        # fp16 logits of an odd vocabulary, four drafts, greedy and sampled sequences mixed
        _accept_case("accept_mixed_f16", slots=5, rows=5, vocab=32003, mixed=True, dtype="f16"),
        # plain sampling: one row of fp32 logits for each of 33 sequences, no drafts
        _accept_case("sample_f32", slots=33, rows=1, vocab=50257, drafted=False, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "norm_rope", "norm_rope", "accept", "accept"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "accept":
        vocab = _log(rng, 1000, 151936)
        rows = rng.randint(1, 16)
        drafted = rows > 1 and rng.random() < 0.6
        each = vocab * (2 * rows - 1 if drafted else rows) * SIZE[dtype] // 2
        slots = max(1, min(_log(rng, 1, 64), MOST_LOGITS // each))
        return _accept_case(None, slots=slots, rows=rows, vocab=vocab, drafted=drafted,
                            mixed=rng.random() < 0.3, dtype=dtype)
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    heads = rng.choice([1, 2, 4, 8])
    q_heads = heads * rng.choice([1, 2, 3, 4, 5])
    rotary = rng.choice([dim, dim, dim // 2, dim // 4])
    most = MOST_BYTES // ((q_heads + heads) * dim * SIZE[dtype])
    tokens = min(_log(rng, 1, 8192), most)
    slots = min(_log(rng, 1, 64), tokens)
    c = {"slots": slots, "rows": tokens // slots, "q_heads": q_heads, "heads": heads, "dim": dim,
         "rotary": rotary, "interleaved": rng.random() < 0.4,
         "scaling": rng.choice(sorted(SCALING)), "base": rng.choice([1e4, 5e5, 1e6, 1e7]),
         "dtype": dtype, "far": _log(rng, 1, 1000000), "tree": rng.random() < 0.3}
    if kind == "norm_rope":
        c["offset"] = rng.choice([0.0, 1.0])
    else:
        c["inverse"] = rng.random() < 0.3
    return _rope_case(None, kind, **c)


# ---- inputs -------------------------------------------------------------------------------

def frequencies(rotary, base, scaling):
    """Radians a position of each pair, and the factor of the rotated channels."""
    n = rotary // 2
    if not scaling:
        return [base ** (-2.0 * i / rotary) for i in range(n)], 1.0
    factor, kind = scaling["factor"], scaling["type"]
    if kind == "ntk":
        base = base * factor ** (rotary / max(rotary - 2, 1))
    f = [base ** (-2.0 * i / rotary) for i in range(n)]
    if kind == "ntk":
        return f, 1.0
    if kind == "linear":
        return [x / factor for x in f], 1.0
    original = scaling["original_length"]
    out = []
    if kind == "bands":
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        for x in f:
            turns = original * x / (2 * math.pi)   # of the original context
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            out.append(keep * x + (1 - keep) * x / factor)
        return out, 1.0
    # yarn: pairs that turn often keep their frequency, those that turn seldom are stretched
    edge = [rotary * math.log(original / (b * 2 * math.pi)) / (2 * math.log(base))
            for b in (scaling["beta_fast"], scaling["beta_slow"])]
    low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rotary - 1)
    for i, x in enumerate(f):
        stretch = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
        out.append(stretch * x / factor + (1 - stretch) * x)
    return out, 0.1 * math.log(factor) + 1.0


def _prepare_rope(s, case, gen):
    b, m, d, dt = case["slots"], case["rows"], case["dim"], DT[case["dtype"]]
    hq, h = case["q_heads"], case["heads"]
    fused = torch.randn(b, m, (hq + 2 * h) * d, device="cuda", generator=gen)
    # heads and channels of sizes of their own, as projections have them
    fused *= torch.exp(0.5 * torch.randn((hq + 2 * h) * d, device="cuda", generator=gen))
    fused = fused.to(dt)
    s["q"] = fused[..., :hq * d].unflatten(-1, (hq, d))
    s["k"] = fused[..., hq * d:(hq + h) * d].unflatten(-1, (h, d))
    start = torch.randint(0, case["far"] + 1, (b,), device="cuda", generator=gen)
    s["starts"], s["positions"] = start.to(torch.int32), None
    if case["tree"]:
        # row j hangs on an earlier row and sits one position behind it
        depth = torch.zeros(b, m, dtype=torch.int64)
        parent = torch.randint(0, 1 << 20, (b, m), device="cuda", generator=gen).cpu()
        for j in range(1, min(m, 64)):
            depth[:, j] = depth.gather(1, (parent[:, j] % j)[:, None])[:, 0] + 1
        depth[:, 64:] = parent[:, 64:] % 64
        s["positions"] = (start[:, None] + depth.cuda()).to(torch.int32)
    f, s["amplitude"] = frequencies(case["rotary"], case["base"], SCALING[case["scaling"]])
    s["frequencies"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    if case["kind"] == "norm_rope":
        for name in ("q_weight", "k_weight"):
            w = 1 - case["offset"] + 0.2 * torch.randn(d, device="cuda", generator=gen)
            s[name] = w.to(dt)


def _normal(shape, dt, gen):
    """2.5 times normal numbers, made in pieces that fit beside the logits."""
    x = torch.empty(shape, dtype=dt, device="cuda")
    flat = x.view(-1, shape[-1])
    for r in range(0, flat.shape[0], 256):
        part = flat[r:r + 256]
        part.copy_(2.5 * torch.randn(part.shape, device="cuda", generator=gen))
    return x


def _prepare_accept(s, case, gen):
    b, m, v, dt = case["slots"], case["rows"], case["vocab"], DT[case["dtype"]]
    x = _normal((b, m, v), dt, gen)
    # rows are more or less decided: one token is lifted above the others
    lift = 6 + 20 * torch.rand(b, m, 1, device="cuda", generator=gen)
    best = torch.randint(0, v, (b, m, 1), device="cuda", generator=gen)
    x.scatter_add_(-1, best, lift.to(dt))
    t = torch.rand(b, device="cuda", generator=gen) * 0.8 + 0.4
    if case["mixed"]:
        t[torch.rand(b, device="cuda", generator=gen) < 0.4] = 0.0
    s["logits"], s["temperature"] = x, t
    s["uniforms"] = torch.rand(b, m, device="cuda", generator=gen)
    s["draft_logits"] = s["drafts"] = s["lengths"] = None
    if m == 1:
        return
    # some sequences bring fewer drafts than the block has room for
    n = torch.randint(0, 4 * m, (b,), device="cuda", generator=gen)
    s["lengths"] = torch.clamp(n, max=m - 1).to(torch.int32)
    if not case["drafted"]:
        # a greedy drafter that agrees with the lifted token more often than not
        other = torch.randint(0, v, (b, m - 1), device="cuda", generator=gen)
        agree = torch.rand(b, m - 1, device="cuda", generator=gen) < 0.8
        s["drafts"] = torch.where(agree, best[:, :-1, 0], other).to(torch.int32)
        return
    # a drafter that knows the target well, and what it drew
    y = _normal((b, m - 1, v), dt, gen)
    for i in range(b):
        y[i] = (0.3 * y[i].float() + 0.9 * x[i, :-1].float()).to(dt)
    s["draft_logits"] = y
    drafts = torch.empty(b, m - 1, dtype=torch.int32, device="cuda")
    for i in range(b):
        z = y[i].float()
        # the largest of logits plus Gumbel numbers is a draw from their softmax
        noise = torch.rand(z.shape, device="cuda", generator=gen).clamp_(1e-10, 1 - 1e-7)
        noise = -torch.log(-torch.log(noise))
        drafts[i] = (z + noise * t[i]).argmax(-1)
    s["drafts"] = drafts


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    s = dict(case)
    if case["kind"] == "accept":
        _prepare_accept(s, case, gen)
    else:
        _prepare_rope(s, case, gen)
    return s


# ---- the plain forms ------------------------------------------------------------------------

def _positions(s):
    if s["positions"] is not None:
        return s["positions"].double()
    rows = torch.arange(s["rows"], device="cuda")
    return (s["starts"].long()[:, None] + rows).double()


def _plain_rope(s):
    # angles of far positions need 64 bits
    angle = _positions(s)[..., None, None] * s["frequencies"]
    if s["inverse"]:
        angle = -angle
    cos = (angle.cos() * s["amplitude"]).float()
    sin = (angle.sin() * s["amplitude"]).float()
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        if s["kind"] == "norm_rope":
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
            x = x * (s[name + "_weight"].float() + s["offset"])
        y = x.clone()
        r = s["rotary"]
        if s["interleaved"]:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = x[..., :r // 2], x[..., r // 2:r]
            y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
        out[name] = y.to(s[name].dtype)
    return out


def _probabilities(x, temperature, mixed):
    """softmax(x / T) of x [slots, rows, V] in 64 bits; the first largest alone where T is 0, as
    it may be in mixed batches."""
    x = x.double()
    top = x.amax(-1, keepdim=True)
    t = temperature.double()[:, None, None]
    e = torch.exp((x - top) / torch.where(t > 0, t, torch.ones_like(t)))
    p = e / e.sum(-1, keepdim=True)
    if mixed:
        at = torch.arange(x.shape[-1], device=x.device)
        first = torch.where(x == top, at, x.shape[-1]).amin(-1, keepdim=True)
        p = torch.where(t > 0, p, (at == first).double())
    return p


def _plain_accept(s):
    b, m = s["slots"], s["rows"]
    p = _probabilities(s["logits"], s["temperature"], s["mixed"])
    u = s["uniforms"].double()
    row = torch.arange(b, device="cuda")
    if m == 1:
        n, left = torch.zeros_like(row), p[:, 0]
        chances = p.new_zeros(b, 0)
    else:
        d = s["drafts"].long()
        mine = p[:, :-1].gather(-1, d[..., None])[..., 0]
        if s["drafted"]:
            q = _probabilities(s["draft_logits"], s["temperature"], s["mixed"])
            # a greedy sequence's draft is its drafter's one choice
            one = torch.zeros_like(q).scatter_(-1, d[..., None], 1.0)
            q = torch.where((s["temperature"] > 0)[:, None, None], q, one)
            theirs = q.gather(-1, d[..., None])[..., 0]
        else:
            theirs = torch.ones_like(mine)
        given = torch.arange(m - 1, device="cuda") < s["lengths"][:, None]
        taken = given & (u[:, :-1] * theirs < mine)
        chances = torch.where(theirs > 0, (mine / theirs).clamp(max=1), (mine > 0).double())
        chances = chances * given
        n = taken.long().cumprod(-1).sum(-1)
        refused = n < s["lengths"]
        at = n.clamp(max=m - 2)
        left = p[row, n]
        if s["drafted"]:
            less = (left - q[row, at]).clamp(min=0)
        else:
            less = left.scatter(-1, d[row, at][:, None], 0.0)
        less = torch.where(less.sum(-1, keepdim=True) > 0, less, left)
        left = torch.where(refused[:, None], less, left)
    total = left.cumsum(-1)
    short = (total <= u[:, -1:] * total[:, -1:]).sum(-1)
    tokens = torch.full((b, m), -1, dtype=torch.int32, device="cuda")
    if m > 1:
        at = torch.arange(m - 1, device="cuda")
        tokens[:, :-1] = torch.where(at < n[:, None], s["drafts"], tokens[:, :-1])
    tokens[row, n] = short.to(torch.int32)
    return {"tokens": tokens, "accepted": n.to(torch.int32), "chances": chances.float()}


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


def _own(s):
    ctx = _context()
    if s["kind"] == "accept":
        tokens, accepted, chances = ctx.sample_accept(
            s["logits"], s["uniforms"], drafts=s["drafts"], draft_logits=s["draft_logits"],
            temperature=s["temperature"], draft_lengths=s["lengths"])
        return {"tokens": tokens, "accepted": accepted, "chances": chances}
    if "rope" not in s:
        # the table that a program keeps beside the model's weights
        import dflash_qmm
        s["rope"] = dflash_qmm.Rope(s["rotary"], base=s["base"], interleaved=s["interleaved"],
                                    scaling=SCALING[s["scaling"]])
    where = {"starts": s["starts"]} if s["positions"] is None else {"positions": s["positions"]}
    if s["kind"] == "rope":
        q, k = ctx.rope(s["rope"], s["q"], s["k"], inverse=s["inverse"], **where)
    else:
        q, k = ctx.qk_norm_rope(s["rope"], s["q"], s["k"], s["q_weight"], s["k_weight"], eps=1e-6,
                                weight_offset=s["offset"], **where)
    return {"q": q, "k": k}


def run(s):
    if own:
        return _own(s)
    return _plain_accept(s) if s["kind"] == "accept" else _plain_rope(s)


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    b, m = case["slots"], case["rows"]
    if case["kind"] == "accept":
        rows = b * (2 * m - 1 if case["drafted"] else m)
        n = rows * case["vocab"]
        # a subtraction, a product, an exponential, a comparison and a sum a logit
        return {"bytes": n * SIZE[case["dtype"]] + b * (16 * m + 12), "flops": 6 * n}
    n = b * m * (case["q_heads"] + case["heads"]) * case["dim"]
    small = 4 * b * (m if case["tree"] else 1) + 4 * case["rotary"]
    # a pair's rotation is four products and two sums; a norm squares, sums and scales twice
    turned = n * case["rotary"] // case["dim"]
    return {"bytes": 2 * n * SIZE[case["dtype"]] + small,
            "flops": 3 * turned + (4 * n if case["kind"] == "norm_rope" else 0)}


# ---- the definition in 64 bits --------------------------------------------------------------

def _exact_rope(s, sign):
    if s["positions"] is not None:
        pos = s["positions"].double()
    else:
        pos = s["starts"].double().unsqueeze(1) + torch.arange(float(s["rows"]), device="cuda",
                                                               dtype=torch.float64)
    turn = torch.polar(torch.full_like(pos, s["amplitude"])[..., None].expand(
        *pos.shape, s["rotary"] // 2).contiguous(), sign * pos[..., None] * s["frequencies"])
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        if s["kind"] == "norm_rope":
            size = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
            x = x / torch.sqrt(size ** 2 / s["dim"] + 1e-6)
            x = x * (s["offset"] + s[name + "_weight"].double())
        turned, rest = x.split((s["rotary"], s["dim"] - s["rotary"]), -1)
        if s["interleaved"]:
            z = torch.view_as_complex(turned.unflatten(-1, (-1, 2)).contiguous())
            y = torch.view_as_real(z * turn[:, :, None]).flatten(-2)
        else:
            z = torch.complex(*turned.chunk(2, -1)) * turn[:, :, None]
            y = torch.cat((z.real, z.imag), -1)
        out[name] = torch.cat((y, rest), -1)
    return out


def _exact_row(x, t):
    """The distribution of one row of logits at temperature t."""
    x = x.double()
    if t == 0:
        p = torch.zeros_like(x)
        p[int(torch.nonzero(x == x.max())[0])] = 1.0
        return p
    # not torch.softmax, which keeps about 32 bits of 64-bit rows here
    w = torch.exp2((x - x.max()) * (math.log2(math.e) / t))
    return w / torch.sum(w)


def _exact_accept(s):
    b, m = s["slots"], s["rows"]
    tokens = torch.full((b, m), -1, dtype=torch.int32)
    accepted = torch.zeros(b, dtype=torch.int32)
    chances = torch.zeros(b, m - 1, dtype=torch.float64)
    u, temperature = s["uniforms"].tolist(), s["temperature"].tolist()
    lengths = [0] * b if s["lengths"] is None else s["lengths"].tolist()
    drafts = [[]] * b if s["drafts"] is None else s["drafts"].tolist()
    for i in range(b):
        t, n, left = temperature[i], 0, None
        for j in range(lengths[i] + 1):
            p = _exact_row(s["logits"][i, j], t)
            if j == lengths[i]:
                left = p if left is None else left
                break
            d = drafts[i][j]
            if s["drafted"] and t > 0:
                q = _exact_row(s["draft_logits"][i, j], t)
            else:
                q = torch.zeros_like(p)
                q[d] = 1.0
            mine, theirs = float(p[d]), float(q[d])
            chances[i, j] = min(1.0, mine / theirs) if theirs > 0 else float(mine > 0)
            if left is not None:
                continue   # behind the first that is refused
            if u[i][j] * theirs < mine:
                tokens[i, j] = d
                n += 1
                continue
            left = torch.relu(p - q)
            left = left if float(left.sum()) > 0 else p
        c = torch.cumsum(left, 0)
        at = torch.searchsorted(c, c[-1] * u[i][m - 1], right=True)
        tokens[i, n], accepted[i] = int(at), n
    return {"tokens": tokens.cuda(), "accepted": accepted.cuda(), "chances": chances.cuda()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "accept":
        return _exact_accept(s)
    return _exact_rope(s, -1.0 if s["inverse"] else 1.0)
