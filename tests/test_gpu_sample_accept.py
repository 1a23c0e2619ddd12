"""The sampled accept against its definition in 64 bits: shapes, types, temperatures, masks, rows
without a distribution, borders, strides, and the law that its tokens follow."""
import itertools
import math

import numpy as np
import pytest
import torch

import dflash_qmm
from gpu_util import announce
from rotation_util import DTYPES, accept, distribution

pytestmark = pytest.mark.gpu

# A draft's chance, from two rows' fp32 sums: an exponent a of 2 has three roundings, 2.5 * 2^-24 |a|
# together, and the mean of |a| over a row's mass is at most the logarithm of its tokens' number,
# 20 here: 34 * 2^-24 of the sum; 13 sums in a row and the exponential's last bits are 20 more.
CHANCE = 2.0 * 54 * 2.0 ** -24


def inputs(seed, batch, rows, vocab, name, drafted, spread=3.0, mixed=False):
    gen = torch.Generator().manual_seed(seed)
    dt = DTYPES[name]
    x = (spread * torch.randn(batch, rows, vocab, generator=gen)).to(dt)
    s = {"logits": x, "uniforms": torch.rand(batch, rows, generator=gen), "drafts": None,
         "draft_logits": None, "draft_lengths": None,
         "temperature": 0.3 + torch.rand(batch, generator=gen)}
    if mixed:
        s["temperature"][::2] = 0
    if rows > 1:
        top = x[:, :-1].float().argmax(-1)
        other = torch.randint(0, vocab, top.shape, generator=gen)
        s["drafts"] = torch.where(torch.rand(top.shape, generator=gen) < 0.7, top,
                                  other).to(torch.int32)
        s["draft_lengths"] = torch.randint(-1, 3 * rows, (batch,), generator=gen).to(torch.int32)
        if drafted:
            y = x[:, :-1].float() + torch.randn(batch, rows - 1, vocab, generator=gen)
            s["draft_logits"] = y.to(dt)
    return s


def on_gpu(s):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}


def oracle(s):
    batch = s["logits"].shape[0]

    def numbers(t):
        return t.double().numpy() if isinstance(t, torch.Tensor) else [float(t)] * batch
    td = s.get("draft_temperature")
    return accept(s["logits"].double().numpy(), s["uniforms"].numpy().astype(np.float64),
                  None if s["drafts"] is None else s["drafts"].numpy(),
                  None if s["draft_lengths"] is None else s["draft_lengths"].numpy(),
                  None if s["draft_logits"] is None else s["draft_logits"].double().numpy(),
                  numbers(s["temperature"]), numbers(s["temperature"] if td is None else td))


# Exponentials are right to 8e-13 of themselves, and so are two rows' sums: 4 of them, twice over.
NEAR = 7e-12


def check(ctx, s, margin=NEAR):
    """One call against the definition; no decision of the inputs may lie nearer to its border
    than the arithmetic's bound."""
    tokens, accepted, chances, near = oracle(s)
    assert near > margin, f"these inputs decide by {near}: take others"
    got = ctx.sample_accept(**on_gpu(s))
    torch.cuda.synchronize()
    assert got[0].cpu().tolist() == tokens.tolist()
    assert got[1].cpu().tolist() == accepted.tolist()
    off = np.abs(got[2].double().cpu().numpy() - chances)
    assert (off <= CHANCE * chances + 1e-37).all(), off.max()
    return got


SIZES = [(1, 1, 1), (1, 1, 2), (3, 2, 1), (2, 3, 7), (1, 8, 300), (5, 1, 1000), (1, 4, 2048),
         (2, 5, 2049), (3, 16, 5000), (2, 64, 257), (33, 1, 4097), (1, 2, 33000), (70, 3, 64)]


@pytest.mark.parametrize("batch,rows,vocab", SIZES)
@pytest.mark.parametrize("name", sorted(DTYPES))
def test_sizes(ctx, batch, rows, vocab, name):
    for drafted, mixed in itertools.product((False, True), (False, True)):
        announce(f"accept {batch} {rows} {vocab} {name} {drafted} {mixed}")
        check(ctx, inputs(vocab + rows, batch, rows, vocab, name, drafted, mixed=mixed))


@pytest.mark.parametrize("name", sorted(DTYPES))
def test_a_large_vocabulary(ctx, name):
    for drafted in (False, True):
        announce(f"accept 151936 {name} {drafted}")
        s = inputs(3, 2, 3, 151936, name, drafted)
        s["logits"][:, :, 7::40000] += 12
        check(ctx, s)


@pytest.mark.parametrize("temperature", [1e-40, 1e-30, 1e-4, 0.01, 50.0, 1e20])
def test_extreme_temperatures(ctx, temperature):
    for name, drafted in itertools.product(sorted(DTYPES), (False, True)):
        announce(f"accept T {temperature} {name} {drafted}")
        s = inputs(17, 4, 4, 500, name, drafted)
        s["temperature"] = torch.full((4,), temperature)
        check(ctx, s, margin=0)


def test_scalar_and_separate_temperatures(ctx):
    for t, td in ((0.8, None), (0.7, 1.3), (0.0, None), (0.9, 0.0), (0.0, 0.6),
                  (torch.tensor([0.5, 0.0, 1.5]), torch.tensor([0.0, 0.7, 0.9])),
                  (1.0, torch.tensor([0.5, 0.0, 1.5])), (torch.tensor([0.5, 0.0, 1.5]), 0.8)):
        for drafted in (False, True):
            s = inputs(18, 3, 5, 400, "f32", drafted)
            s["temperature"], s["draft_temperature"] = t, td
            announce(f"accept T {t} {td}")
            check(ctx, s)


def test_greedy_is_the_argmax_accept(ctx):
    for name in ("bf16", "f16"):   # the types that argmax_accept takes
        s = inputs(19, 1, 8, 3001, name, False)
        s["logits"] = s["logits"].round()   # many equal logits
        s["logits"][0, 3, 5] = math.nan
        s["drafts"] = s["logits"][:, :-1].float().nan_to_num(-100).argmax(-1).to(torch.int32)
        s["drafts"][0, 6] = 9
        s["draft_lengths"] = None
        s["temperature"] = 0.0
        g = on_gpu(s)
        tokens, accepted, _ = ctx.sample_accept(**g)
        want, count = ctx.argmax_accept(g["logits"][0], g["drafts"][0])
        n = int(count)
        assert int(accepted) == n
        assert tokens[0, :n + 1].tolist() == want[:n + 1].tolist()
        assert (tokens[0, n + 1:] == -1).all()


@pytest.mark.parametrize("name", sorted(DTYPES))
def test_masked_logits(ctx, name):
    """-inf and the type's lowest value in most places, and rows that are all the lowest value."""
    low = torch.finfo(DTYPES[name]).min
    for mask, drafted in itertools.product((-math.inf, low), (False, True)):
        announce(f"accept masked {name} {mask}")
        s = inputs(20, 4, 4, 3000, name, drafted)
        keep = torch.rand(s["logits"].shape, generator=torch.Generator().manual_seed(1)) < 0.01
        keep[..., 77] = True
        s["logits"][~keep] = mask
        if drafted:
            s["draft_logits"][~keep[:, :-1]] = mask
        check(ctx, s)
        if mask == low:
            s["logits"][1, 0] = low
            s["logits"][2] = low
            check(ctx, s)
        s["temperature"] = 0.0
        check(ctx, s)


def test_a_draft_that_its_own_distribution_rules_out(ctx):
    s = inputs(21, 2, 3, 100, "f32", True)
    s["draft_lengths"] = None
    for b in range(2):
        s["draft_logits"][b, 0, int(s["drafts"][b, 0])] = -math.inf
    s["logits"][1, 0, int(s["drafts"][1, 0])] = -math.inf
    got = check(ctx, s)
    assert got[2][0, 0] == 1 and got[2][1, 0] == 0


def test_rows_without_a_distribution(ctx):
    """NaN, +inf, nothing above -inf, and temperatures that are none: the draft is refused and no
    token is drawn; other sequences are not touched by it."""
    for drafted, name in itertools.product((False, True), sorted(DTYPES)):
        s = inputs(22, 8, 4, 700, name, drafted)
        s["draft_lengths"] = None
        s["logits"][0, 0, 5] = math.nan
        s["logits"][1, 1, 699] = math.inf
        s["logits"][2, 2] = -math.inf
        s["logits"][3, 3, 0] = math.nan
        s["temperature"][4:7] = torch.tensor([-1.0, math.inf, math.nan])
        if drafted:
            s["draft_logits"][7, 1, 3] = math.nan
        else:
            s["logits"][7, 1] = math.nan
        announce(f"accept without {name} {drafted}")
        got = check(ctx, s)
        assert got[0][0].tolist() == [-1] * 4 and got[0][4:7].tolist() == [[-1] * 4] * 3
        s["temperature"][:] = 0
        check(ctx, s)
    s["logits"][3, 0] = math.nan
    s["temperature"][:] = 0
    assert check(ctx, s)[0][3].tolist() == [-1] * 4


def test_drafts_outside_the_vocabulary(ctx):
    for drafted in (False, True):
        s = inputs(23, 3, 3, 900, "bf16", drafted)
        s["drafts"][:, 0] = torch.tensor([-1, 900, 2 ** 31 - 1])
        s["draft_lengths"] = None
        assert check(ctx, s)[1].tolist() == [0, 0, 0]
        s["temperature"][:] = 0
        check(ctx, s)


@pytest.mark.parametrize("batch,vocab", [(5, 900), (3, 33000), (100, 90000)])
def test_drafts_outside_the_vocabulary_where_p_is_q(ctx, batch, vocab):
    """p - q is 0 throughout: the token comes from p."""
    s = inputs(26, batch, 2, vocab, "bf16", True)
    s["draft_logits"] = s["logits"][:, :-1].clone()
    s["draft_lengths"] = None
    s["drafts"][:] = -1
    announce(f"accept outside, p = q {batch} {vocab}")
    got = check(ctx, s)
    assert (got[1] == 0).all() and (got[0][:, 0] >= 0).all()


@pytest.mark.parametrize("batch,vocab,size", [
    (4, 900, 1e-6), (4, 900, 2.0 ** -16), (4, 900, 2.0 ** -14), (4, 900, 1e-2),
    (3, 60000, 2.0 ** -16), (3, 60000, 2.0 ** -14), (3, 60000, 1e-2), (40, 50000, 1e-2)])
def test_rests_of_nearly_equal_distributions(ctx, batch, vocab, size):
    """Many tokens in which p is nearly q, more of them above it, below it, and equal."""
    s = inputs(31, batch, 2, vocab, "f32", True)
    gen = torch.Generator().manual_seed(28)
    by = torch.randn(batch, 1, vocab, generator=gen) * size
    by[..., ::7] = 0
    s["draft_logits"] = s["logits"][:, :-1] + by
    s["draft_lengths"] = None
    s["drafts"][:] = -1
    announce(f"accept nearly equal {batch} {vocab} {size}")
    # two exponentials and two sums, each right to 8e-13, in a running sum and in the whole: 6.4e-12
    # of p; what is left of p is 0.4 of the size times 6/7
    got = check(ctx, s, margin=2e-11 / size)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("vocab", [900, 30000])
@pytest.mark.parametrize("banned", ["target", "draft"])
def test_rests_of_distributions_that_differ_in_few_tokens(ctx, name, vocab, banned):
    """The same logits, but for a few unlikely tokens that one of the two rules out: every other
    token's p / q is the same number next to 1, a little above or below it."""
    s = inputs(32, 3, 2, vocab, name, True)
    s["draft_logits"] = s["logits"][:, :-1].clone()
    s["draft_lengths"] = None
    s["temperature"][:] = 1.0
    s["drafts"][:] = -1
    s["logits"][:, 0, 5::vocab // 3] = s["draft_logits"][:, 0, 5::vocab // 3] = -1.0
    s["logits" if banned == "target" else "draft_logits"][:, 0, 5::vocab // 3] = -math.inf
    left = [np.maximum(distribution(s["logits"][b, 0].double().numpy(), 1.0) -
                       distribution(s["draft_logits"][b, 0].double().numpy(), 1.0), 0).sum()
            for b in range(3)]
    assert max(left) < 2.0 ** -9 and (vocab == 900 or max(left) < 2.0 ** -15)
    announce(f"accept few tokens {name} {vocab} {banned}")
    got = check(ctx, s, margin=2 * 6.4e-12 / min(left))
    assert (got[1] == 0).all() and (got[0][:, 0] >= 0).all()


def test_the_edges_of_the_random_numbers(ctx):
    """0 takes any draft that can be and the first token that can be; 1 - 2^-24 the last."""
    last = 1 - 2.0 ** -24
    s = inputs(24, 2, 3, 5000, "f32", False)
    s["draft_lengths"] = torch.tensor([2, 0], dtype=torch.int32)
    s["logits"][:, :, :17] = -math.inf
    s["logits"][:, :, 4990:] = -math.inf
    s["logits"][:, 2, 4989] = s["logits"][:, 0, 4989] = 9.0
    s["uniforms"][:] = 0
    tokens, accepted, _ = ctx.sample_accept(**on_gpu(s))
    assert accepted.tolist() == [2, 0] and tokens[0, 2] == 17 and tokens[1, 0] == 17
    s["uniforms"][:] = last
    tokens, accepted, _ = ctx.sample_accept(**on_gpu(s))
    want = oracle(s)
    assert accepted.tolist() == want[1].tolist() and tokens.tolist() == want[0].tolist()
    # numbers outside [0, 1) are the caller's mistake, and still give tokens of the row
    for u in (1.0, 7.0, -3.0, math.nan):
        s["uniforms"][:] = u
        tokens, accepted, _ = ctx.sample_accept(**on_gpu(s))
        assert ((tokens >= -1) & (tokens < 4990)).all() and tokens[1, 0] >= 17


@pytest.mark.parametrize("vocab", [3000, 300000])
def test_many_tokens_of_no_weight_in_front(ctx, vocab):
    """Probabilities under 2^-1000 of the largest are 0, also where hundreds of them side by side
    would come to more: u = 0 takes the first of the others."""
    at = vocab - 700
    x = torch.full((4, 2, vocab), -695.0)      # e^-695 = 2^-1002.7
    x[..., at] = 0
    x[..., at + 1] = -690.0                    # 2^-995.5
    y = torch.full((4, 1, vocab), -695.0)
    y[..., at + 300] = 2.0
    x[2:, 0, at + 300] = 0
    for drafts in ([at, at + 300, at, at + 300], [-1] * 4, [5] * 4):
        for draft_logits in (None, y):
            u = torch.zeros(4, 2)
            u[:, 0] = 1 - 2.0 ** -24
            announce(f"accept of no weight {vocab} {drafts}")
            tokens, accepted, _ = ctx.sample_accept(
                x.cuda(), u.cuda(), torch.tensor(drafts, dtype=torch.int32)[:, None].cuda(),
                draft_logits=None if draft_logits is None else draft_logits.cuda())
            for b in range(4):
                n, d = int(accepted[b]), drafts[b]
                first = at if n or draft_logits is not None or d != at else at + 1
                assert tokens[b, n] == first, (b, n, d, tokens[b].tolist())
                assert n == 0 or d in (at, at + 300)


def test_a_draw_at_its_border(ctx):
    """Two equal tokens: the first's running sum is the half, and u = 0.5 is not passed by it."""
    for name in sorted(DTYPES):
        x = torch.full((2, 1, 4000), -math.inf, dtype=DTYPES[name])
        x[..., 100] = x[..., 3900] = 1.5
        u = torch.tensor([[0.5], [0.5 - 2.0 ** -25]])
        tokens, _, _ = ctx.sample_accept(x.cuda(), u.cuda())
        assert tokens[:, 0].tolist() == [3900, 100]


def test_equal_distributions_accept_everything(ctx):
    """p = q: chances of 1, whatever the numbers are below 1."""
    s = inputs(25, 6, 9, 6000, "bf16", True)
    s["draft_logits"] = s["logits"][:, :-1].clone()
    s["draft_lengths"] = None
    s["uniforms"][:, :-1] = 1 - 2.0 ** -24
    tokens, accepted, chances = ctx.sample_accept(**on_gpu(s))
    assert accepted.tolist() == [8] * 6 and (chances == 1).all()


@pytest.mark.parametrize("drafted", (False, True))
def test_tokens_follow_the_target(ctx, drafted):
    """Over a grid of random numbers the first token of a block is distributed as p: drafts drawn
    from q (every token as often as q has it) and refused, accepted or redrawn.  Steps of the grid
    leave each of the 6 tokens at most 2 borders a draft, off by a step of 1/256 each."""
    n, vocab = 256, 6
    gen = torch.Generator().manual_seed(2)
    p_logits, q_logits = 1.5 * torch.randn(2, vocab, generator=gen)
    p, q = p_logits.double().softmax(0), q_logits.double().softmax(0)
    grid = (torch.arange(n) + 0.5) / n
    u = torch.stack((grid.repeat_interleave(n), grid.repeat(n)), 1)
    law = torch.zeros(vocab, dtype=torch.float64)
    for d in range(vocab):
        if not drafted and d:
            break
        x = torch.stack((p_logits, torch.zeros(vocab)))
        tokens, _, _ = ctx.sample_accept(
            x.cuda().expand(n * n, -1, -1), u.cuda(),
            drafts=torch.full((n * n, 1), d, dtype=torch.int32, device="cuda"),
            draft_logits=q_logits.cuda().expand(n * n, 1, -1) if drafted else None)
        counts = tokens[:, 0].long().cpu().bincount(minlength=vocab).double() / (n * n)
        law += counts * (q[d] if drafted else 1.0)
    assert (law - p).abs().max() <= 4.0 / n


def test_strides(ctx):
    """Rows and sequences apart, at odd offsets; logits and draft logits of one tensor."""
    for name in sorted(DTYPES):
        s = inputs(26, 3, 4, 2500, name, True)
        room = torch.zeros(3, 9, 2611, dtype=DTYPES[name])
        room[:, ::2, 3:2503][:, :4] = s["logits"]
        room[:, 1::2, 111:][:, :3, :2500] = s["draft_logits"]
        want = check(ctx, s)
        g = on_gpu(s)
        far = room.cuda()
        g["logits"] = far[:, ::2, 3:2503][:, :4]
        g["draft_logits"] = far[:, 1::2, 111:][:, :3, :2500]
        announce(f"accept strides {name}")
        got = ctx.sample_accept(**g)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_past_32_bits(ctx):
    s = inputs(27, 2, 2, 5000, "bf16", False)
    s["draft_lengths"] = None
    want = check(ctx, s)
    g = on_gpu(s)
    far = 2 ** 31 + 64
    big = torch.empty(far + 2 * 5000, dtype=torch.bfloat16, device="cuda")
    view = big.as_strided((2, 2, 5000), (far, 5000, 1))
    view.copy_(g["logits"])
    g["logits"] = view
    announce("accept far sequences")
    assert all(torch.equal(a, b) for a, b in zip(ctx.sample_accept(**g), want))
    view = big.as_strided((1, 2, 5000), (far, far, 1))
    one = {k: v[:1].contiguous() if isinstance(v, torch.Tensor) else v
           for k, v in on_gpu(s).items()}
    view.copy_(one["logits"])
    one["logits"] = view
    announce("accept far rows")
    assert all(torch.equal(a, b[:1]) for a, b in zip(ctx.sample_accept(**one), want))


def test_the_same_call_gives_the_same_bits(ctx):
    s = on_gpu(inputs(28, 20, 6, 30000, "bf16", True))
    first = ctx.sample_accept(**s)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(ctx.sample_accept(**s), first))


def test_captured_and_replayed(ctx):
    s = on_gpu(inputs(29, 5, 4, 9000, "f16", True))
    ws = torch.empty(8 << 20, dtype=torch.uint8, device="cuda")
    ctx.sample_accept(**s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ctx.sample_accept(**s, ws=ws)
    for n in range(4):
        s["uniforms"].copy_(torch.rand(5, 4, generator=torch.Generator().manual_seed(n)))
        for a in got:
            a.fill_(7)
        ws.fill_(n * 85)    # what a workspace holds does not matter
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ctx.sample_accept(**s)))


def test_graphs_captured_on_one_stream_run_at_once(ctx):
    """Each has a workspace of its own, apart from the eager calls' too."""
    side, sets, graphs = torch.cuda.Stream(), [], []
    for n in range(2):
        s = on_gpu(inputs(73 + n, 40, 4, 20003, "bf16", True))
        sets.append((s, ctx.sample_accept(**s)))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = ctx.sample_accept(**s)
        graphs.append((graph, got))
    streams = [torch.cuda.Stream() for _ in graphs]
    for n in range(20):
        for (graph, got), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                for a in got:
                    a.fill_(7)
                graph.replay()
        again = ctx.sample_accept(**sets[n % 2][0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, sets[n % 2][1])), n
        for (_, got), (_, want) in zip(graphs, sets):
            assert all(torch.equal(a, b) for a, b in zip(got, want)), n


def test_two_streams_at_once(ctx):
    cases = [on_gpu(inputs(30 + i, 6, 5, 40000, "bf16", True)) for i in range(2)]
    want = [ctx.sample_accept(**s) for s in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, stream in zip(cases, streams):
            got.append(ctx.sample_accept(**s, stream=stream))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def test_a_given_workspace(ctx):
    s = on_gpu(inputs(32, 2, 3, 5000, "f32", True))
    want = ctx.sample_accept(**s)
    small = torch.empty(64, dtype=torch.uint8, device="cuda")
    with pytest.raises(dflash_qmm.DfqError) as e:
        ctx.sample_accept(**s, ws=small)
    assert e.value.status == 3
    ws = torch.full((4 << 20,), 255, dtype=torch.uint8, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(ctx.sample_accept(**s, ws=ws), want))


def at_the_border(s, first):
    """The fp32 numbers nearest to each draft's chance, and their neighbours, as random numbers; a
    step further where one lies within 1e-11 of the chance, which exponentials to 8e-13 in both
    rows and both sums do not tell from it by far."""
    _, _, chances, _ = oracle(s)
    u = torch.from_numpy(chances).float()
    move = torch.arange(u.numel()).view(u.shape) % 3 - 1
    up, down = torch.full_like(u, 2.0), torch.full_like(u, -2.0)
    u = torch.where(move > 0, torch.nextafter(u, up),
                    torch.where(move < 0, torch.nextafter(u, down), u))
    near = (u.double().numpy() - chances) < 1e-11 * chances
    near &= (u.double().numpy() - chances) > -1e-11 * chances
    u = torch.where(torch.from_numpy(near), torch.nextafter(u, up), u).clamp(0, 1 - 2.0 ** -24)
    s["uniforms"][:, :-1] = u
    if first:   # drafts in front of the last are taken, so that each row is judged at its border
        s["uniforms"][:, :-2] = 0


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("vocab", [50, 3000, 33000])
def test_drafts_next_to_their_border(ctx, name, vocab):
    """Random numbers one fp32 step around the chances, which lie some 1e-8 from them: nearer than
    fp32 sums of the rows can tell, and decided as 64-bit sums decide them."""
    for drafted, first in itertools.product((False, True), (False, True)):
        s = inputs(40 + vocab, 24, 4, vocab, name, drafted)
        s["draft_lengths"] = None
        at_the_border(s, first)
        announce(f"accept at the border {vocab} {name} {drafted}")
        check(ctx, s)


@pytest.mark.parametrize("name", sorted(DTYPES))
def test_draws_next_to_their_border(ctx, name):
    """Random numbers within an fp32 step of the running sum's value at some token."""
    for drafted, rows in ((False, 1), (False, 2), (True, 2)):
        s = inputs(50, 40, rows, 4000, name, drafted, spread=1.0)
        s["draft_lengths"] = None
        if rows == 2:
            s["uniforms"][:, 0] = 1 - 2.0 ** -24   # refused, unless the chance is 1
        tokens, accepted, _, _ = oracle(s)
        for b in range(40):
            n = int(accepted[b])
            p = distribution(s["logits"][b, n].double().numpy(), float(s["temperature"][b]))
            left = p
            if n < rows - 1:
                q = np.zeros_like(p)
                q[int(s["drafts"][b, n])] = 1.0
                if drafted:
                    q = distribution(s["draft_logits"][b, n].double().numpy(),
                                     float(s["temperature"][b]))
                left = np.maximum(p - q, 0)
            run = left.cumsum() / left.sum()
            u = torch.tensor(run[500 + 87 * b], dtype=torch.float32)
            u = torch.nextafter(u, torch.tensor(float(b % 3 - 1))) if b % 3 else u
            s["uniforms"][b, -1] = u.clamp(0, 1 - 2.0 ** -24)
        announce(f"draw at the border {name} {drafted} {rows}")
        check(ctx, s)


@pytest.mark.parametrize("name", sorted(DTYPES))
def test_more_units_than_one_search_takes(ctx, name):
    for drafted in (False, True):
        announce(f"accept 700001 {name} {drafted}")
        s = inputs(60, 2, 2, 700001, name, drafted)
        s["uniforms"][0, 0] = 1 - 2.0 ** -24
        check(ctx, s)


def test_many_sequences(ctx):
    for batch, rows, vocab in ((1700, 1, 5000), (900, 3, 2100)):
        for drafted in (False, True):
            announce(f"accept {batch} sequences {drafted}")
            check(ctx, inputs(61, batch, rows, vocab, "bf16", drafted))


def test_a_certain_draft_refused_by_a_number_past_1(ctx):
    """p = q = 1 for one token, and u is not below 1: p is drawn from, which is that token."""
    for drafted in (False, True):
        x = torch.full((1, 2, 3000), -math.inf)
        x[..., 1234] = 0.5
        tokens, accepted, chances = ctx.sample_accept(
            x.cuda(), torch.tensor([[1.0, 0.3]]).cuda(),
            drafts=torch.tensor([[1234]], dtype=torch.int32).cuda(),
            draft_logits=x[:, :1].cuda() if drafted else None)
        assert tokens.tolist() == [[1234, -1]] and accepted.tolist() == [0]
        assert chances.tolist() == [[1.0]]


@pytest.mark.parametrize("name", sorted(DTYPES))
@pytest.mark.parametrize("border", (False, True))
def test_many_logits(ctx, name, border):
    """27 M logits with draft logits, ragged, greedy and bad rows among them, and drafts next to
    their border, which are decided again."""
    s = inputs(70, 190, 4, 20003, name, True, mixed=not border)
    if border:
        s["draft_lengths"] = None
        at_the_border(s, True)
    else:
        s["logits"][0, 0, 7] = math.nan
        s["logits"][1, 1] = -math.inf
        s["draft_logits"][3, 0, 20002] = math.inf
        s["temperature"][5] = -1.0
        s["uniforms"][9:40, 1] = 1 - 2.0 ** -24
    announce(f"accept 27 M logits {name} {border}")
    got = check(ctx, s)
    again = ctx.sample_accept(**on_gpu(s))
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_a_large_call_and_small_ones_agree(ctx):
    """The same sequences in one call and in small ones, whose work is split otherwise."""
    s = on_gpu(inputs(71, 26, 5, 120011, "bf16", True))
    whole = ctx.sample_accept(**s)
    for at in range(0, 26, 9):
        part = {k: v[at:at + 9] if isinstance(v, torch.Tensor) else v for k, v in s.items()}
        got = ctx.sample_accept(**part)
        assert torch.equal(got[0], whole[0][at:at + 9])
        assert torch.equal(got[1], whole[1][at:at + 9])
        off = (got[2] - whole[2][at:at + 9]).abs()
        assert bool((off <= CHANCE * got[2]).all())


def test_a_captured_call_with_draft_logits(ctx):
    s = on_gpu(inputs(72, 190, 4, 20003, "f16", True))
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    ctx.sample_accept(**s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ctx.sample_accept(**s, ws=ws)
    for n in range(3):
        s["uniforms"].copy_(torch.rand(190, 4, generator=torch.Generator().manual_seed(n)))
        ws.fill_(n * 85)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ctx.sample_accept(**s)))
