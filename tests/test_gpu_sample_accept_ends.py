"""The sampled accept at the ends of its arguments: temperatures of any size, and what a temperature
of 0 makes of rows that have no softmax."""
import math

import pytest
import torch

from gpu_util import announce
from rotation_util import DTYPES
from test_gpu_sample_accept import check, inputs

pytestmark = pytest.mark.gpu


def spread_evenly(s, least, step, name):
    """Every logit anew: least + step times a random whole number up to 256."""
    gen = torch.Generator().manual_seed(3)
    for key in ("logits", "draft_logits"):
        if s[key] is not None:
            k = torch.randint(0, 257, s[key].shape, generator=gen).double()
            s[key] = (least + step * k).float().to(DTYPES[name])
    top = s["logits"][:, :-1].float().argmax(-1)
    s["drafts"] = torch.where(torch.rand(top.shape, generator=gen) < 0.5, top,
                              s["drafts"].long()).to(torch.int32)


@pytest.mark.parametrize("drafted", (False, True))
@pytest.mark.parametrize("name", ("bf16", "f32"))
@pytest.mark.parametrize("temperature", [1e36, 3e37, 1e38, 3.4e38])
def test_logits_further_apart_than_fp32_holds(ctx, temperature, name, drafted):
    """Logits over the whole range of the type, whose differences pass it, at temperatures that make
    ordinary exponents of them."""
    announce(f"accept wide {temperature} {name} {drafted}")
    s = inputs(80, 6, 4, 700, name, drafted)
    spread_evenly(s, -3.3e38, 6.6e38 / 256, name)
    s["temperature"] = torch.full((6,), temperature)
    check(ctx, s)


@pytest.mark.parametrize("drafted", (False, True))
@pytest.mark.parametrize("name", ("bf16", "f32"))
def test_wide_logits_over_many_ranges(ctx, name, drafted):
    """The same over rows whose ranges' largest logits differ as much."""
    announce(f"accept wide rows {name} {drafted}")
    s = inputs(81, 2, 3, 20003, name, drafted)
    spread_evenly(s, -3.3e38, 6.6e38 / 256, name)
    for key in ("logits", "draft_logits"):
        if s[key] is not None:
            s[key][..., :9000] = s[key][..., :9000].float().clamp(max=-3.2e38).to(DTYPES[name])
    s["temperature"] = torch.full((2,), 1e38)
    check(ctx, s)


@pytest.mark.parametrize("drafted", (False, True))
@pytest.mark.parametrize("name,step,temperature", [
    ("f32", 2.0 ** -149, 40 * 2.0 ** -149), ("f32", 2.0 ** -149, 2.0 ** -149),
    ("f32", 2.0 ** -140, 1e-41), ("bf16", 2.0 ** -133, 30 * 2.0 ** -133),
    ("bf16", 2.0 ** -133, 1e-38)])
def test_logits_as_small_as_their_temperature(ctx, name, step, temperature, drafted):
    """Temperatures and logits below the least normal number."""
    announce(f"accept small {name} {step} {temperature} {drafted}")
    s = inputs(82, 6, 4, 700, name, drafted)
    spread_evenly(s, -100 * step, step, name)
    s["temperature"] = torch.full((6,), temperature)
    assert (s["temperature"] > 0).all() and s["logits"].float().unique().numel() > 100
    check(ctx, s)


@pytest.mark.parametrize("drafted", (False, True))
@pytest.mark.parametrize("name", ("bf16", "f32"))
@pytest.mark.parametrize("temperature", [2.0 ** -149, 1e-40, 2.0 ** -126])
def test_large_logits_at_the_least_temperatures(ctx, name, temperature, drafted):
    """One token has all of the row, or equal ones share it."""
    announce(f"accept one token {name} {temperature} {drafted}")
    s = inputs(83, 6, 4, 700, name, drafted)
    spread_evenly(s, -3.3e38, 6.6e38 / 256, name)
    s["temperature"] = torch.full((6,), temperature)
    check(ctx, s, margin=0)


def test_rows_at_temperature_0(ctx):
    """NaN is passed over, +inf is the largest, a row of -inf throughout gives its first token, and
    one of NaN throughout none; draft rows are not looked at where the draft's temperature is 0."""
    for name in sorted(DTYPES):
        announce(f"accept T 0 {name}")
        s = inputs(84, 5, 2, 3001, name, False)
        x = s["logits"]
        x[0, 0] = -math.inf
        x[1, 0, 40] = math.inf
        x[2, 0, ::2] = math.nan
        x[3, 0] = math.nan
        x[4, 1] = math.nan
        best = x[2, 0].float().nan_to_num(-math.inf).argmax()
        s["drafts"] = torch.tensor([[0], [40], [int(best)], [7], [int(x[4, 0].float().argmax())]],
                                   dtype=torch.int32)
        s["draft_lengths"], s["temperature"] = None, 0.0
        tokens, accepted, chances = check(ctx, s)
        assert accepted.tolist() == [1, 1, 1, 0, 1]
        assert tokens[:3, 0].tolist() == [0, 40, int(best)]
        assert tokens[3:, 1].tolist() == [-1, -1] and int(tokens[3, 0]) == -1
        assert chances[:, 0].tolist() == [1, 1, 1, 0, 1]
        # a certain draft's own row is not read
        s["draft_logits"], s["draft_temperature"] = torch.full_like(x[:, :1], math.nan), 0.0
        assert all(torch.equal(a, b) for a, b in zip(check(ctx, s), (tokens, accepted, chances)))
        # and one that was drawn has none: refused, and nothing drawn
        s["draft_temperature"] = 1.0
        assert check(ctx, s)[0].tolist() == [[-1, -1]] * 5
