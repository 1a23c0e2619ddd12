"""Head norms of heads and weights of any size against the 64-bit plain form."""
import pytest
import torch

import dflash_qmm
from gpu_util import announce
from rotation_util import DTYPES, check_rotated, rotated

pytestmark = pytest.mark.gpu

# chunks in halves, with idle lanes, over 16 and 32 lanes, and pair by pair
WIDTHS = [(128, 128), (80, 32), (256, 64), (512, 128), (64, 20), (6, 4)]


def normed(ctx, q, weight, eps, rotary, interleaved, offset=0.0):
    """q's norms and rotation from position 3 on against the plain form."""
    rope = dflash_qmm.Rope(rotary, interleaved=interleaved)
    y = ctx.qk_norm_rope(rope, q, None, weight, eps=eps, weight_offset=offset, start=3)
    torch.cuda.synchronize()
    # eps reaches the kernel as an fp32 number
    eps = torch.tensor(eps, dtype=torch.float32).double().item()
    pos = (3 + torch.arange(q.shape[1])).expand(q.shape[0], -1)
    want, size = rotated(q.cpu(), pos, rope.frequencies, interleaved=interleaved,
                         weight=None if weight is None else weight.cpu(), offset=offset, eps=eps)
    assert bool(torch.isfinite(want).all())
    check_rotated(y, want, size, q.dtype, True)


@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("dim,rotary", WIDTHS)
@pytest.mark.parametrize("name", ("bf16", "f32"))
def test_weights_that_are_far_from_their_heads(ctx, name, dim, rotary, interleaved):
    """Large heads with small weights and small heads with large ones: outputs are ordinary numbers,
    the norm's factor times the weight is not."""
    announce(f"norms far {name} {dim} {rotary} {interleaved}")
    gen = torch.Generator(device="cuda").manual_seed(31)
    q = torch.randn(2, 3, 3, dim, device="cuda", generator=gen)
    w = torch.randn(dim, device="cuda", generator=gen)
    w = w.sign() * (0.5 + w.abs())
    for size, weight in ((2e17, 1e-25), (1e-16, 1e26)):
        for kind in (DTYPES[name], torch.float32):
            normed(ctx, (q * size).to(DTYPES[name]), (w * weight).to(kind), 0.0, rotary,
                   interleaved)


@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("dim,rotary", WIDTHS)
@pytest.mark.parametrize("name", sorted(DTYPES))
def test_heads_whose_squares_are_no_normal_numbers(ctx, name, dim, rotary, interleaved):
    """Down to the type's least number with an eps of nearly nothing, beside ordinary heads."""
    announce(f"norms small {name} {dim} {rotary} {interleaved}")
    dt = DTYPES[name]
    f = torch.finfo(dt)
    least = f.smallest_normal * f.eps
    gen = torch.Generator(device="cuda").manual_seed(32)
    q = torch.randn(1, 6, 5, dim, device="cuda", generator=gen)
    w = torch.randn(dim, device="cuda", generator=gen).to(dt)
    size = torch.tensor([1.0, 1e-15, 1e-19, 1e-21, 1e-30, 0.0]).cuda()
    if name == "f16":
        size = torch.tensor([1.0, 1e-3, 1e-4, 1e-5, 1e-6, 0.0]).cuda()
    q = (q * size[:, None, None]).to(dt)
    q[:, 5] = 3 * least
    q[:, :, 1] = 1.5          # neighbours in the same waves
    q[:, 2, 4] = 1e4
    # a head that rounds to zeros has no norm with an eps of 0
    q[..., 0] = torch.where(q[..., 0] == 0, 3 * least, q[..., 0].double()).to(dt)
    for eps in (0.0, 1e-42, 1e-38, 3e-31):
        for weight in (w, None):
            normed(ctx, q, weight, eps, rotary, interleaved)
