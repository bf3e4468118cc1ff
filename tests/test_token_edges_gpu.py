"""The token-level policy operators at the edges of their definitions: steps at
a clip bound."""
import math

import pytest
import torch

import _token_ref as ref64

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")


def _near(bound, g, steps=12):
    """(lp, old) in fp32 with lp - old within `steps` ulps of lp of log(bound);
    small values among them, whose ulps are fine."""
    k = torch.arange(-steps, steps + 1)
    old = -2.0 ** (-6.0 * torch.rand(400, 1, generator=g))
    lp = (old.double() + math.log(bound)).float()
    return lp + k * 2.0 ** (torch.floor(torch.log2(lp.abs())) - 23), old.expand(-1, 2 * steps + 1).contiguous()


@pytest.mark.parametrize("low,high,dual", [(0.2, 0.28, 3.0), (0.2, None, None), (0.09, 0.16, 1.5), (0.33, 0.34, 1.1),
                                           (0.0, 0.05, None)])
def test_steps_at_a_clip_bound(low, high, dual):
    """Every step is on the side of the 64-bit definition with the caller's
    bounds, a few ulps from one too (fp32 inputs hold no step nearer than 1e-13
    of a bound other than the bound 1 itself, where both sides agree on 'not
    held').  A ratio is off by two ulps of expf and its difference's rounding, a
    term by one of a product more: 8 u."""
    _cuda()
    import rl_triton
    g = torch.Generator().manual_seed(5)
    top = low if high is None else high
    bounds = [1.0 - low, 1.0 + top] + ([] if dual is None else [dual])
    lp, old = (torch.cat(x) for x in zip(*(_near(b, g) for b in bounds)))
    lp, old = torch.cat([lp, lp]), torch.cat([old, old])
    adv = 0.5 + torch.rand(lp.shape, generator=g)
    adv[: len(adv) // 2] *= -1
    kw = dict(clip_low=low, clip_high=high, dual_clip=dual, reduction="sum")
    ld = lp.double().requires_grad_(True)
    want, stats = ref64.policy(ld, old.double(), adv.double(), **kw)
    (wg,) = torch.autograd.grad(want, ld)
    leaf = lp.cuda().requires_grad_(True)
    loss, st = rl_triton.compute_policy_loss(leaf, old.cuda(), adv.cuda(), return_stats=True, **kw)
    (grad,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(grad.cpu() == 0, wg == 0)
    torch.testing.assert_close(grad.cpu().double(), wg, rtol=8 * U, atol=0.0)
    assert abs(float(st["clip_fraction"]) - stats["clip_fraction"]) <= U
    size = float(((lp.double() - old.double()).exp() * adv.double()).abs().sum())
    assert abs(float(loss.detach()) - float(want.detach())) <= 8 * U * size
