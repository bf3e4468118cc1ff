"""The token-level policy operators' autograd functions without a GPU, on meta
tensors: second derivatives."""
import pytest
import torch

from rl_triton import _native as nat

META = dict(device="meta")


def _losses():
    """(name, a function of one differentiable tensor to a scalar, its shape)."""
    tok = torch.zeros(4, 3, dtype=torch.long, **META)
    lp, adv = torch.zeros(4, 3, **META), torch.zeros(4, **META)
    return [
        ("token_logprobs", lambda x: nat.ops.token_logprobs(x, tok, None, 1.0, True)[0].sum(), (4, 3, 5)),
        ("policy_loss", lambda x: nat.ops.policy_loss(x, lp, adv, None, None, 0.2, 0.2, 0.0, 0.0, 3, 0, 1.0, False)[0],
         (4, 3)),
        ("policy_loss_logits", lambda x: nat.ops.policy_loss_logits(x, tok, lp, adv, None, None, 0.2, 0.2, 0.0, 0.0, 3,
                                                                    0.0, False, 1.0, 0, 1.0)[0], (4, 3, 5)),
        ("preference_loss", lambda x: nat.ops.preference_loss(x, None, None, None, None, None, 0.1, 0.0, 0, False)[0],
         (4, 3)),
        ("preference_loss of pairs", lambda x: nat.ops.preference_loss(x[:2], x[2:], None, None, None, None, 0.1, 0.0, 0,
                                                                       False)[0], (4, 3)),
    ]


@pytest.mark.parametrize("k", range(5))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("leaf", [True, False])
def test_a_second_derivative_raises(k, dtype, leaf):
    """With create_graph the gradient is there, and nothing that is made of it
    can lose its own gradient."""
    _, loss, shape = _losses()[k]
    x = torch.zeros(shape, dtype=dtype, requires_grad=True, **META)
    value = loss(x if leaf else 2.0 * x)
    (g,) = torch.autograd.grad(value, x, create_graph=True)
    assert g.shape == x.shape and g.dtype == dtype and g.requires_grad
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(g.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        (value + g.float().square().sum()).backward()
    (g,) = torch.autograd.grad(loss(x if leaf else 2.0 * x), x)  # without it, as ever
    assert not g.requires_grad


def test_a_second_derivative_by_the_incoming_gradient_raises():
    _, loss, shape = _losses()[1]
    x, up = torch.zeros(shape, requires_grad=True, **META), torch.ones((), requires_grad=True, **META)
    (g,) = torch.autograd.grad(loss(x), x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        torch.autograd.grad(g.sum(), up)
