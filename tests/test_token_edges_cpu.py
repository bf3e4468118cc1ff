"""The token-level policy operators' autograd functions without a GPU, on meta
tensors: second derivatives, forward-mode tangents, inputs that are constants."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

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


@pytest.mark.parametrize("k", range(5))
@pytest.mark.parametrize("requires", [True, False])
def test_forward_mode_tangents_are_refused(k, requires):
    _, loss, shape = _losses()[k]
    x = torch.zeros(shape, requires_grad=requires, **META)
    with fwd.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|jvp"):
            loss(fwd.make_dual(x, torch.ones(shape, **META)))
    assert loss(x).shape == ()


def test_tangents_of_the_losses_other_inputs_are_refused():
    tok = torch.zeros(4, 3, dtype=torch.long, **META)
    tail = (0.2, 0.2, 0.0, 0.1, 3, 0)
    for k in range(3):
        with fwd.dual_level():
            rest = [torch.zeros(4, 3, **META) for _ in range(3)]  # old, advantages, reference
            rest[k] = fwd.make_dual(rest[k], torch.ones(4, 3, **META))
            old, adv, refl = rest
            with pytest.raises(NotImplementedError, match="forward-mode"):
                nat.ops.policy_loss(torch.zeros(4, 3, **META), old, adv, None, refl, *tail, 1.0, False)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                nat.ops.policy_loss_logits(torch.zeros(4, 3, 5, **META), tok, old, adv, None, refl, *tail[:5], 0.0,
                                           False, 1.0, 0, 1.0)
    with fwd.dual_level():
        refl = fwd.make_dual(torch.zeros(4, 3, **META), torch.ones(4, 3, **META))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            nat.ops.preference_loss(torch.zeros(4, 3, **META), None, refl, None, None, None, 0.1, 0.0, 0, False)


def test_the_losses_other_inputs_are_constants():
    """No gradient flows to them, required or not, as the docstrings say."""
    lp, old, adv, refl = (torch.zeros(4, 3, requires_grad=True, **META) for _ in range(4))
    loss = nat.ops.policy_loss(lp, old, adv, None, refl, 0.2, 0.2, 0.0, 0.1, 3, 0, 1.0, False)[0]
    got = torch.autograd.grad(loss, (lp, old, adv, refl), allow_unused=True)
    assert got[0] is not None and got[1:] == (None, None, None)
    loss = nat.ops.preference_loss(lp, None, refl, None, None, None, 0.1, 0.0, 0, False)[0]
    assert torch.autograd.grad(loss, (lp, refl), allow_unused=True)[1] is None


def test_wait_tries_are_the_threads_own():
    import threading
    assert nat.lib.rls_wait_tries(5) == -1
    seen = []
    th = threading.Thread(target=lambda: seen.append(nat.lib.rls_wait_tries(-1)))
    th.start()
    th.join()
    assert seen == [-1]
    assert nat.lib.rls_wait_tries(-7) == 5 and nat.lib.rls_wait_tries(-1) == -1
