"""The token-level policy operators at the edges of their definitions: steps at
a clip bound, tokens whose own logit is -inf, ratios past the range of fp32,
responses with a token of log-probability -inf.  Tolerances of log-probabilities,
entropies and gradients as in test_token_ops_gpu.py."""
import math

import pytest
import torch

import _token_ref as ref64
from test_token_ops_gpu import S, close, make, tol_ent, tol_grad, tol_lp

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")


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


@pytest.mark.parametrize("temp", [0.7, 0.8, 1.0, 1.1, 1.5])
@pytest.mark.parametrize("v", [18, 600, 1025, 5003, 131072, 300001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_whose_logit_is_minus_infinity(v, dtype, temp):
    """A masked action that was taken: log-probability -inf, the entropy and all
    gradients as ever, and a policy loss with ratio 0."""
    _cuda()
    import rl_triton
    x, tok, _, g = make(2, 3, v, dtype, seed=v, pad=5)
    tok[0, 1], tok[1, 0], tok[1, 2] = v - 1, v - 5, v - 3
    up, up_h = torch.randn(2, 3, generator=g), torch.randn(2, 3, generator=g)
    bf16 = dtype == torch.bfloat16
    xd = x.double().requires_grad_(True)
    lp64, h64 = ref64.logprobs(xd, tok, None, temp)
    (wg,) = torch.autograd.grad([lp64, h64], xd, [up.double(), up_h.double()])
    xc = x.cuda().requires_grad_(True)
    lp, h = rl_triton.compute_token_logprobs(xc, tok.cuda(), temperature=temp, return_entropy=True)
    (got,) = torch.autograd.grad([lp, h], xc, [up.cuda(), up_h.cuda()])
    assert int((lp == -INF).sum()) == 3
    close(lp, lp64, **tol_lp(v))
    close(h, h64, **tol_ent(v))
    close(got, wg, **tol_grad(v, 4.0 / temp, bf16))
    with torch.no_grad():
        close(rl_triton.compute_token_logprobs(xc, tok.cuda(), temperature=temp), lp64, **tol_lp(v))
    old = (torch.where(lp64 > -INF, lp64, torch.tensor(-4.0, dtype=torch.float64)) - 0.05).detach().float()
    adv = torch.tensor([[1.0, -0.5, 0.7], [1.5, -1.0, -0.3]])
    for ent in (0.0, 0.02):
        xd = x.double().requires_grad_(True)
        lp64, h64 = ref64.logprobs(xd, tok, None, temp)
        want, _ = ref64.policy(lp64, old.double(), adv.double(), entropy=h64, entropy_coef=ent)
        (wg,) = torch.autograd.grad(want, xd)
        assert torch.isfinite(want) and torch.isfinite(wg).all()
        loss, lp = rl_triton.compute_policy_loss_from_logits(xc, tok.cuda(), old.cuda(), adv.cuda(), entropy_coef=ent,
                                                             temperature=temp)
        (got,) = torch.autograd.grad(loss, xc)
        close(lp, lp64, **tol_lp(v))
        close(loss, want, rtol=2 * U, atol=12 * (S(v) + 8 * U + ent * tol_ent(v)["atol"]))
        close(got, wg, **tol_grad(v, 4 * float(wg.abs().max()), bf16))


@pytest.mark.parametrize("v", [0, 18, 2000])
def test_a_ratio_past_fp32_times_an_advantage_of_zero(v):
    """exp(lp - old) is finite in 64 bits and infinite in fp32: the term of a step
    with advantage 0 (all rewards of its group alike) is 0 all the same; v = 0: from
    log-probabilities."""
    _cuda()
    import rl_triton
    x, tok, _, _ = make(2, 3, max(v, 2), seed=3)
    lp64 = ref64.logprobs(x.double(), tok)[0]
    old = (lp64 - 0.1).float()
    old[0, 1] = old[1, 2] = -150.0
    adv = torch.tensor([[0.5, 0.0, 0.3], [0.2, -0.4, -0.0]])
    leaf = (x if v else lp64.float()).cuda().requires_grad_(True)
    exact = leaf.detach().cpu().double().requires_grad_(True)
    args = [t.cuda() for t in ((tok, old, adv) if v else (old, adv))]
    fn = rl_triton.compute_policy_loss_from_logits if v else rl_triton.compute_policy_loss
    for dual in (None, 2.0):
        out = fn(leaf, *args, dual_clip=dual)
        loss = out[0] if v else out
        lpd = ref64.logprobs(exact, tok)[0] if v else exact
        want, _ = ref64.policy(lpd, old.double(), adv.double(), dual_clip=dual)
        (wg,) = torch.autograd.grad(want, exact)
        (got,) = torch.autograd.grad(loss, leaf)
        assert torch.isfinite(want) and torch.isfinite(wg).all()
        close(loss, want, rtol=2 * U, atol=12 * (S(max(v, 2)) + 8 * U))
        close(got, wg, **tol_grad(max(v, 2), 4 * float(wg.abs().max()), False))


@pytest.mark.parametrize("loss,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0)])
@pytest.mark.parametrize("normalized", [False, True])
def test_preference_with_a_rejected_token_of_probability_zero(loss, smoothing, normalized):
    """The pair's x is +inf: -log sig(x) and the hinge are 0, and so is its
    gradient; with smoothing -e log sig(-x) is +inf."""
    _cuda()
    import rl_triton
    g = torch.Generator().manual_seed(7)
    lp, refl = -3 * torch.rand(6, 9, generator=g), -3 * torch.rand(6, 9, generator=g)
    lp[4, 3] = -INF  # the second pair's rejected response
    leaf = lp.cuda().requires_grad_(True)
    kw = dict(beta=0.3, loss=loss, label_smoothing=smoothing, length_normalized=normalized)
    got, good, bad = rl_triton.compute_preference_loss(leaf, refl.cuda(), **kw)
    (grad,) = torch.autograd.grad(got, leaf)
    assert bad[1] == -INF and torch.isfinite(bad[[0, 2]]).all() and torch.isfinite(good).all()
    if smoothing:
        assert got == INF
        return
    keep = [0, 2]  # the other pairs, their mean over all three
    ld = lp.double().requires_grad_(True)
    a, b = ld[:3][keep], ld[3:][keep]
    want, _, _ = ref64.preference(a, b, (refl[:3][keep].double(), refl[3:][keep].double()), (None, None), 0.3, loss,
                                  smoothing, normalized)
    want = want * 2 / 3
    (wg,) = torch.autograd.grad(want, ld)
    close(got, want, rtol=128 * U, atol=1e-7)
    close(grad, wg, rtol=128 * U, atol=1e-9)
    assert (grad[[1, 4]] == 0).all()


def test_gradients_with_create_graph():
    """The same values, and an error once one of them is differentiated."""
    _cuda()
    import rl_triton as rl
    x, tok, _, g = make(4, 6, 2000, seed=2)
    old, adv = -torch.rand(4, 6, generator=g).cuda(), torch.randn(4, generator=g).cuda()
    tok = tok.cuda()
    logits, lp = x.cuda(), -torch.rand(4, 6, generator=g).cuda()
    for leaf, f in [(lp, lambda z: rl.compute_policy_loss(z, old, adv)),
                    (logits, lambda z: rl.compute_policy_loss_from_logits(z, tok, old, adv)[0]),
                    (lp, lambda z: rl.compute_preference_loss(z)[0]),
                    (lp, lambda z: rl.compute_preference_loss((z[:2], z[2:]))[0])]:
        z = leaf.clone().requires_grad_(True)
        (want,) = torch.autograd.grad(f(z), z)
        value = f(z)
        (got,) = torch.autograd.grad(value, z, create_graph=True)
        assert torch.equal(got, want) and got.requires_grad and not want.requires_grad
        with pytest.raises(RuntimeError, match="not implemented"):
            (value + got.square().sum()).backward()


def test_operators_check_their_tensors():
    """Called without the functions in front: sizes and types that the kernels
    would read or write past are refused before anything is launched."""
    _cuda()
    ops = torch.ops.rl_triton
    C = dict(device="cuda")
    x, tok, lp = torch.zeros(4, 3, 5, **C), torch.zeros(4, 3, dtype=torch.long, **C), torch.zeros(4, 3, **C)
    long = torch.zeros(4, 3, 2000, **C)
    small, row, one = lp[:2], lp[:, 0], torch.ones((), **C)
    none = torch.empty(0, **C)
    order, norm = torch.empty(0, dtype=torch.int32, **C), torch.zeros(5, **C)

    def refuses(match, op, *args):
        with pytest.raises(RuntimeError, match=match):
            op(*args)

    # logits
    for f in (lambda *a: ops.token_logprobs(*a, 1.0, False), lambda *a: ops._token_logprobs(*a, 1.0, True, True),
              lambda z, t, m: ops.policy_loss_logits(z, t, lp, lp, m, None, 0.2, 0.2, 0.0, 0.0, 3, 0.0, False, 1.0, 0,
                                                     1.0),
              lambda z, t, m: ops._token_logprobs_backward(z, t, m, order, none, lp, None, 1.0)):
        for grad in (False, True):
            z = x.clone().requires_grad_(grad)
            refuses("float32 or bfloat16", f, x.half().requires_grad_(grad), tok, None)
            refuses("float32 or bfloat16", f, x.double().requires_grad_(grad), tok, None)
            refuses("tokens: expected shape", f, z, tok[:2], None)
            refuses("tokens: expected integers", f, z, lp, None)
            refuses("mask: expected shape", f, z, tok, small)
            refuses("mask: expected bool", f, z, tok, lp.to(torch.complex64))
            refuses("num_envs, seq_len, vocab", f, x[0].clone().requires_grad_(grad), tok[0], None)
    refuses("num_envs, seq_len, vocab", ops._grad_buffer, lp)
    back = ops._token_logprobs_backward
    refuses("row_stats", back, long, tok, None, order, none, lp, None, 1.0)
    refuses("row_stats", back, long, tok, None, order, torch.zeros(4, 3, 7, **C), lp, None, 1.0)
    refuses("row_stats", back, long, tok, None, order, torch.zeros(4, 3, 8, dtype=torch.float64, **C), lp, None, 1.0)
    refuses("order: expected shape", back, x, tok, lp, torch.zeros(12, dtype=torch.int32, **C), none, lp, None, 1.0)
    refuses("g_logprobs", back, x, tok, None, order, none, small, None, 1.0)
    refuses("g_entropy", back, x, tok, None, order, none, lp, row, 1.0)

    # policy losses
    tail = (0.2, 0.2, 0.0, 0.0, 3, 0)
    for f in (lambda o, a, m, r: ops.policy_loss(lp, o, a, m, r, *tail, 1.0, False),
              lambda o, a, m, r: ops.policy_loss(lp.clone().requires_grad_(True), o, a, m, r, *tail, 1.0, False),
              lambda o, a, m, r: ops.policy_loss_logits(x, tok, o, a, m, r, *tail[:5], 0.0, False, 1.0, 0, 1.0),
              lambda o, a, m, r: ops._policy_loss_backward_(lp.clone(), lp, o, a, m, r, norm, one, *tail, 1.0, True),
              lambda o, a, m, r: ops._policy_loss_logits_backward_(x.clone(), x, tok, o, a, m, r, norm, order, none, one,
                                                                   *tail[:5], 0.0, 1.0, 0, 1.0, True)):
        refuses("old_logprobs: expected shape", f, small, lp, None, None)
        refuses("old_logprobs: expected floating", f, tok, lp, None, None)
        refuses("advantages: expected shape", f, lp, small, None, None)
        refuses("advantages: expected shape", f, lp, row[:2], None, None)
        refuses("advantages: expected shape", f, lp, one, None, None)
        refuses("ref_logprobs: expected shape", f, lp, row, None, row)
        refuses("mask: expected shape", f, lp, row, row, None)
    refuses("logprobs: expected shape", ops.policy_loss, row, row, row, None, None, *tail, 1.0, False)
    loss_back = ops._policy_loss_backward_
    refuses("grad: expected", loss_back, small, lp, lp, lp, None, None, norm, one, *tail, 1.0, True)
    refuses("grad: expected", loss_back, lp.bfloat16(), lp, lp, lp, None, None, norm, one, *tail, 1.0, True)
    refuses("grad_loss", loss_back, lp, lp, lp, lp, None, None, norm, lp, *tail, 1.0, True)
    refuses("norm: expected shape", loss_back, lp, lp, lp, lp, lp, None, norm[:4], one, *tail, 1.0, True)
    back = lambda g, nrm, up=one: ops._policy_loss_logits_backward_(  # noqa: E731
        g, x, tok, lp, lp, lp, None, nrm, order, none, up, *tail[:5], 0.0, 1.0, 0, 1.0, True)
    refuses("grad: expected shape", back, x[:2], norm)
    refuses("grad: expected", back, x.bfloat16(), norm)
    refuses("contiguous", back, torch.zeros(4, 5, 3, **C).transpose(1, 2), norm)
    refuses("norm: expected shape", back, x.clone(), none)
    refuses("grad_loss", back, x.clone(), norm, lp)

    # preference loss
    for grad in (False, True):
        z = lp.clone().requires_grad_(grad)
        f = lambda *a: ops.preference_loss(*a, 0.1, 0.0, 0, False)  # noqa: E731
        refuses("2 \\* pairs", f, z[:3], None, None, None, None, None)
        refuses("chosen: expected shape", f, z[0], None, None, None, None, None)
        refuses("go with it", f, z, None, None, lp, None, None)
        refuses("as many responses", f, z, z[:2], None, None, None, None)
        refuses("alike", f, z, z, lp, None, None, None)
        refuses("alike", f, z, z, lp, row, None, None)
        refuses("ref_chosen: expected shape", f, z, None, small, None, None, None)
        refuses("ref_chosen: expected shape", f, z, None, row[:2], None, None, None)
        refuses("chosen_mask: expected shape", f, z, None, None, None, small, None)
        refuses("ref_rejected: expected shape", f, z, z, row, row[:3], None, None)
        refuses("rejected_mask: expected shape", f, z, z, None, None, None, row)
    f = ops._preference_loss_backward
    coef = torch.ones(2, 2, **C)
    refuses("coef: expected shape", f, torch.ones(3, 2, **C), one, None, None, 3, 3, False)
    refuses("coef: expected", f, coef.double(), one, None, None, 3, 3, False)
    refuses("coef: expected", f, coef, one, None, None, -1, 3, False)
    refuses("grad_loss", f, coef, coef, None, None, 3, 3, False)
    refuses("chosen_mask: expected shape", f, coef, one, lp, None, 3, 3, False)
    refuses("chosen_mask: expected shape", f, coef, one, small, None, 3, 0, True)
    refuses("rejected_mask: expected shape", f, coef, one, None, lp, 3, 3, False)
    torch.cuda.synchronize()


@pytest.mark.parametrize("v,dtype,n,t", [(5000, torch.float32, 2, 4), (131072, torch.bfloat16, 2, 4),
                                         (131072, torch.float32, 3, 40), (60000, torch.bfloat16, 30, 20)])
def test_a_wait_that_runs_out(v, dtype, n, t, monkeypatch):
    """Without a try the CTAs of a row do not get one another's sums: the kernel
    ends, the rows that count are NaN (nothing wrong passes for a result), the
    workspace says so, and the next call is as ever."""
    _cuda()
    import rl_triton
    from rl_triton import _native as nat
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    x, tok, mask, g = make(n, t, v, dtype, seed=1)
    old, adv = -3 * torch.rand(n, t, generator=g), torch.randn(n, t, generator=g)
    x, tok, mask, old, adv = (a.cuda() for a in (x, tok, mask, old, adv))
    x.requires_grad_(True)

    def call():
        loss, lp = rl_triton.compute_policy_loss_from_logits(x, tok, old, adv, mask)
        return loss.detach(), lp, torch.autograd.grad(loss, x)[0]

    want = call()
    assert nat.workspace_error() == 0 and torch.isfinite(want[0])
    assert nat.lib.rls_wait_tries(0) == -1
    try:
        loss, lp, grad = call()
        torch.cuda.synchronize()
        assert nat.workspace_error() == 8 and nat.workspace_error() == 0
        assert torch.isnan(loss) and torch.isnan(lp[mask]).all() and torch.isnan(grad[mask]).all()
        assert (lp[~mask] == 0).all() and (grad[~mask] == 0).all()
        monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "1")
        with pytest.raises(RuntimeError, match="wait ran out"):
            call()
    finally:
        assert nat.lib.rls_wait_tries(-1) == 0
    for a, b in zip(call(), want):
        assert torch.equal(a, b)


def test_an_assumed_device_is_the_token_operators_alone():
    """The other entry points still look where their arrays are (pinned host
    memory here, which a kernel could reach)."""
    _cuda()
    from rl_triton import _native as nat
    r, out = torch.ones(2, 8).pin_memory(), torch.zeros(2, 8).pin_memory()
    ws, wsb = nat.workspace(torch.device("cuda", 0), nat.stream_handle(torch.device("cuda", 0)), 1 << 20)

    def call():
        return nat.lib.rls_discounted_returns(r.data_ptr(), r.data_ptr(), None, None, 0, out.data_ptr(), 2, 8, 0.99, 0, None,
                                              ws, wsb, nat.stream_handle(torch.device("cuda", 0)))

    assert call() == nat.RLS_ENOTDEVICE
    assert nat.lib.rls_assume_device(0) == -1
    try:
        assert call() == nat.RLS_ENOTDEVICE
    finally:
        assert nat.lib.rls_assume_device(-1) == 0
    torch.cuda.synchronize()
    assert (out == 0).all()
