"""The token-level policy operators against their plain 64-bit forms.

Tolerances.  With u = 2^-24 (half an ulp of fp32), a row of V logits is summed
in chains of at most V / 128 + 32 additions, each ex2 is good to 2^-22 and the
rounded factor log2(e) / temperature moves a logit by at most u |z|:
    S(V) = (V / 128 + 32) u + 4 u + max|z| u          (relative, of a sum)
a log-probability is off by S plus its own rounding; an entropy, a weighted sum
of logarithms of up to L = log V + max|z|, by 4 L S; a gradient, a product of p,
of the incoming gradients and of a difference of logarithms, by 4 L S of the
largest of its parts; the bf16 gradient by half an ulp (2^-9) more.  The policy
loss's terms are good to 8 u of (r |A| + |x| + 1), and are added in fp64."""
import math

import numpy as np
import pytest
import torch

import _token_ref as ref64

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")


def _cuda():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")


def S(v, z=40.0):
    return (v / 128 + 36 + z) * U


def tol_lp(v, z=40.0):
    return dict(rtol=2 * U, atol=S(v, z))


def tol_ent(v, z=40.0):
    return dict(rtol=2 * U, atol=4 * (math.log(v) + z) * S(v, z))


def tol_grad(v, top, bf16, z=40.0):
    return dict(rtol=(2.0 ** -8 if bf16 else 2 * U), atol=4 * (math.log(v) + z) * S(v, z) * top + 1e-37)


def close(got, want, rtol, atol):
    torch.testing.assert_close(got.detach().cpu().double(), want.detach().double(), rtol=rtol, atol=atol,
                               equal_nan=True)


def make(n, t, v, dtype=torch.float32, seed=0, scale=2.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = (scale * torch.randn(n, t, v, generator=g)).to(dtype)
    if pad:
        x[..., v - pad:] = -INF
    tok = torch.randint(0, v - pad, (n, t), generator=g)
    x.scatter_add_(2, tok[..., None], (math.log(v) * torch.rand(n, t, 1, generator=g)).to(dtype))
    mask = torch.rand(n, t, generator=g) < 0.7
    if n > 1:
        mask[1] = False  # a row of the batch with nothing to count
    return x, tok, mask, g


SIZES = [(2, 3, 1), (1, 1, 2), (3, 5, 4), (2, 7, 5), (4, 9, 18), (2, 3, 33), (3, 4, 64), (2, 3, 127), (2, 5, 200),
         (2, 3, 511), (2, 3, 1000), (2, 3, 1024), (2, 3, 1025), (3, 5, 2049), (2, 4, 5003), (2, 3, 8192),
         (2, 3, 32771), (1, 1, 50021), (2, 2, 131072), (1, 3, 200003)]


@pytest.mark.parametrize("n,t,v", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logprobs_entropy_and_gradient(n, t, v, dtype):
    _cuda()
    import rl_triton
    x, tok, mask, g = make(n, t, v, dtype, seed=v, pad=min(3, v // 4))
    g_lp, g_h = torch.randn(n, t, generator=g), torch.randn(n, t, generator=g)
    xd = x.double().requires_grad_(True)
    lp64, h64 = ref64.logprobs(xd, tok, mask, 0.7)
    (want,) = torch.autograd.grad([lp64, h64], xd, [g_lp.double(), g_h.double()])
    xc = x.cuda().requires_grad_(True)
    lp, h = rl_triton.compute_token_logprobs(xc, tok.cuda(), mask.cuda(), temperature=0.7, return_entropy=True)
    assert lp.dtype == h.dtype == torch.float32 and lp.shape == h.shape == (n, t)
    (got,) = torch.autograd.grad([lp, h], xc, [g_lp.cuda(), g_h.cuda()])
    assert got.dtype == dtype
    close(lp, lp64, **tol_lp(v))
    close(h, h64, **tol_ent(v))
    close(got, want, **tol_grad(v, 4.0 / 0.7, dtype == torch.bfloat16))
    assert (got[~mask.cuda()] == 0).all()
    # without the entropy, by either gradient alone, and without a gradient
    only = rl_triton.compute_token_logprobs(xc, tok.cuda(), mask.cuda(), temperature=0.7)
    (got,) = torch.autograd.grad(only, xc, g_lp.cuda())
    (want,) = torch.autograd.grad(ref64.logprobs(xd, tok, mask, 0.7)[0], xd, g_lp.double())
    close(only, lp64, **tol_lp(v))
    close(got, want, **tol_grad(v, 4.0 / 0.7, dtype == torch.bfloat16))
    with torch.no_grad():
        close(rl_triton.compute_token_logprobs(xc, tok.cuda(), mask.cuda(), temperature=0.7), lp64, **tol_lp(v))


@pytest.mark.parametrize("v", [7, 300, 1500, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_entropy_gradient_alone(v, dtype):
    _cuda()
    import rl_triton
    x, tok, _, g = make(2, 3, v, dtype, seed=5)
    up = torch.randn(2, 3, generator=g)
    xd = x.double().requires_grad_(True)
    (want,) = torch.autograd.grad(ref64.logprobs(xd, tok)[1], xd, up.double())
    xc = x.cuda().requires_grad_(True)
    _, h = rl_triton.compute_token_logprobs(xc, tok.cuda(), return_entropy=True)
    (got,) = torch.autograd.grad(h, xc, up.cuda())
    close(got, want, **tol_grad(v, 4.0, dtype == torch.bfloat16))


@pytest.mark.parametrize("v", [19, 700, 5001, 70003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_logits(v, dtype):
    """Slices of the steps, a vocabulary cut from a padded one, steps outside
    envs, an expanded batch, a transposed vocabulary."""
    _cuda()
    import rl_triton
    x, _, _, g = make(3, 6, v + 5, dtype, seed=v)
    base = x.cuda()
    views = [base[:, :-1, :v], base[:, 1:, 3:v + 3], base.transpose(0, 1)[:, :, 1:], base[:1, :, :v].expand(3, 6, v),
             base[:, ::2, :v], base.transpose(1, 2).contiguous().transpose(1, 2), base[:, 2:3], base[1:2, :, 5:]]
    for view in views:
        n, t, w = view.shape
        tok = torch.randint(0, w, (n, t), generator=g)
        up = torch.randn(n, t, generator=g)
        xd = view.detach().cpu().double().requires_grad_(True)
        lp64, _ = ref64.logprobs(xd, tok)
        (want,) = torch.autograd.grad(lp64, xd, up.double())
        leaf = view.detach().requires_grad_(True)
        lp = rl_triton.compute_token_logprobs(leaf, tok.cuda())
        (got,) = torch.autograd.grad(lp, leaf, up.cuda())
        close(lp, lp64, **tol_lp(w))
        close(got, want, **tol_grad(w, 4.0, dtype == torch.bfloat16))
        # the loss from the same view
        old, adv = lp64.detach().float(), up
        loss, _ = rl_triton.compute_policy_loss_from_logits(leaf, tok.cuda(), old.cuda(), adv.cuda())
        (got,) = torch.autograd.grad(loss, leaf)
        (want,) = torch.autograd.grad(ref64.policy(ref64.logprobs(xd, tok)[0], old.double(), adv.double())[0], xd)
        close(got, want, **tol_grad(w, 4.0 / (n * t), dtype == torch.bfloat16))


@pytest.mark.parametrize("v", [6, 100, 3001, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_special_logits(v, dtype):
    _cuda()
    import rl_triton
    low = torch.finfo(dtype).min
    x = torch.randn(1, 8, v, generator=torch.Generator().manual_seed(v)).to(dtype)
    x[0, 0] = low                       # all at the type's lowest value: uniform
    x[0, 1, 1:] = low                   # one token left
    x[0, 2, 1:] = -INF
    x[0, 3] = -INF                      # nothing left: NaN, as the formula gives
    x[0, 4, 2] = float("nan")
    x[0, 5, 2] = INF
    x[0, 6] = 1e30                      # a large constant: uniform
    x[0, 7, : v // 2] = -3e4
    tok = torch.zeros(1, 8, dtype=torch.long)
    xc = x.cuda().requires_grad_(True)
    lp, h = rl_triton.compute_token_logprobs(xc, tok.cuda(), return_entropy=True)
    (g,) = torch.autograd.grad([lp, h], xc, [torch.ones_like(lp), torch.ones_like(h)])
    lp, h, g = lp[0].cpu().double(), h[0].cpu().double(), g[0].cpu().double()
    uniform = -math.log(v)
    for k in (0, 6):
        assert abs(lp[k] - uniform) < 1e-5 and abs(h[k] + uniform) < 1e-4
        want = torch.full((v,), -1.0 / v, dtype=torch.float64)
        want[0] += 1.0
        close(g[k], want, rtol=2 ** -7, atol=1e-5)
    for k in (1, 2):
        assert lp[k] == 0 and h[k] == 0 and (g[k] == 0).all()
    for k in (3, 4, 5):
        assert math.isnan(lp[k]) and math.isnan(h[k]) and torch.isnan(g[k]).all()
    want, _ = ref64.logprobs(x[:, 7:].double(), tok[:, 7:])
    close(lp[7:], want[0], **tol_lp(v, 30000.0 if v < 4 else 40.0))
    # the same rows behind a mask: nothing of them is seen
    mask = torch.ones(1, 8, dtype=torch.bool)
    mask[0, 3:6] = False
    lp, h = rl_triton.compute_token_logprobs(xc, tok.cuda(), mask.cuda(), return_entropy=True)
    (g,) = torch.autograd.grad([lp, h], xc, [torch.ones_like(lp), torch.ones_like(h)])
    assert torch.isfinite(lp).all() and torch.isfinite(g).all()
    assert (lp[0, 3:6] == 0).all() and (h[0, 3:6] == 0).all() and (g[0, 3:6] == 0).all()


@pytest.mark.parametrize("v", [5, 2000])
def test_tokens_outside_the_vocabulary(v, monkeypatch):
    _cuda()
    import rl_triton
    x = torch.randn(1, 4, v).cuda().requires_grad_(True)
    tok = torch.tensor([[0, -100, v, 1]]).cuda()
    with pytest.raises(AssertionError, match="outside the vocabulary"):
        rl_triton.compute_token_logprobs(x, tok)
    masked = torch.tensor([[1, 0, 0, 1]]).cuda()
    lp = rl_triton.compute_token_logprobs(x, tok, masked)  # not used there
    assert torch.isfinite(lp).all()
    (g,) = torch.autograd.grad(lp.sum(), x)
    assert torch.isfinite(g).all() and (g[0, 1:3] == 0).all()
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    lp = rl_triton.compute_token_logprobs(x, tok)
    assert torch.isnan(lp[0, 1:3]).all() and torch.isfinite(lp[0, [0, 3]]).all()
    loss, lp = rl_triton.compute_policy_loss_from_logits(x, tok, torch.zeros(1, 4).cuda(), torch.ones(1, 4).cuda())
    (g,) = torch.autograd.grad(loss, x)
    assert torch.isnan(loss) and torch.isnan(g[0, 1:3]).all() and torch.isfinite(g[0, [0, 3]]).all()


@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8, torch.int32, torch.int64, torch.float32, torch.bfloat16,
                                   torch.float16])
def test_mask_types_agree(dtype):
    _cuda()
    import rl_triton
    x, tok, mask, g = make(4, 6, 37, seed=3)
    old, adv = -torch.rand(4, 6, generator=g), torch.randn(4, 6, generator=g)
    a = rl_triton.compute_token_logprobs(x.cuda(), tok.cuda(), mask.cuda())
    b = rl_triton.compute_token_logprobs(x.cuda(), tok.int().cuda(), mask.to(dtype).cuda())
    assert torch.equal(a, b)
    l1 = rl_triton.compute_policy_loss(a, old.cuda(), adv.cuda(), mask.cuda(), reduction="sequence")
    l2 = rl_triton.compute_policy_loss(a, old.cuda(), adv.cuda(), mask.to(dtype).cuda(), reduction="sequence")
    assert torch.equal(l1, l2)
    p1 = rl_triton.compute_preference_loss(a, None, mask.cuda())[0]
    p2 = rl_triton.compute_preference_loss(a, None, mask.to(dtype).cuda())[0]
    p3 = rl_triton.compute_preference_loss((a[:2], a[2:]), None, (mask[:2].cuda(), mask[2:].to(dtype).cuda()))[0]
    assert torch.equal(p1, p2) and torch.equal(p1, p3)


def _policy_inputs(n, t, seed, per_env):
    g = torch.Generator().manual_seed(seed)
    lp = -3.0 * torch.rand(n, t, generator=g) - 0.01
    old = lp + 0.3 * torch.randn(n, t, generator=g)
    ref = lp + 0.3 * torch.randn(n, t, generator=g)
    adv = torch.randn((n,) if per_env else (n, t), generator=g)
    mask = torch.rand(n, t, generator=g) < 0.6
    if n > 1:
        mask[0] = False
    return lp, old, ref, adv, mask


POLICY_SIZES = [(1, 1), (2, 1), (1, 7), (3, 5), (5, 128), (9, 131), (1, 70001), (2000, 17), (700, 513)]


@pytest.mark.parametrize("n,t", POLICY_SIZES)
@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
@pytest.mark.parametrize("masked", [False, True])
def test_policy_loss(n, t, reduction, masked):
    _cuda()
    import rl_triton
    kls, k = ["k1", "k2", "k3"], n + t
    per_env, dual = k % 2 == 0, 1.5 if k % 3 else None
    lp, old, refl, adv, mask = _policy_inputs(n, t, k, per_env)
    m = mask if masked else None
    kw = dict(clip_low=0.2, clip_high=0.3, dual_clip=dual, kl_coef=0.1, kl=kls[k % 3], reduction=reduction)
    if masked:  # what stands at mask 0 is not used
        for x in (old, refl) + (() if per_env else (adv,)):
            x[~mask] = float("nan")
    lpd = lp.double().requires_grad_(True)
    want, stats = ref64.policy(lpd, old.double(), adv.double(), m, refl.double(), **kw)
    (wg,) = torch.autograd.grad(want, lpd)
    lpc = lp.cuda().requires_grad_(True)
    mc = None if m is None else m.cuda()
    loss, got = rl_triton.compute_policy_loss(lpc, old.cuda(), adv.cuda(), mc, refl.cuda(), return_stats=True, **kw)
    # terms are at most about 6 in size, each good to 8 u of (r |A| + |x| + 1)
    each = 8 * U * 12
    terms = (int(mask.sum()) if masked else n * t) if reduction == "sum" else 1
    close(loss, want, rtol=2 * U, atol=each * max(terms, 1))
    (g,) = torch.autograd.grad(loss, lpc)
    close(g, wg, rtol=8 * U, atol=each * (1.0 if reduction == "sum" else float(wg.abs().max()) + 1e-12))
    for key, val in stats.items():
        np.testing.assert_allclose(float(got[key]), val, rtol=4 * U, atol=each, err_msg=key)


def test_policy_loss_nothing_counts_and_empty():
    _cuda()
    import rl_triton
    for reduction in ("token", "sequence", "sum"):
        lp = torch.randn(3, 5).cuda().requires_grad_(True)
        loss, st = rl_triton.compute_policy_loss(lp, lp.detach(), lp.detach(), torch.zeros(3, 5).cuda(),
                                                 reduction=reduction, return_stats=True)
        (g,) = torch.autograd.grad(loss, lp)
        assert float(loss) == 0 and (g == 0).all() and float(st["num_steps"]) == 0
        x = torch.randn(3, 5, 2000).cuda().requires_grad_(True)
        loss, _ = rl_triton.compute_policy_loss_from_logits(x, torch.zeros(3, 5, dtype=torch.long).cuda(),
                                                            lp.detach(), lp.detach(), torch.zeros(3, 5).cuda(),
                                                            reduction=reduction, entropy_coef=0.1)
        (g,) = torch.autograd.grad(loss, x)
        assert float(loss) == 0 and (g == 0).all()
    for shape in ((0, 5), (3, 0)):
        e = torch.zeros(shape).cuda().requires_grad_(True)
        loss = rl_triton.compute_policy_loss(e, e.detach(), e.detach(), torch.zeros(shape).cuda())
        (g,) = torch.autograd.grad(loss, e)
        assert float(loss) == 0 and g.shape == shape
        x = torch.zeros(*shape, 7).cuda().requires_grad_(True)
        tok = torch.zeros(shape, dtype=torch.long).cuda()
        assert rl_triton.compute_token_logprobs(x, tok).shape == shape
        loss, lp = rl_triton.compute_policy_loss_from_logits(x, tok, e.detach(), e.detach())
        (g,) = torch.autograd.grad(loss, x)
        assert float(loss) == 0 and lp.shape == shape and g.shape == x.shape
    z = torch.zeros(0, 4).cuda().requires_grad_(True)
    loss, a, b = rl_triton.compute_preference_loss(z)
    (g,) = torch.autograd.grad(loss, z)
    assert float(loss) == 0 and a.shape == b.shape == (0,) and g.shape == (0, 4)
    z = torch.zeros(4, 0).cuda().requires_grad_(True)
    loss, a, b = rl_triton.compute_preference_loss(z)
    (g,) = torch.autograd.grad(loss, z)
    np.testing.assert_allclose(float(loss), math.log(2.0), rtol=4 * U)
    assert (a == 0).all() and g.shape == (4, 0)


@pytest.mark.parametrize("v", [2, 18, 600, 4099, 50021, 131072])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ent", [0.0, 0.02])
def test_policy_loss_from_logits(v, dtype, ent):
    _cuda()
    import rl_triton
    n, t = 3, 4
    x, tok, mask, g = make(n, t, v, dtype, seed=v + 1, pad=1 if v > 2 else 0)
    xd = x.double().requires_grad_(True)
    lp64, h64 = ref64.logprobs(xd, tok, mask, 1.3)
    old = (lp64 + 0.3 * torch.randn(n, t, generator=g)).detach().float()
    refl = (lp64 + 0.3 * torch.randn(n, t, generator=g)).detach().float()
    adv = torch.randn(n, t, generator=g)
    for reduction, m in (("token", mask), ("sequence", mask), ("sum", None)):
        lp64, h64 = ref64.logprobs(xd, tok, m, 1.3)
        kw = dict(kl_coef=0.1, dual_clip=3.0, reduction=reduction)
        want, stats = ref64.policy(lp64, old.double(), adv.double(), m, refl.double(), entropy=h64, entropy_coef=ent,
                                   **kw)
        (wg,) = torch.autograd.grad(want, xd)
        xc = x.cuda().requires_grad_(True)
        loss, lp, st = rl_triton.compute_policy_loss_from_logits(
            xc, tok.cuda(), old.cuda(), adv.cuda(), None if m is None else m.cuda(), refl.cuda(), entropy_coef=ent,
            temperature=1.3, return_stats=True, **kw)
        assert not lp.requires_grad
        close(lp, lp64, **tol_lp(v))
        many = n * t if reduction == "sum" else 1
        top = float(wg.abs().max()) + 1e-6
        close(loss, want, rtol=2 * U, atol=many * 12 * (S(v) + 8 * U + ent * tol_ent(v)["atol"]))
        (got,) = torch.autograd.grad(loss, xc)
        close(got, wg, **tol_grad(v, 4 * top, dtype == torch.bfloat16))
        np.testing.assert_allclose(float(st["entropy"]), stats["entropy"], rtol=4 * U, atol=tol_ent(v)["atol"])
        with torch.no_grad():
            again, _ = rl_triton.compute_policy_loss_from_logits(
                xc, tok.cuda(), old.cuda(), adv.cuda(), None if m is None else m.cuda(), refl.cuda(),
                entropy_coef=ent, temperature=1.3, **kw)
        close(again, loss.detach().cpu(), rtol=4 * U, atol=many * 12 * S(v))


@pytest.mark.parametrize("v", [18, 5000])
def test_incoming_gradients(v):
    """The gradient follows the incoming one: the one it was made for, another,
    zero, and a second pass over a retained graph; the first one stays as it was."""
    _cuda()
    import rl_triton
    x, tok, mask, g = make(3, 5, v, seed=1)
    lp, old, refl, adv, _ = _policy_inputs(3, 5, 2, False)
    args = [a.cuda() for a in (tok, old, adv, mask, refl)]
    for scale in (1.0, 0.25):
        xc = x.cuda().requires_grad_(True)
        loss, _ = rl_triton.compute_policy_loss_from_logits(xc, *args, kl_coef=0.1, entropy_coef=0.01,
                                                            grad_scale=scale)
        one = torch.autograd.grad(loss, xc, retain_graph=True)[0]
        kept = one.clone()
        third = torch.autograd.grad(3.0 * loss, xc, retain_graph=True)[0]
        zero = torch.autograd.grad(0.0 * loss, xc, retain_graph=True)[0]
        (0.25 * loss).backward()
        assert torch.equal(one, kept)
        torch.testing.assert_close(third, 3 * one, rtol=8 * U, atol=1e-12)
        torch.testing.assert_close(xc.grad, 0.25 * one, rtol=8 * U, atol=1e-12)
        assert (zero == 0).all()
        lpc = lp.cuda().requires_grad_(True)
        loss = rl_triton.compute_policy_loss(lpc, *args[1:], kl_coef=0.1, grad_scale=scale)
        one = torch.autograd.grad(loss, lpc, retain_graph=True)[0]
        kept = one.clone()
        third = torch.autograd.grad(3.0 * loss, lpc, retain_graph=True)[0]
        (0.25 * loss).backward()
        assert torch.equal(one, kept)
        torch.testing.assert_close(third, 3 * one, rtol=8 * U, atol=1e-12)
        torch.testing.assert_close(lpc.grad, 0.25 * one, rtol=8 * U, atol=1e-12)


def test_no_second_derivative():
    _cuda()
    import rl_triton
    x, tok, _, _ = make(1, 2, 9)
    xc = x.cuda().requires_grad_(True)
    (g,) = torch.autograd.grad(rl_triton.compute_token_logprobs(xc, tok.cuda()).sum(), xc, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


PREF_SIZES = [(1, 1, 1), (1, 5, 9), (3, 17, 17), (4, 128, 64), (130, 33, 40), (2, 20001, 3)]


@pytest.mark.parametrize("b,tc,tr", PREF_SIZES)
@pytest.mark.parametrize("loss,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("ipo", 0.0), ("hinge", 0.0)])
@pytest.mark.parametrize("normalized", [False, True])
def test_preference_loss(b, tc, tr, loss, smoothing, normalized):
    """Sums are fp64: a reward is off by its rounding, the loss and the
    coefficients likewise (x up to 100 goes through exp: 128 u)."""
    _cuda()
    import rl_triton
    g = torch.Generator().manual_seed(b + tc)
    lp = [-3 * torch.rand(b, t, generator=g) for t in (tc, tr)]
    per_pair = (b + tc) % 2 == 1
    refs = [x.sum(1) + torch.randn(b, generator=g) if per_pair else x + 0.2 * torch.randn(x.shape, generator=g)
            for x in lp]
    masks = [torch.rand(x.shape, generator=g) < 0.8 for x in lp]
    if b > 2:
        masks[0][1] = False
        masks[1][2] = False
    if not per_pair:
        for r, m in zip(refs, masks):
            r[~m] = INF
    ld = [x.double().requires_grad_(True) for x in lp]
    want, wa, wb = ref64.preference(*ld, [r.double() for r in refs], masks, 0.1, loss, smoothing, normalized)
    wg = torch.autograd.grad(want, ld)
    lc = [x.cuda().requires_grad_(True) for x in lp]
    kw = dict(beta=0.1, loss=loss, label_smoothing=smoothing, length_normalized=normalized)
    got, a, bb = rl_triton.compute_preference_loss(tuple(lc), [r.cuda() for r in refs], [m.cuda() for m in masks], **kw)
    tol = dict(rtol=128 * U, atol=1e-7)
    close(got, want, **tol)
    close(a, wa, **tol)
    close(bb, wb, **tol)
    assert not a.requires_grad
    gg = torch.autograd.grad(2.0 * got, lc)
    for x, y in zip(gg, wg):
        close(x, 2.0 * y, rtol=128 * U, atol=1e-9)
    if tc == tr:  # one tensor with both halves
        whole = torch.cat(lp).cuda().requires_grad_(True)
        got2, a2, b2 = rl_triton.compute_preference_loss(whole, torch.cat(refs).cuda(), torch.cat(masks).cuda(), **kw)
        assert torch.equal(got2, got) and torch.equal(a2, a) and torch.equal(b2, bb)
        (g2,) = torch.autograd.grad(2.0 * got2, whole)
        assert torch.equal(g2, torch.cat(gg))


@pytest.mark.parametrize("b,t", [(3, 5), (1, 1), (5, 7), (2, 130)])
def test_preference_halves_off_the_vector_boundary(b, t):
    _cuda()
    import rl_triton
    g = torch.Generator().manual_seed(t)
    lp = -torch.rand(2 * b, t, generator=g)
    refl = -torch.rand(2 * b, t, generator=g)
    lc = lp.cuda().requires_grad_(True)
    loss, a, r = rl_triton.compute_preference_loss(lc, refl.cuda())
    (got,) = torch.autograd.grad(loss, lc)
    ld = lp.double().requires_grad_(True)
    want, wa, wr = ref64.preference(ld[:b], ld[b:], (refl[:b].double(), refl[b:].double()))
    (wg,) = torch.autograd.grad(want, ld)
    close(loss, want, rtol=16 * U, atol=1e-7)
    close(a, wa, rtol=16 * U, atol=1e-7)
    close(r, wr, rtol=16 * U, atol=1e-7)
    close(got, wg, rtol=16 * U, atol=1e-9)


@pytest.mark.parametrize("v", [18, 3000])
def test_gradients_against_differences(v):
    """(L(x + h d) - L(x - h d)) / 2h along random directions: with h = 2^-6 the
    fp32 losses' rounding is worth 2^7 u of their size and the third derivative
    h^2 of the terms, which are of the order of 1 (the clip's kinks are left out
    by a wide clip)."""
    _cuda()
    import rl_triton
    x, tok, mask, g = make(3, 8, v, seed=11, scale=1.0)
    lp, old, refl, adv, _ = _policy_inputs(3, 8, 4, False)
    tok, mask, old, refl, adv = (a.cuda() for a in (tok, mask, old, refl, adv))
    mask[1] = True

    def policy(z):
        base = rl_triton.compute_token_logprobs(x.cuda(), tok, mask)
        return rl_triton.compute_policy_loss_from_logits(z, tok, base + 0.1, adv, mask, base - 0.1, clip_low=0.9,
                                                         clip_high=9.0, kl_coef=0.2, entropy_coef=0.1)[0]

    def pref(z):
        q = rl_triton.compute_token_logprobs(z, tok, mask)
        return rl_triton.compute_preference_loss((q[:1], q[1:2]), None, (mask[:1], mask[1:2]), beta=0.3)[0]

    def both(z):
        q, h = rl_triton.compute_token_logprobs(z, tok, mask, 0.8, return_entropy=True)
        return (q.square().mean() + h.mean())

    h = 2.0 ** -6
    for f in (policy, pref, both):
        xc = x.cuda().requires_grad_(True)
        (grad,) = torch.autograd.grad(f(xc), xc)
        for k in range(3):
            d = torch.randn(x.shape, generator=g).cuda()
            with torch.no_grad():
                up, down = float(f(xc + h * d)), float(f(xc - h * d))
            slope = float((grad.double() * d.double()).sum())
            size = abs(up) + abs(down) + 1.0
            assert abs((up - down) / (2 * h) - slope) <= size * (2 ** 7 * 4 * U + 16 * h * h)


def test_bf16_logprobs_inputs():
    _cuda()
    import rl_triton
    lp, old, refl, adv, mask = _policy_inputs(4, 9, 6, False)
    low = [a.bfloat16() for a in (lp, old, refl, adv)]
    lc = low[0].cuda().requires_grad_(True)
    loss = rl_triton.compute_policy_loss(lc, low[1].cuda(), low[3].cuda(), mask.cuda(), low[2].cuda(), kl_coef=0.1)
    (g,) = torch.autograd.grad(loss, lc)
    ld = low[0].double().requires_grad_(True)
    want, _ = ref64.policy(ld, low[1].double(), low[3].double(), mask, low[2].double(), kl_coef=0.1)
    (wg,) = torch.autograd.grad(want, ld)
    close(loss, want, rtol=2 * U, atol=96 * U)
    assert g.dtype == torch.bfloat16
    close(g, wg, rtol=2 ** -8, atol=96 * U)
    lc = low[0].cuda().requires_grad_(True)
    loss, _, _ = rl_triton.compute_preference_loss(lc, low[1].cuda(), mask.cuda())
    (g,) = torch.autograd.grad(loss, lc)
    assert g.dtype == torch.bfloat16 and g.shape == lc.shape


def test_runs_on_the_current_stream_and_repeats_exactly():
    """Inputs made on a stream of their own; the same call gives the same bits."""
    _cuda()
    import rl_triton
    x, tok, mask, _ = make(16, 64, 5000, torch.bfloat16, seed=2)
    _, old, refl, adv, _ = _policy_inputs(16, 64, 2, False)
    side = torch.cuda.Stream()
    outs = []
    for k in range(3):
        with torch.cuda.stream(side if k else torch.cuda.current_stream()):
            xc = x.cuda(non_blocking=False).mul(1.0).requires_grad_(True)
            loss, lp = rl_triton.compute_policy_loss_from_logits(xc, tok.cuda(), old.cuda(), adv.cuda(), mask.cuda(),
                                                                 refl.cuda(), kl_coef=0.1, reduction="sequence")
            (g,) = torch.autograd.grad(loss, xc)
            l2, a, b = rl_triton.compute_preference_loss(lp, refl.cuda(), mask.cuda())
            outs.append([t.detach().clone() for t in (loss, lp, g, l2, a, b)])
        torch.cuda.synchronize()
    for other in outs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(outs[0], other))


def test_offsets_past_32_bits():
    """Rows that start beyond 2^31 elements of a strided tensor."""
    _cuda()
    import rl_triton
    v, rows = 4001, 3
    step = (1 << 30) + 13
    flat = torch.empty(step * (rows - 1) + v + 1, dtype=torch.bfloat16, device="cuda")
    x = flat[1:].as_strided((rows, 1, v), (step, v, 1))
    vals, tok, _, _ = make(rows, 1, v, torch.bfloat16, seed=8)
    x.copy_(vals.cuda())
    xd = vals.double().requires_grad_(True)
    want, _ = ref64.logprobs(xd, tok)
    (wg,) = torch.autograd.grad(want.sum(), xd)
    leaf = x.detach().requires_grad_(True)
    lp = rl_triton.compute_token_logprobs(leaf, tok.cuda())
    (g,) = torch.autograd.grad(lp.sum(), leaf)
    close(lp, want, **tol_lp(v))
    close(g, wg, **tol_grad(v, 4.0, True))


def test_large_batches_of_short_rows():
    _cuda()
    import rl_triton
    x, tok, _, g = make(300, 128, 18, seed=9)
    xd = x.double().requires_grad_(True)
    lp64, h64 = ref64.logprobs(xd, tok)
    old = (lp64 + 0.1).detach().float()
    adv = torch.randn(300, 128, generator=g)
    want, _ = ref64.policy(lp64, old.double(), adv.double(), entropy=h64, entropy_coef=0.01)
    (wg,) = torch.autograd.grad(want, xd)
    xc = x.cuda().requires_grad_(True)
    loss, lp = rl_triton.compute_policy_loss_from_logits(xc, tok.cuda(), old.cuda(), adv.cuda(), entropy_coef=0.01)
    (got,) = torch.autograd.grad(loss, xc)
    close(lp, lp64, **tol_lp(18))
    close(loss, want, rtol=2 * U, atol=12 * (S(18) + 8 * U))
    close(got, wg, **tol_grad(18, 4 * float(wg.abs().max()), False))


def _train_step(x, tok, old, adv, mask, refl):
    import rl_triton
    loss, lp, stats = rl_triton.compute_policy_loss_from_logits(x, tok, old, adv, mask, refl, kl_coef=0.1,
                                                                entropy_coef=0.01, return_stats=True)
    lp2, h = rl_triton.compute_token_logprobs(x, tok, mask, return_entropy=True)
    pref, a, b = rl_triton.compute_preference_loss(lp2, refl, mask)
    pol = rl_triton.compute_policy_loss(lp2, old, adv, mask, refl, kl_coef=0.1)
    return loss, lp, stats["kl"], h, pref, a, b, pol


def _step_inputs(v=700):
    x, tok, mask, _ = make(4, 16, v, seed=4)
    _, old, refl, adv, _ = _policy_inputs(4, 16, 4, False)
    return [a.cuda() for a in (x, tok, old, adv, mask, refl)]


def test_compile_fullgraph_matches_eager(monkeypatch):
    _cuda()
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    args = _step_inputs()
    torch._dynamo.reset()

    def step(*a):
        return _train_step(*a)

    compiled = torch.compile(step, fullgraph=True)
    for need in (False, True):
        xs = [args[0].clone().requires_grad_(need) for _ in range(2)]
        want, got = step(xs[0], *args[1:]), compiled(xs[1], *args[1:])
        for p, q in zip(want, got):
            torch.testing.assert_close(p, q)
        if need:
            (want[0] + want[4] + want[7] + want[3].mean()).backward()
            (got[0] + got[4] + got[7] + got[3].mean()).backward()
            torch.testing.assert_close(xs[0].grad, xs[1].grad)


def test_graph_capture_of_a_training_step(monkeypatch):
    _cuda()
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    args = _step_inputs(2500)
    x = args[0].clone().requires_grad_(True)

    def step():
        out = _train_step(x, *args[1:])
        (g,) = torch.autograd.grad(out[0] + out[4] + out[7], x)
        return [*out, g]

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(want, out):
        torch.testing.assert_close(p, q.detach())


@pytest.mark.parametrize("v", [1500, 40000, 131072])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_likely_tokens_keep_their_relative_accuracy(v, dtype):
    """A token with nearly all of the probability: the log-probability's error
    is that of the sum of the others, S(V), relative to the log-probability
    itself (rows of more than 1024 logits)."""
    _cuda()
    import rl_triton
    x = torch.randn(1, 24, v, generator=torch.Generator().manual_seed(v)).to(dtype)
    tok = torch.arange(24)[None] * 37 % v
    top = (math.log(v) + torch.arange(24) * 0.75)[None, :, None].to(dtype)
    x.scatter_(2, tok[..., None], top)
    lp = rl_triton.compute_token_logprobs(x.cuda(), tok.cuda())
    want, _ = ref64.logprobs(x.double(), tok)
    assert float(want.max()) > -1e-5
    torch.testing.assert_close(lp.cpu().double(), want, rtol=2 * S(v), atol=0.0)


def test_refusals():
    _cuda()
    import rl_triton as rl
    x, lp = torch.zeros(2, 3, 5).cuda(), torch.zeros(2, 3).cuda()
    tok = torch.zeros(2, 3, dtype=torch.long).cuda()

    def refuses(match, fn, *args, **kw):
        with pytest.raises(AssertionError, match=match):
            fn(*args, **kw)

    refuses("num_envs, seq_len, vocab", rl.compute_token_logprobs, x[0], tok[0])
    refuses("float32 or bfloat16", rl.compute_token_logprobs, x.half(), tok)
    refuses("tokens shape", rl.compute_token_logprobs, x, tok[:, :2])
    refuses("expected integers", rl.compute_token_logprobs, x, lp)
    refuses("mask shape", rl.compute_token_logprobs, x, tok, lp[:1])
    refuses("vocabulary is empty", rl.compute_token_logprobs, x[..., :0], tok)
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        refuses("temperature", rl.compute_token_logprobs, x, tok, None, bad)
    refuses("must be on cuda", rl.compute_token_logprobs, x, tok.cpu())
    refuses("old_logprobs shape", rl.compute_policy_loss, lp, lp[:1], lp)
    refuses("advantages shape", rl.compute_policy_loss, lp, lp, lp[:, :2])
    refuses("needs ref_logprobs", rl.compute_policy_loss, lp, lp, lp, kl_coef=0.1)
    refuses("kl must be", rl.compute_policy_loss, lp, lp, lp, kl="k4")
    refuses("reduction must be", rl.compute_policy_loss, lp, lp, lp, reduction="mean")
    refuses("dual_clip", rl.compute_policy_loss, lp, lp, lp, dual_clip=1.0)
    refuses("negative", rl.compute_policy_loss, lp, lp, lp, clip_low=-0.1)
    refuses("must be on cuda", rl.compute_policy_loss, lp, lp.cpu(), lp)
    refuses("mask shape", rl.compute_policy_loss_from_logits, x, tok, lp, lp, lp[:1])
    refuses("2 \\* pairs", rl.compute_preference_loss, lp[:1])
    refuses("loss must be", rl.compute_preference_loss, lp, loss="dpo")
    refuses("label_smoothing", rl.compute_preference_loss, lp, label_smoothing=0.5)
    refuses("belongs to the sigmoid", rl.compute_preference_loss, lp, loss="ipo", label_smoothing=0.1)
    refuses("beta", rl.compute_preference_loss, lp, beta=0.0)
    refuses("neither", rl.compute_preference_loss, lp, lp[:, :2])
    refuses("both or none", rl.compute_preference_loss, (lp, lp), (lp, None))
    refuses("alike for both", rl.compute_preference_loss, (lp, lp), (lp, lp[:, 0]))
    refuses("pairs, len", rl.compute_preference_loss, (lp, lp[:1]))
    with pytest.raises(RuntimeError, match="must be on"):  # the operator itself, without the function's checks
        torch.ops.rl_triton._token_logprobs(x, tok.cpu(), None, 1.0, False, False)


def test_operator_schemas_and_fake_kernels(monkeypatch):
    """torch.library.opcheck: schema and fake kernel consistency."""
    _cuda()
    monkeypatch.setenv("RL_TRITON_CORRECTNESS_WARNINGS", "0")
    ops = torch.ops.rl_triton
    for v in (9, 1100):
        x, tok, mask, _ = make(3, 4, v, seed=v)
        x, tok, mask = x.cuda(), tok.cuda(), mask.cuda()
        lp, old, refl, adv, _ = (a.cuda() for a in _policy_inputs(3, 4, 1, False))
        out = ops._token_logprobs(x, tok, mask, 1.0, True, True)
        checks = [
            (ops._grad_buffer, (x[:, 1:],)),
            (ops._token_logprobs, (x, tok, mask, 1.0, True, True)),
            (ops._token_logprobs_backward, (x, tok, mask, out[3], out[2], lp, lp, 1.0)),
            (ops._policy_loss, (lp, old, adv, mask, refl, 0.2, 0.2, 0.0, 0.1, 3, 1, 1.0, True, True)),
            (ops._policy_loss_logits, (x, tok, old, adv, mask, refl, 0.2, 0.2, 0.0, 0.1, 3, 0.01, True, 1.0, 0, 1.0,
                                       True)),
            (ops._preference_loss, (lp[:2], None, refl[:2], None, mask[:2], None, 0.1, 0.0, 0, False)),
            (ops._preference_loss_backward, (torch.ones(2, 3).cuda(), torch.ones(()).cuda(), None, None, 4, 5, False)),
        ]
        for op, args in checks:
            torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("n,t", [(1, 1), (3, 7), (40, 33), (1, 70001), (3000, 3)])
def test_row_order(n, t):
    """A permutation of the steps, those that count first."""
    _cuda()
    from rl_triton import _native as nat
    mask = (torch.rand(n, t, generator=torch.Generator().manual_seed(n)) < 0.5).cuda()
    order = torch.empty(n * t + 1, dtype=torch.int32, device="cuda")
    ws, wsb = nat.workspace(mask.device, nat.stream_handle(mask.device), 1 << 20)
    st = nat.lib.rls_row_order(mask.data_ptr(), nat.MASK_U8, n, t, order.data_ptr(), ws, wsb,
                               nat.stream_handle(mask.device))
    assert st == nat.RLS_OK
    o = order.cpu().long()
    k = int(mask.sum())
    flat = mask.flatten().cpu()
    assert int(o[0]) == k
    assert torch.equal(torch.sort(o[1:]).values, torch.arange(n * t))
    assert flat[o[1:1 + k]].all() and not flat[o[1 + k:]].any()


@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
def test_long_rows_behind_a_ragged_mask(reduction):
    """Many rows, most of them masked, so that every team has skipped rows."""
    _cuda()
    import rl_triton
    n, t, v = 40, 50, 1200
    x, tok, _, g = make(n, t, v, torch.bfloat16, seed=17)
    mask = (torch.arange(t)[None] >= torch.randint(0, 10, (n, 1), generator=g)) & \
        (torch.arange(t)[None] < torch.randint(5, t, (n, 1), generator=g))
    mask[::4] = False
    x[~mask] = float("nan")
    xd = torch.where(mask[..., None], x, torch.zeros_like(x)).double().requires_grad_(True)
    lp64, h64 = ref64.logprobs(xd, tok, mask)
    old = (lp64 + 0.1 * torch.randn(n, t, generator=g)).detach().float()
    adv = torch.randn(n, generator=g)
    want, _ = ref64.policy(lp64, old.double(), adv.double(), mask, entropy=h64, entropy_coef=0.01, reduction=reduction)
    (wg,) = torch.autograd.grad(want, xd)
    xc = x.cuda().requires_grad_(True)
    loss, lp = rl_triton.compute_policy_loss_from_logits(xc, tok.cuda(), old.cuda(), adv.cuda(), mask.cuda(),
                                                         entropy_coef=0.01, reduction=reduction)
    (got,) = torch.autograd.grad(loss, xc)
    many = int(mask.sum()) if reduction == "sum" else 1
    close(lp, lp64, **tol_lp(v))
    close(loss, want, rtol=2 * U, atol=many * 12 * (S(v) + 8 * U + 0.01 * tol_ent(v)["atol"]))
    close(got, wg, **tol_grad(v, 4 * float(wg.abs().max()), True))
    assert (got[~mask.cuda()] == 0).all()


def test_example_runs():
    _cuda()
    import importlib.util
    import os
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "token_policy_update.py")
    spec = importlib.util.spec_from_file_location("token_policy_update", at)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    h = m.main(steps=12, envs=32, length=16, vocab=1200, out=lambda s: None)
    assert all(math.isfinite(v) for d in h for v in d.values())
    assert h[-1]["reward"] > h[0]["reward"] + 0.2  # the policy learns the task
