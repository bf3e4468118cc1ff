"""The token-level policy operators without a GPU: what the C entry points and
the Python functions refuse before anything is launched, the public names and
signatures, and the plain 64-bit forms that the GPU tests compare with (their
gradients against differences)."""
import ctypes
import inspect

import pytest
import torch

import _token_ref as ref64
from rl_triton import _native as nat

EINVAL, EALIGN, EWORKSPACE, ENOTDEVICE = 1, 2, 3, nat.RLS_ENOTDEVICE
L = nat.lib


def _host():
    buf = (ctypes.c_float * 4096)()
    base = ctypes.addressof(buf)
    return buf, base + (16 - base % 16) % 16


def _policy(**kw):
    d = dict(clip_low=0.2, clip_high=0.2, dual_clip=0.0, kl_coef=0.0, entropy_coef=0.0, kl_kind=nat.KL_K3,
             reduction=nat.REDUCE_TOKEN)
    return nat.Policy(**{**d, **kw})


def test_signatures():
    import rl_triton
    want = {
        "compute_token_logprobs": "(logits, tokens, mask=None, temperature=1.0, return_entropy=False)",
        "compute_policy_loss": "(logprobs, old_logprobs, advantages, mask=None, ref_logprobs=None, clip_low=0.2, "
                               "clip_high=None, dual_clip=None, kl_coef=0.0, kl='k3', reduction='token', "
                               "grad_scale=1.0, return_stats=False)",
        "compute_policy_loss_from_logits": "(logits, tokens, old_logprobs, advantages, mask=None, ref_logprobs=None, "
                                           "clip_low=0.2, clip_high=None, dual_clip=None, kl_coef=0.0, kl='k3', "
                                           "entropy_coef=0.0, temperature=1.0, reduction='token', grad_scale=1.0, "
                                           "return_stats=False)",
        "compute_preference_loss": "(logprobs, ref_logprobs=None, mask=None, beta=0.1, loss='sigmoid', "
                                   "label_smoothing=0.0, length_normalized=False)",
    }
    for name, sig in want.items():
        fn = getattr(rl_triton, name)
        assert name in rl_triton.__all__
        ps = [p.replace(annotation=inspect.Parameter.empty) for p in inspect.signature(fn).parameters.values()]
        assert str(inspect.Signature(ps)) == sig


def test_host_tensors_are_refused():
    import rl_triton
    x, tok, lp = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3)
    with pytest.raises(AssertionError, match="CUDA"):
        rl_triton.compute_token_logprobs(x, tok)
    with pytest.raises(AssertionError, match="CUDA"):
        rl_triton.compute_policy_loss(lp, lp, lp)
    with pytest.raises(AssertionError, match="CUDA"):
        rl_triton.compute_policy_loss_from_logits(x, tok, lp, lp)
    with pytest.raises(AssertionError, match="CUDA"):
        rl_triton.compute_preference_loss(lp)


def test_entry_points_refuse_bad_arguments():
    _, a = _host()
    lp = lambda **k: L.rls_token_logprobs(  # noqa: E731
        *[k.get(n, v) for n, v in dict(x=a, es=8, ss=4, tok=a, mask=None, kind=0, order=None, out=a, ent=None, st=None,
                                       n=2, t=2, v=4, temp=1.0, dt=0, s=None).items()])
    assert lp(x=None) == lp(tok=None) == lp(out=None) == EINVAL
    assert lp(v=0) == lp(v=1 << 31) == lp(n=-1) == lp(dt=2) == lp(es=-1) == EINVAL
    assert lp(temp=0.0) == lp(temp=-1.0) == lp(temp=float("inf")) == lp(temp=float("nan")) == EINVAL
    assert lp(kind=nat.MASK_U8) == lp(mask=a) == lp(mask=a, kind=6) == EINVAL  # a mask and its kind go together
    assert lp(order=a) == EINVAL                                              # an order needs its mask
    assert lp(x=a + 2) == lp(tok=a + 4) == lp(out=a + 4) == lp(mask=a + 2, kind=nat.MASK_F32) == EALIGN
    assert lp() == ENOTDEVICE
    assert lp(n=0) == lp(t=0) == 0

    def bwd(**k):
        d = dict(x=a, es=8, ss=4, tok=a, mask=None, kind=0, order=None, st=a, gl=a, ge=None, g=a, ges=8, gss=4, n=2, t=2,
                 v=4, temp=1.0, dt=0, s=None)
        return L.rls_token_logprobs_backward(*{**d, **k}.values())

    assert bwd(g=None) == EINVAL
    assert bwd(v=2000, st=None, es=4000, ss=2000, ges=4000, gss=2000) == EINVAL  # long rows need their statistics
    assert bwd(gss=3) == bwd(ges=5) == EINVAL                                    # rows that overlap
    assert bwd(ges=4, gss=8) == ENOTDEVICE                                       # the envs inside the steps are fine
    assert bwd(g=a + 2) == EALIGN
    assert bwd() == ENOTDEVICE

    def pol(**k):
        d = dict(lp=a, old=a, adv=a, per=0, ref=None, mask=None, kind=0, p=_policy(), scale=1.0, norm=None, loss=a,
                 stats=None, g=None, n=2, t=2, ws=a, wsb=4096, s=None)
        d.update(k)
        d["p"] = ctypes.byref(d["p"]) if d["p"] is not None else None
        return L.rls_policy_loss(*d.values())

    assert pol(lp=None) == pol(old=None) == pol(adv=None) == pol(loss=None) == pol(p=None) == pol(ws=None) == EINVAL
    assert pol(p=_policy(kl_kind=0)) == pol(p=_policy(reduction=3)) == EINVAL
    assert pol(mask=a, kind=nat.MASK_U8) == EINVAL                              # a mean under a mask needs norm
    assert pol(lp=a + 4) == pol(g=a + 4) == pol(loss=a + 2) == EALIGN
    assert pol() == ENOTDEVICE

    def pref(**k):
        d = dict(c=a, r=a, rc=None, rr=None, rp=0, mc=None, mr=None, kind=0, b=2, tc=2, tr=2, beta=0.1, e=0.0, k=0,
                 ln=0, loss=a, good=a, bad=a, coef=a, ws=a, wsb=4096, s=None)
        return L.rls_preference_loss(*{**d, **k}.values())

    assert pref(c=None) == pref(r=None) == pref(loss=None) == pref(good=None) == pref(ws=None) == EINVAL
    assert pref(k=3) == pref(beta=float("nan")) == pref(beta=0.0, k=1) == pref(b=-1) == pref(mc=a) == EINVAL
    assert pref(wsb=64) == EWORKSPACE
    assert pref(c=a + 2) == EALIGN
    assert pref() == ENOTDEVICE
    assert L.rls_row_order(a, nat.MASK_U8, 1 << 20, 1 << 12, a, a, 4096, None) == EINVAL  # rows past 31 bits
    assert L.rls_row_order(a, nat.MASK_U8, 2, 2, a, a, 4096, None) == ENOTDEVICE


def test_assumed_device_is_the_threads_own():
    import threading
    assert L.rls_assume_device(0) == -1
    seen = []
    th = threading.Thread(target=lambda: seen.append(L.rls_assume_device(-1)))
    th.start()
    th.join()
    assert seen == [-1]
    assert L.rls_assume_device(-1) == 0 and L.rls_assume_device(-1) == -1


def test_operators_refuse_tensors_of_another_device():
    """Straight calls of the operators, without the functions' checks."""
    x, lp = torch.zeros(2, 3, 5, device="meta"), torch.zeros(2, 3)
    with pytest.raises((RuntimeError, NotImplementedError)):
        nat.ops._token_logprobs(torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long), None, 1.0, False, False)
    out = nat.ops.token_logprobs(x, torch.zeros(2, 3, dtype=torch.long, device="meta"), None, 1.0, True)
    assert out[0].shape == out[1].shape == (2, 3) and lp.shape == (2, 3)


def test_plain_forms_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 7, generator=g, dtype=torch.float64)
    tok = torch.randint(0, 7, (2, 3), generator=g)
    mask = torch.tensor([[1, 0, 1], [1, 1, 0]])
    old = ref64.logprobs(x, tok)[0] + 0.05
    adv = torch.randn(2, 3, generator=g, dtype=torch.float64)

    def f(z):
        lp, h = ref64.logprobs(z, tok, mask, 0.9)
        a, _ = ref64.policy(lp, old, adv, mask, old - 0.1, clip_low=0.9, clip_high=5.0, kl_coef=0.3, entropy=h,
                            entropy_coef=0.1, reduction="sequence")
        b, _, _ = ref64.preference(lp[:1], lp[1:], masks=(mask[:1], mask[1:]), smoothing=0.1)
        return a + b

    assert torch.autograd.gradcheck(f, (x.requires_grad_(True),), eps=1e-6, atol=1e-7)
