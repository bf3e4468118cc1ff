"""compute_policy_loss, compute_policy_loss_from_logits -- the clipped policy
loss with a KL term that takes the advantages of the estimators, with its
gradient (no counterpart in the reference, which ends at the advantages)."""
from __future__ import annotations

import torch

from rl_triton import _native as nat
from rl_triton.ops import _scan
from rl_triton.ops._scan import _CORRECTNESS_WARNINGS, _float_ok, _placed, _warn_copies
from rl_triton.ops.token_logprobs import _finished, _logits_args, _mask_arg

_op = nat.ops.policy_loss.default
_op_logits = nat.ops.policy_loss_logits.default

_REDUCTIONS = {"token": nat.REDUCE_TOKEN, "sequence": nat.REDUCE_SEQUENCE, "sum": nat.REDUCE_SUM}
_KL = {"k1": nat.KL_K1, "k2": nat.KL_K2, "k3": nat.KL_K3}


def compute_policy_loss(
    logprobs: torch.Tensor,
    old_logprobs: torch.Tensor,
    advantages: torch.Tensor,
    mask: torch.Tensor | None = None,
    ref_logprobs: torch.Tensor | None = None,
    clip_low: float = 0.2,
    clip_high: float | None = None,
    dual_clip: float | None = None,
    kl_coef: float = 0.0,
    kl: str = "k3",
    reduction: str = "token",
    grad_scale: float = 1.0,
    return_stats: bool = False,
):
    """
    The clipped policy loss over the steps that count (mask not 0):

        r    = exp(logprobs - old_logprobs)
        term = -min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A)
               (where A < 0 at most -dual_clip A, with dual_clip given)
               + kl_coef KL
        KL   = lp - ref ("k1"), (lp - ref)^2 / 2 ("k2"),
               exp(ref - lp) - (ref - lp) - 1 ("k3")
        loss = sum(term) / number of steps                       ("token")
             = mean over the sequences of their mean term        ("sequence";
               sequences without a step that counts are left out)
             = sum(term)                                         ("sum")

    Differentiable with respect to logprobs; the gradient is written in the
    same pass for an incoming gradient of `grad_scale` (the loss itself is not
    scaled).  The backward pass computes it anew only if the incoming gradient
    is another one: give the factor that loss.backward() will see (1 / the number
    of accumulated minibatches, a loss scale) to spare that.  The other inputs are
    constants of the loss: no gradient flows to old_logprobs, advantages or
    ref_logprobs, whether they require one or not.

    Args:
        logprobs, old_logprobs, ref_logprobs: [num_envs, seq_len], float32 or
            bfloat16; ref_logprobs is needed where kl_coef is not 0.
        advantages: [num_envs, seq_len], or [num_envs] (one for each sequence).
        mask: [num_envs, seq_len] bool, integer or floating ({0, 1}), optional.
            What the other arrays hold at mask 0 is not used.
        clip_high: 1 + clip_high bounds the ratio above; clip_low where not given.

    Returns:
        loss (scalar float32; 0 where no step counts), or (loss, stats) when
        return_stats is True: a dict of scalars, means over the steps that
        count: "kl" (to ref, in the chosen form), "approx_kl" (r - 1 - log r),
        "clip_fraction" (steps whose gradient the clip holds), and "num_steps".
    """
    assert logprobs.dim() == 2, f"logprobs must have shape [num_envs, seq_len], got {logprobs.shape}"
    assert logprobs.is_cuda, "logprobs must be on CUDA"
    assert _float_ok(logprobs), f"logprobs: expected float32 or bfloat16, got {logprobs.dtype}"
    c = _policy_args(logprobs.shape, old_logprobs, advantages, mask, ref_logprobs, clip_low, clip_high, dual_clip,
                     kl_coef, kl, reduction)
    _placed(logprobs, old_logprobs, advantages, mask, ref_logprobs)
    if _scan._PERF_WARNINGS:
        _warn_copies({"logprobs": logprobs, "old_logprobs": old_logprobs, "advantages": advantages, "mask": mask,
                      "ref_logprobs": ref_logprobs})
    loss, stats = _op(logprobs, old_logprobs, advantages, mask, ref_logprobs, *c, grad_scale, return_stats)
    if _CORRECTNESS_WARNINGS():
        _finished(logprobs)
    return (loss, _stats(stats, False)) if return_stats else loss


def compute_policy_loss_from_logits(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    old_logprobs: torch.Tensor,
    advantages: torch.Tensor,
    mask: torch.Tensor | None = None,
    ref_logprobs: torch.Tensor | None = None,
    clip_low: float = 0.2,
    clip_high: float | None = None,
    dual_clip: float | None = None,
    kl_coef: float = 0.0,
    kl: str = "k3",
    entropy_coef: float = 0.0,
    temperature: float = 1.0,
    reduction: str = "token",
    grad_scale: float = 1.0,
    return_stats: bool = False,
):
    """
    compute_token_logprobs and compute_policy_loss in one pass over the logits:
    each row's log-probability is taken and its gradient written while the row
    is at hand, so the logits are read once and their gradient written once.
    The loss has one term more, the entropy bonus:

        term = (as in compute_policy_loss) - entropy_coef entropy

    Differentiable with respect to the logits alone.  Arguments as there;
    `grad_scale` matters more here, since another incoming
    gradient costs a second pass over the logits.  The logits must not change
    before the backward pass.

    Returns:
        (loss, logprobs), logprobs [num_envs, seq_len] float32 without a
        gradient, or (loss, logprobs, stats) when return_stats is True; stats
        then also holds "entropy".
    """
    checks = _CORRECTNESS_WARNINGS()
    _logits_args(logits, tokens, mask, temperature, checks)
    c = _policy_args(logits.shape[:2], old_logprobs, advantages, None, ref_logprobs, clip_low, clip_high, dual_clip,
                     kl_coef, kl, reduction)
    _placed(logits, tokens, old_logprobs, advantages, mask, ref_logprobs)
    if _scan._PERF_WARNINGS:
        _warn_copies({"old_logprobs": old_logprobs, "advantages": advantages, "mask": mask,
                      "ref_logprobs": ref_logprobs})
    loss, lp, _, stats = _op_logits(logits, tokens, old_logprobs, advantages, mask, ref_logprobs, *c[:5], entropy_coef,
                                    return_stats, temperature, c[5], grad_scale)
    if checks:
        _finished(logits)
    return (loss, lp, _stats(stats, True)) if return_stats else (loss, lp)


def _policy_args(shape, old_logprobs, advantages, mask, ref_logprobs, clip_low, clip_high, dual_clip, kl_coef, kl,
                 reduction):
    """Checks; (clip_low, clip_high, dual_clip, kl_coef, kl, reduction) as the
    operators take them."""
    for name, t in (("old_logprobs", old_logprobs), ("ref_logprobs", ref_logprobs)):
        if t is not None:
            assert _float_ok(t), f"{name}: expected float32 or bfloat16, got {t.dtype}"
            assert t.shape == shape, f"{name} shape {t.shape} != {shape}"
    assert _float_ok(advantages), f"advantages: expected float32 or bfloat16, got {advantages.dtype}"
    assert advantages.shape == shape or advantages.shape == shape[:1], \
        f"advantages shape {advantages.shape} is neither {shape} nor {shape[:1]}"
    _mask_arg(mask, shape)
    assert kl in _KL, f"kl must be one of {sorted(_KL)}, got {kl!r}"
    assert reduction in _REDUCTIONS, f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}"
    assert kl_coef == 0.0 or ref_logprobs is not None, "kl_coef needs ref_logprobs"
    high = clip_low if clip_high is None else clip_high
    assert clip_low >= 0.0 and high >= 0.0, f"clip bounds must not be negative, got {clip_low}, {high}"
    assert dual_clip is None or dual_clip > 1.0, f"dual_clip must be greater than 1, got {dual_clip}"
    return clip_low, high, dual_clip or 0.0, kl_coef, _KL[kl], _REDUCTIONS[reduction]


def _stats(stats, entropy):
    d = {"kl": stats[0], "approx_kl": stats[1], "clip_fraction": stats[2]}
    if entropy:
        d["entropy"] = stats[3]
    d["num_steps"] = stats[4]
    return d
