"""compute_preference_loss -- the paired preference loss over token
log-probabilities, with its gradient (no counterpart in the reference)."""
from __future__ import annotations

import torch

from rl_triton import _native as nat
from rl_triton.ops import _scan
from rl_triton.ops._scan import _CORRECTNESS_WARNINGS, _float_ok, _placed, _warn_copies
from rl_triton.ops.token_logprobs import _finished, _mask_arg

_op = nat.ops.preference_loss.default

_KINDS = {"sigmoid": nat.PREFERENCE_SIGMOID, "ipo": nat.PREFERENCE_IPO, "hinge": nat.PREFERENCE_HINGE}


def compute_preference_loss(
    logprobs,
    ref_logprobs=None,
    mask=None,
    beta: float = 0.1,
    loss: str = "sigmoid",
    label_smoothing: float = 0.0,
    length_normalized: bool = False,
):
    """
    The preference loss of pairs of responses, one preferred to the other.
    Per response, over its steps that count (mask not 0):

        s = sum(logprobs - ref_logprobs)      (/ their number, with
                                               length_normalized; 0 of none)

    and per pair, with x = beta (s_chosen - s_rejected):

        "sigmoid"  -(1 - e) log sig(x) - e log sig(-x),   e = label_smoothing
        "ipo"      (x / beta - 1 / (2 beta))^2
        "hinge"    max(0, 1 - x)

    The loss is the mean over the pairs.  Differentiable with respect to the
    log-probabilities (compute_token_logprobs gives them from the logits); the
    reference's are constants, no gradient flows to them.

    Args:
        logprobs: [2 * pairs, seq_len], the preferred responses in the first
            half and the others, in the same order, in the second (as one
            forward pass over both gives them); or a pair of tensors
            ([pairs, len_a], [pairs, len_b]).  float32 or bfloat16.
        ref_logprobs: the reference policy's, per step in the layout of
            logprobs, or summed per response: [2 * pairs], or ([pairs],
            [pairs]).  None: 0.
        mask: in the layout of logprobs, bool, integer or floating ({0, 1}).

    Returns:
        (loss, chosen_rewards, rejected_rewards): a scalar and beta s of either
        response [pairs], float32, the rewards without a gradient.
    """
    assert loss in _KINDS, f"loss must be one of {sorted(_KINDS)}, got {loss!r}"
    assert 0.0 <= label_smoothing < 0.5, f"label_smoothing must be in [0, 0.5), got {label_smoothing}"
    assert label_smoothing == 0.0 or loss == "sigmoid", "label_smoothing belongs to the sigmoid loss"
    assert 0.0 < beta < float("inf"), f"beta must be positive and finite, got {beta}"
    if isinstance(logprobs, torch.Tensor):
        sides = [("logprobs", logprobs, ref_logprobs, mask)]
        assert logprobs.dim() == 2 and logprobs.shape[0] % 2 == 0, \
            f"logprobs must have shape [2 * pairs, seq_len], got {logprobs.shape}"
    else:
        assert len(logprobs) == 2, "logprobs: one tensor with both halves, or (chosen, rejected)"
        refs = (None, None) if ref_logprobs is None else tuple(ref_logprobs)
        masks = (None, None) if mask is None else tuple(mask)
        assert len(refs) == 2 and len(masks) == 2, "ref_logprobs and mask must be pairs like logprobs"
        assert (refs[0] is None) == (refs[1] is None), "ref_logprobs: give both or none"
        sides = [(f"logprobs[{k}]", logprobs[k], refs[k], masks[k]) for k in range(2)]
        assert all(t.dim() == 2 for t in logprobs) and logprobs[0].shape[0] == logprobs[1].shape[0], \
            f"logprobs must be [pairs, len] and [pairs, len], got {logprobs[0].shape} and {logprobs[1].shape}"
    for name, lp, ref, m in sides:
        assert lp.is_cuda, f"{name} must be on CUDA"
        assert _float_ok(lp), f"{name}: expected float32 or bfloat16, got {lp.dtype}"
        if ref is not None:
            assert _float_ok(ref), f"reference of {name}: expected float32 or bfloat16, got {ref.dtype}"
            assert ref.shape == lp.shape or ref.shape == lp.shape[:1], \
                f"reference of {name}: shape {ref.shape} is neither {lp.shape} nor {lp.shape[:1]}"
        _mask_arg(m, lp.shape, f"mask of {name}")
    first = sides[0][1]
    if len(sides) == 2 and sides[0][2] is not None:
        assert sides[0][2].dim() == sides[1][2].dim(), "ref_logprobs: per step or per response, alike for both"
    _placed(first, *(t for s in sides for t in s[1:]))
    if _scan._PERF_WARNINGS:
        _warn_copies({f"{what} of {s[0]}": t for s in sides for what, t in zip(("values", "reference", "mask"), s[1:])})
    lp, ref, m = sides[0][1:]
    lp2, ref2, m2 = sides[1][1:] if len(sides) == 2 else (None, None, None)
    value, good, bad = _op(lp, lp2, ref, ref2, m, m2, beta, label_smoothing, _KINDS[loss], length_normalized)
    if _CORRECTNESS_WARNINGS():
        _finished(first)
    return value, good, bad
