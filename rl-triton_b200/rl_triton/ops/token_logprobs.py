"""compute_token_logprobs -- log-probabilities (and entropies) of the tokens a
policy took, from its logits, with their gradient (no counterpart in the
reference, whose V-trace takes the log-probabilities as given:
src/rl_triton/ops/vtrace.py)."""
from __future__ import annotations

import torch

from rl_triton import _native as nat
from rl_triton.ops._scan import _CORRECTNESS_WARNINGS, _float_ok, _perf_warn, _placed

_op = nat.ops.token_logprobs.default


def compute_token_logprobs(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    mask: torch.Tensor | None = None,
    temperature: float = 1.0,
    return_entropy: bool = False,
):
    """
    Log-probabilities of the tokens taken, in one pass over the logits:

        z = logits / temperature
        logprobs[n, t] = z[n, t, tokens[n, t]] - logsumexp(z[n, t])
        entropy[n, t]  = -sum_v p[v] log p[v],  p = softmax(z[n, t])

    Differentiable with respect to the logits (the backward pass reads them
    once more and writes their gradient in their own type).

    Args:
        logits: [num_envs, seq_len, vocab], float32 or bfloat16.  The vocabulary
            must be contiguous (else a copy is made); the steps may be strided
            (logits[:, :-1] and the like) and need no alignment.  Entries may be
            -inf (tokens that cannot be taken).
        tokens: [num_envs, seq_len], any integer type.
        mask: [num_envs, seq_len] bool, integer or floating ({0, 1}), optional.
            Steps with mask 0 have log-probability and entropy 0, and their
            logits and tokens are not used: their gradient is 0.
        temperature: divides the logits; the gradient is that of the logits.

    A token outside the vocabulary at a step that counts gives NaN there.

    Returns:
        logprobs [num_envs, seq_len] float32, or (logprobs, entropy) when
        return_entropy is True.
    """
    checks = _CORRECTNESS_WARNINGS()
    _logits_args(logits, tokens, mask, temperature, checks)
    _placed(logits, tokens, mask)
    lp, ent = _op(logits, tokens, mask, temperature, return_entropy)
    if checks:
        _finished(logits)
    return (lp, ent) if return_entropy else lp


def _logits_args(logits, tokens, mask, temperature, checks):
    assert logits.is_cuda, "logits must be on CUDA"
    shape = logits.shape
    assert len(shape) == 3, f"logits must have shape [num_envs, seq_len, vocab], got {shape}"
    assert _float_ok(logits), f"logits: expected float32 or bfloat16, got {logits.dtype}"
    assert shape[2] > 0, "logits: the vocabulary is empty"
    steps = shape[:2]
    assert tokens.shape == steps, f"tokens shape {tokens.shape} != {steps} of the logits"
    assert tokens.dtype in _INTEGERS, f"tokens: expected integers, got {tokens.dtype}"
    assert 0.0 < temperature < float("inf"), f"temperature must be positive and finite, got {temperature}"
    _mask_arg(mask, steps)
    if shape[2] > 1 and logits.stride(2) != 1:
        _perf_warn("logits: the vocabulary is not contiguous; a copy will be made.")
    if checks and not torch.cuda.is_current_stream_capturing():
        bad = (tokens < 0) | (tokens >= shape[2])
        assert not (bad if mask is None else bad & (mask != 0)).any(), \
            "tokens: a step that counts has a token outside the vocabulary"


_INTEGERS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


def _finished(ref):
    """RL_TRITON_CORRECTNESS_WARNINGS=1: wait for the call and raise if one of
    its bounded device waits ran out."""
    if not torch.cuda.is_current_stream_capturing():
        nat.raise_if_device_error(ref.device)


def _mask_arg(mask, shape, name="mask"):
    if mask is None:
        return
    assert mask.shape == shape, f"{name} shape {mask.shape} != {shape}"
    assert not mask.is_complex(), f"{name}: expected bool, integers or floats, got {mask.dtype}"
