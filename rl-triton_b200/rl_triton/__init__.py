"""rl_triton (B200 build) -- drop-in for the seven return-estimation scans of
simonsays1980/rl-triton v0.1.3, computed by hand-written sm_100a CUDA kernels
(librlscan.so) instead of Triton.  Same function names, signatures, module
paths and error behaviour as the reference's src/rl_triton/__init__.py, plus
fused PPO epilogues (compute_gae_normalized, compute_gae_value_loss) and the
observation-skip masking mode (compute_gae_obs_skip) the reference does not
have, and the token-level policy operators around them: log-probabilities from
logits (compute_token_logprobs), the clipped policy loss (compute_policy_loss,
compute_policy_loss_from_logits) and the paired preference loss
(compute_preference_loss), each with its gradient."""

__version__ = "0.1.3"

from rl_triton.ops.gae import compute_gae
from rl_triton.ops.retrace import compute_retrace
from rl_triton.ops.prefix_sum import compute_episodic_prefix_sum
from rl_triton.ops.returns import compute_discounted_returns, compute_eligibility_traces, compute_lambda_returns
from rl_triton.ops.vtrace import compute_vtrace
from rl_triton.ops.fused import (  # additions: fused PPO epilogues and masking modes
    compute_gae_normalized,
    compute_gae_obs_skip,
    compute_gae_value_loss,
)
from rl_triton.ops.token_logprobs import compute_token_logprobs  # additions: token-level policy operators
from rl_triton.ops.policy_loss import compute_policy_loss, compute_policy_loss_from_logits
from rl_triton.ops.preference_loss import compute_preference_loss

__all__ = [
    "compute_discounted_returns",
    "compute_eligibility_traces",
    "compute_episodic_prefix_sum",
    "compute_gae",
    "compute_gae_normalized",
    "compute_gae_obs_skip",
    "compute_gae_value_loss",
    "compute_lambda_returns",
    "compute_policy_loss",
    "compute_policy_loss_from_logits",
    "compute_preference_loss",
    "compute_retrace",
    "compute_token_logprobs",
    "compute_vtrace",
]
