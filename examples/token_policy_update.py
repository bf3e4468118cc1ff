"""Training steps of a small token policy with the package's operators: roll
out, score, estimate advantages, update; then a preference step.

    python examples/token_policy_update.py [--steps K] [--envs N] [--length T] [--vocab V]

The task: a token at or above half the vocabulary earns 1.  Every row starts
with a prompt and ends with padding (mask 0).  Per step:

  1. sample responses; their log-probabilities under the policy that sampled
     them, and under the frozen reference  (compute_token_logprobs)
  2. advantages over the response tokens     (compute_gae_obs_skip)
  3. clipped policy loss with a KL term and an entropy bonus, from the logits
     (compute_policy_loss_from_logits), and the optimizer step
  4. a preference step: for each pair of responses the one with the higher
     reward is preferred                     (compute_preference_loss)
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "rl-triton_b200"))

import rl_triton  # noqa: E402


class Policy(torch.nn.Module):
    """Logits of the next token, and a value, from the token before."""

    def __init__(self, vocab, width=64):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, width)
        self.mix = torch.nn.Linear(width, width)
        self.head = torch.nn.Linear(width, vocab)
        self.value = torch.nn.Linear(width, 1)

    def forward(self, tokens):
        h = torch.tanh(self.mix(self.embed(tokens)))
        return self.head(h), self.value(h)[..., 0]


@torch.no_grad()
def rollout(policy, envs, length, vocab, gen):
    """Tokens [envs, length + 1] (the first is the start), the mask of the
    response steps and their rewards."""
    dev = next(policy.parameters()).device
    tokens = torch.randint(0, vocab, (envs, 1), device=dev, generator=gen)
    for _ in range(length):
        logits, _ = policy(tokens[:, -1])
        tokens = torch.cat([tokens, torch.multinomial(logits.softmax(-1), 1, generator=gen)], 1)
    at = torch.arange(length, device=dev)
    ends = torch.randint(length // 2 + 1, length + 1, (envs, 1), device=dev, generator=gen)
    mask = (at >= length // 8) & (at < ends)
    rewards = (tokens[:, 1:] >= vocab // 2).float() * mask
    return tokens, mask, rewards


def main(steps=20, envs=64, length=32, vocab=2048, seed=0, out=print):
    torch.manual_seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    policy = Policy(vocab).cuda()
    reference = Policy(vocab).cuda()
    reference.load_state_dict(policy.state_dict())
    opt = torch.optim.Adam(policy.parameters(), lr=2e-2)
    history = []
    for step in range(steps):
        tokens, mask, rewards = rollout(policy, envs, length, vocab, gen)
        before, taken = tokens[:, :-1], tokens[:, 1:]
        with torch.no_grad():
            logits, values = policy(before)
            old = rl_triton.compute_token_logprobs(logits, taken, mask)
            ref = rl_triton.compute_token_logprobs(reference(before)[0], taken, mask)
            adv, returns = rl_triton.compute_gae_obs_skip(rewards, values, mask, gamma=0.9, lambda_=0.9)
            adv = (adv - adv[mask].mean()) / (adv[mask].std() + 1e-6)
        for _ in range(4):
            logits, values = policy(before)
            loss, _, stats = rl_triton.compute_policy_loss_from_logits(
                logits, taken, old, adv, mask, ref, clip_low=0.2, clip_high=0.28, kl_coef=0.01, entropy_coef=1e-3,
                return_stats=True)
            value_loss = ((values - returns)[mask] ** 2).mean()
            opt.zero_grad()
            (loss + 0.5 * value_loss).backward()
            opt.step()

        # pairs of responses: the better one first
        score = (rewards.sum(1) / mask.sum(1)).view(2, -1)
        better = score[0] >= score[1]
        rows = torch.arange(envs, device="cuda").view(2, -1)
        order = torch.cat([torch.where(better, rows[0], rows[1]), torch.where(better, rows[1], rows[0])])
        logprobs = rl_triton.compute_token_logprobs(policy(before[order])[0], taken[order], mask[order])
        pref, good, bad = rl_triton.compute_preference_loss(logprobs, ref[order], mask[order], beta=0.1)
        opt.zero_grad()
        (0.1 * pref).backward()
        opt.step()
        history.append(dict(reward=float(rewards.sum() / mask.sum()), loss=float(loss.detach()), kl=float(stats["kl"]),
                            entropy=float(stats["entropy"]), preference=float(pref.detach()),
                            margin=float((good - bad).mean())))
        out(f"step {step}: " + ", ".join(f"{k} {v:.4f}" for k, v in history[-1].items()))
    return history


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--envs", type=int, default=64)
    ap.add_argument("--length", type=int, default=32)
    ap.add_argument("--vocab", type=int, default=2048)
    a = ap.parse_args()
    main(a.steps, a.envs, a.length, a.vocab)
