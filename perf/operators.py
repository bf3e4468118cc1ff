"""The token-level policy operators: what they are timed on and checked against.

    log-probabilities (and entropies) of the tokens taken, from the policy's logits
    the clipped policy loss with a KL term, from log-probabilities or from the logits
    the paired preference loss, from log-probabilities or from the logits

Each case is one call (with its gradient where a training step takes one) of
real size.  run() computes it with elementary torch operations in 32 bits, or,
where `own` is set, through the rl_triton package.
"""
import math
import os
import sys

import torch

own = False

_CLIP_LOW, _CLIP_HIGH = 0.2, 0.28


def _package():
    """The package lies in rl-triton_b200/ beside this folder."""
    at = os.path.join(os.getcwd(), "rl-triton_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import rl_triton
    return rl_triton


# ---------------------------------------------------------------------------
# Cases.  op: logprobs | policy_logits | policy | preference | preference_logits
# envs, steps, vocab: logits [envs, steps, vocab] (for the preference loss envs
#   counts the pairs); dtype: of the logits (log-probabilities are float32)
# mask: none | ragged (responses of random length between a prompt and padding,
#   one row in 8 left empty)
# pad: last columns of the vocabulary that are -inf (a padded head)
# ---------------------------------------------------------------------------
def listed():
    return [
        # one sampled token of one sequence, scored as it is generated: latency
        dict(name="logprobs_one_token", op="logprobs", envs=1, steps=1, vocab=131072, dtype="bf16", train=False,
             entropy=True, mask="none", pad=0),
        # old / reference log-probabilities of a rollout batch before the update
        dict(name="logprobs_score", op="logprobs", envs=16, steps=512, vocab=131072, dtype="bf16", train=False,
             entropy=False, mask="ragged", pad=0),
        # log-probabilities and entropies with their gradient, odd sizes, a padded head
        dict(name="logprobs_train_odd", op="logprobs", envs=3, steps=341, vocab=50021, dtype="fp32", train=True,
             entropy=True, mask="ragged", pad=21),
        # a discrete-control batch: the benchmark's 4096 x 128 rollout with 18 actions
        dict(name="logprobs_actions", op="logprobs", envs=4096, steps=128, vocab=18, dtype="fp32", train=True,
             entropy=True, mask="none", pad=0),
        # the update of a language-model policy: loss and gradient from the logits
        dict(name="policy_logits_large", op="policy_logits", envs=8, steps=1024, vocab=131072, dtype="bf16",
             mask="ragged", pad=0, ref=True, entropy_coef=0.0, dual_clip=0.0, reduction="token", per_row_adv=True),
        # the same with an entropy bonus at odd sizes, averaged by sequence
        dict(name="policy_logits_odd", op="policy_logits", envs=5, steps=397, vocab=32003, dtype="bf16",
             mask="ragged", pad=3, ref=True, entropy_coef=0.01, dual_clip=3.0, reduction="sequence",
             per_row_adv=False),
        # a discrete-control update on the benchmark's rollout size
        dict(name="policy_logits_actions", op="policy_logits", envs=4096, steps=128, vocab=18, dtype="fp32",
             mask="none", pad=0, ref=False, entropy_coef=0.01, dual_clip=0.0, reduction="token", per_row_adv=False),
        # a small minibatch whose log-probabilities are at hand: latency
        dict(name="policy_small", op="policy", envs=8, steps=128, mask="ragged", ref=True, dual_clip=0.0,
             reduction="token", per_row_adv=True),
        # a whole batch of log-probabilities
        dict(name="policy_batch", op="policy", envs=4096, steps=2048, mask="ragged", ref=True, dual_clip=3.0,
             reduction="sequence", per_row_adv=False),
        # a few pairs of short responses: latency
        dict(name="preference_small", op="preference", envs=4, steps=257, mask="ragged", loss="sigmoid",
             smoothing=0.0, normalized=False),
        # a large batch of pairs
        dict(name="preference_batch", op="preference", envs=512, steps=4096, mask="ragged", loss="ipo",
             smoothing=0.0, normalized=True),
        # a preference step from the logits of both responses to their gradient
        dict(name="preference_logits", op="preference_logits", envs=4, steps=512, vocab=65536, dtype="bf16",
             mask="ragged", pad=0, loss="sigmoid", smoothing=0.1, normalized=False),
    ]


_MOST_LOGIT_BYTES = 1.6e9  # of a drawn case; the largest listed one has 2.1e9


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "policy_logits", "policy_logits", "policy", "preference",
                     "preference_logits"])
    mask = rng.choice(["none", "ragged"])
    if op == "policy":
        envs = _log_int(rng, 1, 4096)
        return dict(op=op, envs=envs, steps=_log_int(rng, 1, min(131072, (1 << 23) // envs)), mask=mask,
                    ref=rng.random() < 0.6, dual_clip=rng.choice([0.0, 3.0]),
                    reduction=rng.choice(["token", "sequence", "sum"]), per_row_adv=rng.random() < 0.5)
    pref = dict(loss=rng.choice(["sigmoid", "ipo", "hinge"]), smoothing=0.0, normalized=rng.random() < 0.5)
    if pref["loss"] == "sigmoid":
        pref["smoothing"] = rng.choice([0.0, 0.1])
    if op == "preference":
        envs = _log_int(rng, 1, 512)
        return dict(op=op, envs=envs, steps=_log_int(rng, 1, min(131072, (1 << 21) // envs)), mask=mask, **pref)
    dtype = rng.choice(["bf16", "fp32"])
    size = 2 if dtype == "bf16" else 4
    vocab = _log_int(rng, 2, 262144)
    rows = max(2, min(1 << 20, int(_MOST_LOGIT_BYTES / (size * vocab))))
    if op == "preference_logits":
        rows //= 2
    steps = _log_int(rng, 1, min(8192, rows))
    envs = _log_int(rng, 1, min(4096, max(1, rows // steps)))
    c = dict(op=op, envs=envs, steps=steps, vocab=vocab, dtype=dtype, mask=mask,
             pad=rng.choice([0, min(vocab // 4, 7)]))
    if op == "logprobs":
        return dict(c, train=rng.random() < 0.6, entropy=rng.random() < 0.5)
    if op == "policy_logits":
        return dict(c, ref=rng.random() < 0.6, entropy_coef=rng.choice([0.0, 0.01]), dual_clip=rng.choice([0.0, 3.0]),
                    reduction=rng.choice(["token", "sequence", "sum"]), per_row_adv=rng.random() < 0.5)
    return dict(c, **pref)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _mask(case, rows, g):
    """Prompt, response, padding: the response starts in the first quarter and
    ends in the last half; one row in 8 has none."""
    n, t = rows, case["steps"]
    if case["mask"] == "none":
        return None
    first = (torch.rand(n, 1, device="cuda", generator=g) * 0.25 * t).floor()
    last = ((0.5 + 0.5 * torch.rand(n, 1, device="cuda", generator=g)) * t).ceil()
    at = torch.arange(t, device="cuda")[None, :]
    m = (at >= first) & (at < last)
    m[torch.arange(n, device="cuda") % 8 == 7] = False
    return m


def _logits(case, rows, g):
    """Logits with one likely token per step (the sampled one, mostly), and the
    tokens' log-probabilities under them."""
    n, t, v = rows, case["steps"], case["vocab"]
    live = v - case["pad"]
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    x = torch.randn(n, t, v, device="cuda", dtype=dtype, generator=g).mul_(2.0)
    tok = torch.randint(0, live, (n, t), device="cuda", generator=g)
    boost = (math.log(live) + 2.0 * torch.randn(n, t, device="cuda", generator=g)).to(dtype)
    x.scatter_add_(2, tok[..., None], boost[..., None])
    if case["pad"]:
        x[..., live:] = float("-inf")
    lse = torch.stack([torch.logsumexp(row.float(), dim=-1) for row in x])
    lp = torch.gather(x, 2, tok[..., None])[..., 0].float() - lse
    return x, tok, lp


def _behind(lp, spread, g):
    """Log-probabilities of a policy near the one that gives lp."""
    return (lp + spread * torch.randn(lp.shape, device="cuda", generator=g)).clamp_(max=-1e-4)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, n, t = case["op"], case["envs"], case["steps"]
    s = dict(case=case)
    rows = 2 * n if op in ("preference", "preference_logits") else n  # chosen rows first, then rejected ones
    if op.endswith("logits") or op == "logprobs":
        s["logits"], s["tokens"], lp = _logits(case, rows, g)
    else:
        lp = -torch.empty(rows, t, device="cuda").exponential_(0.8, generator=g) - 1e-3
    s["mask"] = _mask(case, rows, g)
    if op == "logprobs":
        s["g_lp"] = torch.randn(n, t, device="cuda", generator=g)
        s["g_h"] = 0.01 * torch.randn(n, t, device="cuda", generator=g)
    if op in ("policy", "policy_logits"):
        s["old"] = _behind(lp, 0.15, g)
        s["ref"] = _behind(lp, 0.3, g) if case["ref"] else None
        s["adv"] = 0.4 + torch.randn((n,) if case["per_row_adv"] else (n, t), device="cuda", generator=g)
    if op in ("preference", "preference_logits"):
        s["ref"] = _behind(lp, 0.1, g)
    if op in ("policy", "preference"):
        s["lp"] = lp
    return s


# ---------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------
def _run_own(s):
    rl, c = _package(), s["case"]
    op, n = c["op"], c["envs"]
    if c.get("train", True):
        s["logits" if "logits" in s else "lp"].requires_grad_(True)
    if op == "logprobs":
        out = rl.compute_token_logprobs(s["logits"], s["tokens"], s["mask"], return_entropy=c["entropy"])
        if not c["train"]:
            return out
        outs, ups = (out, (s["g_lp"], s["g_h"])) if c["entropy"] else ((out,), (s["g_lp"],))
        (grad,) = torch.autograd.grad(outs, s["logits"], ups)
        return [o.detach() for o in outs] + [grad]
    kw = {}
    if op in ("policy", "policy_logits"):
        kw = dict(mask=s["mask"], ref_logprobs=s["ref"], clip_low=_CLIP_LOW, clip_high=_CLIP_HIGH,
                  dual_clip=c["dual_clip"] or None, kl_coef=0.05 if c["ref"] else 0.0, reduction=c["reduction"])
    if op == "policy":
        loss = rl.compute_policy_loss(s["lp"], s["old"], s["adv"], **kw)
        (grad,) = torch.autograd.grad(loss, s["lp"])
        return loss.detach(), grad
    if op == "policy_logits":
        loss, lp = rl.compute_policy_loss_from_logits(s["logits"], s["tokens"], s["old"], s["adv"],
                                                      entropy_coef=c["entropy_coef"], **kw)
        (grad,) = torch.autograd.grad(loss, s["logits"])
        return loss.detach(), lp.detach(), grad
    m, ref = s["mask"], s["ref"]
    lp = s["lp"] if op == "preference" else rl.compute_token_logprobs(s["logits"], s["tokens"], m)
    loss, good, bad = rl.compute_preference_loss(lp, ref, m, beta=0.1, loss=c["loss"],
                                                 label_smoothing=c["smoothing"], length_normalized=c["normalized"])
    (grad,) = torch.autograd.grad(loss, s["lp"] if op == "preference" else s["logits"])
    return loss.detach(), good, bad, grad


# ---------------------------------------------------------------------------
# The plain form: 32 bits, elementary operations, gradients from the formulas
# ---------------------------------------------------------------------------
def _log_softmax(logits):
    z = logits.float()
    z = z - z.amax(-1, keepdim=True)
    return z - z.exp().sum(-1, keepdim=True).log()


def _taken(logp, tokens, m):
    lp = torch.gather(logp, 2, tokens[..., None])[..., 0]
    return lp if m is None else torch.where(m, lp, 0.0)


def _entropy(logp, p, m):
    h = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    return h if m is None else torch.where(m, h, 0.0)


def _logits_grad(logp, p, tokens, g_lp, g_h, h, m, dtype):
    """g_lp (1[token] - p) - g_h p (log p + H), zero where the mask is."""
    w = g_lp[..., None] if g_h is None else g_lp[..., None] + g_h[..., None] * torch.where(p > 0, logp + h[..., None],
                                                                                          0.0)
    d = -p * w
    d.scatter_add_(2, tokens[..., None], g_lp[..., None])
    if m is not None:
        d = torch.where(m[..., None], d, 0.0)
    return d.to(dtype)


def _weights(m, shape, reduction):
    """What each step's term counts for in the loss."""
    keep = torch.ones(shape, device="cuda") if m is None else m.float()
    if reduction == "sum":
        return keep
    if reduction == "token":
        return keep / keep.sum().clamp(min=1.0)
    each = keep.sum(1, keepdim=True)
    return keep / each.clamp(min=1.0) / (each > 0).float().sum().clamp(min=1.0)


def _policy_terms(c, s, lp):
    """Each step's loss term and its derivative by the log-probability."""
    adv = s["adv"][:, None] if c["per_row_adv"] else s["adv"]
    ratio = (lp - s["old"]).exp()
    free = ratio * adv
    held = ratio.clamp(1.0 - _CLIP_LOW, 1.0 + _CLIP_HIGH) * adv
    term = -torch.minimum(free, held)
    d = torch.where(free <= held, -free, 0.0)
    if c["dual_clip"]:
        cap = -c["dual_clip"] * adv
        over = (adv < 0) & (term > cap)
        term, d = torch.where(over, cap, term), torch.where(over, 0.0, d)
    if c["ref"]:
        x = s["ref"] - lp
        term = term + 0.05 * (x.exp() - x - 1.0)
        d = d + 0.05 * (1.0 - x.exp())
    return term, d


def _policy_plain(s):
    c = s["case"]
    w = _weights(s["mask"], s["old"].shape, c["reduction"])
    if c["op"] == "policy":
        term, d = _policy_terms(c, s, s["lp"])
        return torch.where(w > 0, w * term, 0.0).sum(), torch.where(w > 0, w * d, 0.0)
    logp = _log_softmax(s["logits"])
    p = logp.exp()
    lp = _taken(logp, s["tokens"], s["mask"])
    term, d = _policy_terms(c, s, lp)
    h = g_h = None
    if c["entropy_coef"]:
        h = _entropy(logp, p, s["mask"])
        term, g_h = term - c["entropy_coef"] * h, -c["entropy_coef"] * w
    return (torch.where(w > 0, w * term, 0.0).sum(), lp,
            _logits_grad(logp, p, s["tokens"], w * d, g_h, h, s["mask"], s["logits"].dtype))


def _preference_plain(s):
    c, n, m = s["case"], s["case"]["envs"], s["mask"]
    if c["op"] == "preference_logits":
        logp = _log_softmax(s["logits"])
        lp = _taken(logp, s["tokens"], m)
    else:
        lp = s["lp"]
    keep = torch.ones_like(lp) if m is None else m.float()
    each = keep.sum(1).clamp(min=1.0) if c["normalized"] else torch.ones_like(keep[:, 0])
    score = torch.where(keep > 0, lp - s["ref"], 0.0).sum(1) / each
    beta, margin = 0.1, score[:n] - score[n:]
    x = beta * margin
    if c["loss"] == "sigmoid":
        e = c["smoothing"]
        down = torch.log1p((-x.abs()).exp())
        term = (1.0 - e) * (down - x.clamp(max=0.0)) + e * (down + x.clamp(min=0.0))
        d = beta * (1.0 / (1.0 + (-x).exp()) - (1.0 - e))
    elif c["loss"] == "ipo":
        term, d = (margin - 0.5 / beta) ** 2, 2.0 * (margin - 0.5 / beta)
    else:
        term, d = (1.0 - x).clamp(min=0.0), torch.where(x < 1.0, -beta, 0.0)
    d = torch.cat([d, -d]) / n / each
    grad = keep * d[:, None]
    if c["op"] == "preference_logits":
        grad = _logits_grad(logp, logp.exp(), s["tokens"], grad, None, None, m, s["logits"].dtype)
    return term.sum() / n, beta * score[:n], beta * score[n:], grad


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["op"] in ("policy", "policy_logits"):
        return _policy_plain(state)
    if c["op"] in ("preference", "preference_logits"):
        return _preference_plain(state)
    logp = _log_softmax(state["logits"])
    outs = [_taken(logp, state["tokens"], state["mask"])]
    p = logp.exp() if c["train"] or c["entropy"] else None
    if c["entropy"]:
        outs.append(_entropy(logp, p, state["mask"]))
    if c["train"]:
        outs.append(_logits_grad(logp, p, state["tokens"], state["g_lp"], state["g_h"] if c["entropy"] else None,
                                 outs[-1], state["mask"], state["logits"].dtype))
    return outs if len(outs) > 1 else outs[0]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op, n, t = case["op"], case["envs"], case["steps"]
    rows = (2 * n if op in ("preference", "preference_logits") else n) * t
    keep = 1 if case["mask"] == "ragged" else 0  # bytes of the mask
    tokens = rows * keep
    if op in ("policy", "policy_logits"):
        tokens += rows * 4 * (1 + int(case["ref"])) + 4 * (n if case["per_row_adv"] else rows)
    if op in ("preference", "preference_logits"):
        tokens += rows * 4 + 8 * n
    if op in ("policy", "preference"):
        return {"bytes": tokens + 8 * rows, "flops": 30 * rows}
    size = 2 if case["dtype"] == "bf16" else 4
    cells = rows * case["vocab"]
    train = case.get("train", True)
    # a masked step's logits need not be read (its gradient is zeros): by _mask(),
    # half of a row plus an eighth is kept on average
    seqs = rows // t
    read = 0.625 * (1 - (seqs // 8) / seqs) if keep else 1.0
    tokens += 8 * rows + (4 * rows if op != "preference_logits" else 0)
    if op == "logprobs":
        tokens += 4 * rows * int(case["entropy"]) + (4 * rows * (1 + int(case["entropy"])) if train else 0)
    return {"bytes": tokens + cells * size * (read + int(train)),
            "flops": cells * read * (9 if train else 4) + 30 * rows}


# ---------------------------------------------------------------------------
# The definitions in 64 bits; gradients by differentiation
# ---------------------------------------------------------------------------
def _exact_logprobs(logits, tokens, m, entropy):
    lsm = torch.log_softmax(logits, dim=-1)
    lp = lsm.gather(2, tokens.unsqueeze(2)).squeeze(2)
    h = None
    if entropy:
        finite = torch.isfinite(logits)
        h = -(lsm.exp() * lsm.masked_fill(~finite, 0.0)).sum(dim=2)
    if m is not None:
        lp = lp.masked_fill(~m, 0.0)
        h = None if h is None else h.masked_fill(~m, 0.0)
    return lp, h


def _exact_mean(terms, m, reduction):
    if m is not None:
        terms = terms.masked_fill(~m, 0.0)
    count = torch.full(terms.shape[:1], terms.shape[1], dtype=torch.float64, device=terms.device) if m is None \
        else m.sum(dim=1).double()
    if reduction == "sum":
        return terms.sum()
    if reduction == "token":
        return terms.sum() / max(float(count.sum()), 1.0)
    some = count > 0
    return (terms.sum(dim=1)[some] / count[some]).sum() / max(int(some.sum()), 1)


def _exact_policy(c, s, lp, h):
    old, adv = s["old"].double(), s["adv"].double()
    adv = adv.unsqueeze(1) if c["per_row_adv"] else adv
    r = torch.exp(lp - old)
    gain = torch.where(adv >= 0, adv * torch.clamp(r, max=1 + _CLIP_HIGH), adv * torch.clamp(r, min=1 - _CLIP_LOW))
    if c["dual_clip"]:
        gain = torch.where(adv < 0, torch.maximum(gain, c["dual_clip"] * adv), gain)
    terms = -gain
    if c["ref"]:
        away = s["ref"].double() - lp
        terms = terms + 0.05 * (torch.expm1(away) - away)
    if h is not None:
        terms = terms - c["entropy_coef"] * h
    return _exact_mean(terms, s["mask"], c["reduction"])


def _exact_preference(c, s, lp):
    m, n = s["mask"], c["envs"]
    rel = lp - s["ref"].double()
    if m is not None:
        rel = rel.masked_fill(~m, 0.0)
    score = rel.sum(dim=1)
    if c["normalized"]:
        score = score / (rel.shape[1] if m is None else m.sum(dim=1).clamp(min=1))
    good, bad = score[:n], score[n:]
    gap = good - bad
    if c["loss"] == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        each = -(1 - c["smoothing"]) * ls(0.1 * gap) - c["smoothing"] * ls(-0.1 * gap)
    elif c["loss"] == "ipo":
        each = (gap - 5.0).square()
    else:
        each = torch.relu(1 - 0.1 * gap)
    return each.mean(), 0.1 * good, 0.1 * bad


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    train = case.get("train", True)
    if "lp" in s:
        x = lp = s["lp"].detach().double().requires_grad_(True)
        h = None
    else:
        x = s["logits"].detach().double().requires_grad_(train)
        s["logits"] = None
        lp, h = _exact_logprobs(x, s["tokens"], s["mask"], case.get("entropy") or case.get("entropy_coef"))
    if op == "logprobs":
        outs = [lp] if h is None else [lp, h]
        if train:
            ups = [s["g_lp"].double()] + ([] if h is None else [s["g_h"].double()])
            outs = outs + list(torch.autograd.grad(outs, x, ups))
        outs = [o.detach() for o in outs]
        return outs if len(outs) > 1 else outs[0]
    if op in ("policy", "policy_logits"):
        loss = _exact_policy(case, s, lp, h)
        (grad,) = torch.autograd.grad(loss, x)
        return (loss.detach(), grad) if op == "policy" else (loss.detach(), lp.detach(), grad)
    loss, good, bad = _exact_preference(case, s, lp)
    (grad,) = torch.autograd.grad(loss, x)
    return loss.detach(), good.detach(), bad.detach(), grad
