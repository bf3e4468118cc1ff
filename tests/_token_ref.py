"""Plain 64-bit forms of the token-level policy operators (CPU), written from
their formulas; gradients by automatic differentiation in 64 bits."""
import torch

INF = float("inf")


def logprobs(logits, tokens, mask=None, temperature=1.0):
    """(logprobs, entropy) of 64-bit logits; steps with mask 0 give 0."""
    n, t, v = logits.shape
    keep = torch.ones(n, t, dtype=torch.bool) if mask is None else mask != 0
    z = logits / temperature
    z = torch.where(keep[..., None], z, torch.zeros_like(z))
    logp = torch.log_softmax(z, -1)
    tok = torch.where(keep, tokens.long(), torch.zeros_like(tokens.long()))
    lp = logp.gather(2, tok[..., None])[..., 0]
    live = logp > -INF
    safe = torch.where(live, logp, torch.zeros_like(logp))
    h = -(torch.where(live, safe.exp(), torch.zeros_like(safe)) * safe).sum(-1)
    zero = torch.zeros_like(lp)
    return torch.where(keep, lp, zero), torch.where(keep, h, zero)


def reduce(terms, keep, reduction):
    terms = torch.where(keep, terms, torch.zeros_like(terms))
    count = keep.sum(1)
    if reduction == "sum":
        return terms.sum()
    if reduction == "token":
        return terms.sum() / max(int(count.sum()), 1)
    some = count > 0
    return (terms.sum(1) / count.clamp(min=1)).sum() / max(int(some.sum()), 1)


def policy(lp, old, adv, mask=None, ref=None, clip_low=0.2, clip_high=None, dual_clip=None, kl_coef=0.0, kl="k3",
           reduction="token", entropy=None, entropy_coef=0.0):
    """(loss, dict of statistics)."""
    keep = torch.ones(lp.shape, dtype=torch.bool) if mask is None else mask != 0
    zero = torch.zeros_like(lp)
    high = clip_low if clip_high is None else clip_high
    adv = adv[:, None].expand_as(lp) if adv.dim() == 1 else adv
    old, adv = torch.where(keep, old, zero), torch.where(keep, adv, zero)
    lr = torch.where(keep, lp, zero) - old
    r = lr.exp()
    free, held = r * adv, r.clamp(1 - clip_low, 1 + high) * adv
    term = -torch.minimum(free, held)
    clipped = free > held
    if dual_clip is not None:
        cap = -dual_clip * adv
        over = (adv < 0) & (term > cap)
        term, clipped = torch.where(over, cap, term), clipped | over
    est = zero
    if ref is not None:
        x = torch.where(keep, ref, zero) - torch.where(keep, lp, zero)
        est = {"k1": -x, "k2": 0.5 * x * x, "k3": torch.expm1(x) - x}[kl]
        term = term + kl_coef * est
    if entropy is not None:
        term = term - entropy_coef * torch.where(keep, entropy, zero)
    n = max(int(keep.sum()), 1)
    mean = lambda a: float(torch.where(keep, a.double(), zero).sum() / n)  # noqa: E731
    stats = {"kl": mean(est), "approx_kl": mean(torch.expm1(lr) - lr), "clip_fraction": mean(clipped),
             "num_steps": float(keep.sum())}
    if entropy is not None:
        stats["entropy"] = mean(entropy)
    return reduce(term, keep, reduction), stats


def preference(chosen, rejected, refs=(None, None), masks=(None, None), beta=0.1, loss="sigmoid", smoothing=0.0,
               normalized=False):
    scores = []
    for lp, ref, mask in zip((chosen, rejected), refs, masks):
        keep = torch.ones(lp.shape, dtype=torch.bool) if mask is None else mask != 0
        zero = torch.zeros_like(lp)
        x = torch.where(keep, lp, zero)
        if ref is not None and ref.dim() == 2:
            x = x - torch.where(keep, ref, zero)
        s = x.sum(1)
        if ref is not None and ref.dim() == 1:
            s = s - ref
        scores.append(s / keep.sum(1).clamp(min=1) if normalized else s)
    gap = scores[0] - scores[1]
    if loss == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        term = -(1 - smoothing) * ls(beta * gap) - smoothing * ls(-beta * gap)
    elif loss == "ipo":
        term = (gap - 1 / (2 * beta)) ** 2
    else:
        term = (1 - beta * gap).clamp(min=0)
    return (term.mean() if len(term) else term.sum()), beta * scores[0], beta * scores[1]
