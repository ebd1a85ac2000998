"""64-bit definitions of the token-policy operators and of the AdamW step, for the tests."""

import torch

NEG_INF = float("-inf")


def rows(logits, tokens, counted, temperature):
    """Per row (log-probabilities of every column, logp, entropy) in 64 bits; rows that do not count are computed on
    zeros. Differentiable."""
    z = torch.where(counted[..., None], logits.double(), 0.0) / temperature
    log_p = torch.log_softmax(z, -1)
    logp = log_p.gather(-1, tokens.long().clamp(0, logits.shape[-1] - 1)[..., None])[..., 0]
    plogp = torch.where(log_p == NEG_INF, 0.0, log_p.exp() * torch.where(log_p == NEG_INF, 0.0, log_p))
    return log_p, logp, -plogp.sum(-1)


def weights(logits, tokens, mask):
    w = torch.ones(tokens.shape, dtype=torch.float64) if mask is None else mask.double()
    return torch.where((tokens >= 0) & (tokens < logits.shape[-1]), w, 0.0)


def policy(logits, tokens, old, adv, ref, mask, *, lo, hi, kl_coef, kind, entropy_coef, temperature, mean=True):
    """(loss, (surrogate, kl, entropy, clip fraction), logp, dL/dlogp, dL/dH) in 64 bits."""
    w = weights(logits, tokens, mask)
    counted = w != 0
    _, logp, entropy = rows(logits, tokens, counted, temperature)
    logp, entropy = logp.detach().requires_grad_(), entropy.detach().requires_grad_()
    ratio = torch.where(counted, logp - old.double(), 0.0).exp()
    adv = torch.where(counted, adv.double(), 0.0)
    free, cut = -adv * ratio, -adv * ratio.clamp(lo, hi)
    surrogate = torch.max(free, cut)
    if ref is None:
        kl = torch.zeros_like(logp)
    else:
        d = torch.where(counted, ref.double() - logp, 0.0)
        kl = {"k1": -d, "k2": d * d / 2, "k3": d.exp() - d - 1}[kind]
    total = w.sum()
    inv = 1 / total if total != 0 else torch.tensor(0.0, dtype=torch.float64)
    loss = (w * (surrogate - entropy_coef * entropy)).sum()
    if kl_coef:
        loss = loss + kl_coef * (w * kl).sum()
    loss = loss * inv if mean else loss
    da, db = torch.autograd.grad(loss, (logp, entropy), allow_unused=True)
    stats = [(inv * (w * x).sum()).item() for x in (surrogate, kl, entropy, (cut > free).double())]
    return loss.item(), stats, torch.where(counted, logp, 0.0).detach(), da, db if db is not None else 0 * da


def preference(logits, tokens, ref, bounds, mask, *, beta, smoothing=0.0, kind="sigmoid", average=False,
               temperature=1.0):
    """``bounds``: (first, last) row of each sequence over the flattened rows."""
    w = weights(logits, tokens, mask).flatten()
    _, logp, _ = rows(logits, tokens, weights(logits, tokens, mask) != 0, temperature)
    logp = logp.detach().flatten().requires_grad_()
    lps = []
    for a, b in bounds:
        s, c = (w[a:b] * logp[a:b]).sum(), w[a:b].sum()
        lps.append(s if not average else s / c if c != 0 else 0 * s)
    lps = torch.stack(lps)
    rewards = beta * (lps - (0 if ref is None else ref.double()))
    h = rewards[0::2] - rewards[1::2]
    sig = torch.nn.functional.logsigmoid
    loss = {"sigmoid": -(1 - smoothing) * sig(h) - smoothing * sig(-h), "hinge": torch.relu(1 - h),
            "ipo": (h / beta - 0.5 / beta) ** 2}[kind].mean()
    da, = torch.autograd.grad(loss, logp)
    return loss.item(), lps.detach(), rewards.detach(), da.view(tokens.shape)


def logits_grad(logits, tokens, counted, temperature, a, b):
    """Gradient of the logits for dL/dlogp = a, dL/dH = b, and a bound of what fp32 arithmetic may add to it.

    The bound: log2 p is a difference of fp32 numbers of its size, so p is off by at most |log p| 2^-21 + 3e-5 relative
    (the second term: the row's log-sum in fp32, of up to 2^17 terms); the products around it add 2^-22."""
    log_p, _, entropy = rows(logits, tokens, counted, temperature)
    p = log_p.exp()
    safe = torch.where(log_p == NEG_INF, 0.0, log_p)
    a, b = torch.where(counted, a, 0.0)[..., None], torch.where(counted, b, 0.0)[..., None]
    onehot = torch.zeros_like(p)
    onehot.scatter_(-1, tokens.long().clamp(0, p.shape[-1] - 1)[..., None], 1.0)
    g = (a * (onehot - p) - b * p * (safe + entropy[..., None])) / temperature
    rel = safe.abs() * 2.0 ** -21 + 3e-5
    size = (a.abs() + b.abs() * (safe.abs() + entropy[..., None])) * p
    bound = (size * rel + b.abs() * p * 3e-5 * (1 + entropy[..., None]) + a.abs() * onehot * 3e-5) / temperature
    return g, bound


def rounding(x, dtype):
    """Half a step of ``dtype`` around ``x``: relative, and the spacing of its subnormal numbers."""
    info = torch.finfo(dtype)
    return x.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2


def logp_bound(logp):
    """|logp| 2^-22 for (z - m) / T and its difference with ln s; 1e-5 for ln s (sum of up to 2^17 fp32 terms, each
    exp2 within 2^-22 of its value and its argument within |d| 2^-23)."""
    return logp.abs() * 2.0 ** -22 + 1e-5


def adamw(p, g, m, v, t, *, lr, betas, eps, weight_decay, clip=1.0):
    """One step in 64 bits: (p, m, v)."""
    g = g.double() * clip
    m = betas[0] * m.double() + (1 - betas[0]) * g
    v = betas[1] * v.double() + (1 - betas[1]) * g * g
    hat_m, hat_v = m / (1 - betas[0] ** t), v / (1 - betas[1] ** t)
    return p.double() * (1 - lr * weight_decay) - lr * hat_m / (hat_v.sqrt() + eps), m, v
