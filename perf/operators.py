"""What is measured of the token-policy operators: log-probabilities, the clipped policy loss, the preference loss and
the AdamW step over many tensors. ``run`` computes a case in its plain form, or calls the framework where ``own``."""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
LOSS_SCALE = {"bf16": 1.0, "fp16": 4096.0, "fp32": 1.0}  # keeps a mean loss's gradients inside fp16's range
NEG_INF = float("-inf")

CLIP, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04
BETA, SMOOTHING = 0.1, 0.05
LR, BETAS, EPS, DECAY, MAX_NORM = 3e-4, (0.9, 0.999), 1e-8, 0.01, 1.0
BLOCK = 256  # elements that share a scale of the 8-bit states, and the alignment of a tensor in the arenas
STEP0, SEED = 10, 7


def listed():
    return [
        # scoring the tokens that a few sequences produced in one decoding step: latency
        {"name": "logprobs, one step", "op": "logprobs", "rows": 4, "batch": 0, "vocab": 131072, "dtype": "bf16",
         "backward": False, "masked": 0.0, "banned": False, "temperature": 0.8},
        # reference log-probabilities of a batch of full sequences (logits shifted by one position, odd vocabulary)
        {"name": "logprobs, reference pass", "op": "logprobs", "rows": 4094, "batch": 2, "vocab": 50001,
         "dtype": "fp32", "backward": False, "masked": 0.1, "banned": False, "temperature": 1.0},
        # log-probabilities and entropies with gradients back to the logits
        {"name": "logprobs with gradient", "op": "logprobs", "rows": 2048, "batch": 0, "vocab": 65536, "dtype": "bf16",
         "backward": True, "masked": 0.0, "banned": True, "temperature": 1.0},
        # a policy minibatch of one short response
        {"name": "policy, short", "op": "policy", "rows": 33, "batch": 0, "vocab": 32000, "dtype": "bf16",
         "entropy": 0.0, "masked": 0.0, "banned": False, "temperature": 1.0},
        # padded responses with prompts masked out, odd vocabulary, shifted rows, entropy bonus
        {"name": "policy, padded", "op": "policy", "rows": 2043, "batch": 9, "vocab": 50001, "dtype": "fp32",
         "entropy": 0.01, "masked": 0.3, "banned": True, "temperature": 0.9},
        # a large minibatch over a large vocabulary
        {"name": "policy, large", "op": "policy", "rows": 8192, "batch": 0, "vocab": 131072, "dtype": "bf16",
         "entropy": 0.001, "masked": 0.1, "banned": False, "temperature": 1.0},
        # one pair of short answers
        {"name": "preference, one pair", "op": "preference", "pairs": 1, "shortest": 20, "longest": 90, "behind": 0,
         "vocab": 32000, "dtype": "bf16"},
        # ragged packed answers, odd vocabulary, rows behind the last sequence
        {"name": "preference, ragged", "op": "preference", "pairs": 6, "shortest": 1, "longest": 400, "behind": 17,
         "vocab": 50001, "dtype": "fp16"},
        # a full preference batch
        {"name": "preference, large", "op": "preference", "pairs": 8, "shortest": 300, "longest": 700, "behind": 0,
         "vocab": 65536, "dtype": "bf16"},
        # the actor and critic of the benchmark (MLPs 512-256-128), clipped
        {"name": "adamw, actor-critic", "op": "adamw", "layout": "mlp", "width": 512, "layers": 3, "dtype": "fp32",
         "bits": 32, "clip": True},
        # many odd tensors of every size, 8-bit states
        {"name": "adamw, ragged 8-bit", "op": "adamw", "layout": "ragged", "width": 2000000, "layers": 150,
         "dtype": "fp32", "bits": 8, "clip": False},
        # a transformer's bf16 weights, 8-bit states, clipped
        {"name": "adamw, blocks 8-bit", "op": "adamw", "layout": "blocks", "width": 1024, "layers": 24,
         "dtype": "bf16", "bits": 8, "clip": True},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "adamw"])
    if op == "adamw":
        layout = rng.choice(["mlp", "ragged", "blocks"])
        width = {"mlp": lambda: _log_uniform(rng, 16, 2048), "ragged": lambda: _log_uniform(rng, 500, 2000000),
                 "blocks": lambda: 8 * _log_uniform(rng, 8, 128)}[layout]()
        layers = {"mlp": lambda: rng.randint(1, 6), "ragged": lambda: _log_uniform(rng, 2, 150),
                  "blocks": lambda: rng.randint(1, 24)}[layout]()
        return {"op": op, "layout": layout, "width": width, "layers": layers, "dtype": rng.choice(["bf16", "fp32"]),
                "bits": rng.choice([8, 32]), "clip": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = _log_uniform(rng, 1000, 131072)
    if rng.random() < 0.5:
        vocab = max(1024, vocab // 1024 * 1024)
    most = 2 ** 29 // vocab  # half of the largest listed case's logits
    if op == "preference":
        pairs = _log_uniform(rng, 1, 16)
        longest = _log_uniform(rng, 2, max(3, min(2000, most // (2 * pairs))))
        return {"op": op, "pairs": pairs, "shortest": rng.randint(1, longest), "longest": longest,
                "behind": rng.choice([0, rng.randint(1, 40)]), "vocab": vocab, "dtype": dtype}
    rows = _log_uniform(rng, 1, min(16384, most))
    batch = rng.choice([0, 0, rng.randint(1, 12)])
    if batch:
        rows = max(1, rows // batch) * batch
    case = {"op": op, "rows": rows, "batch": batch, "vocab": vocab, "dtype": dtype,
            "masked": rng.choice([0.0, rng.uniform(0.05, 0.9)]), "banned": rng.random() < 0.3,
            "temperature": rng.choice([1.0, rng.uniform(0.5, 1.5)])}
    if op == "logprobs":
        return case | {"backward": rng.random() < 0.5}
    return case | {"entropy": rng.choice([0.0, rng.uniform(0.0005, 0.02)])}


# ---- sizes that follow from a case ----------------------------------------------------------------------------------
def _lengths(case):
    r = random.Random(case["pairs"] * 1000003 + case["longest"])
    return [r.randint(case["shortest"], case["longest"]) for _ in range(2 * case["pairs"])]


def _prompts(case):
    """Leading tokens of each sequence that belong to its prompt (no loss)."""
    r = random.Random(case["pairs"] * 7919 + case["longest"])
    return [r.randint(0, n // 2) for n in _lengths(case)]


def _shapes(case):
    width, layers = case["width"], case["layers"]
    if case["layout"] == "mlp":  # an actor and a critic: halving hidden layers, 96 / 99 inputs, 29 actions
        hidden = [max(4, width >> k) for k in range(layers)]
        shapes = [(29,)]
        for inputs, outputs in ((96, 29), (99, 1)):
            sizes = [inputs] + hidden + [outputs]
            for a, b in zip(sizes[:-1], sizes[1:]):
                shapes += [(b, a), (b,)]
        return shapes
    if case["layout"] == "blocks":  # embedding, then attention projections, feed-forward and gains of each block
        block = [(width, width)] * 4 + [(4 * width, width), (width, 4 * width), (width,), (width,)]
        return [(32768, width)] + block * layers + [(width,)]
    r = random.Random(width * 31 + layers)
    return [(int(math.exp(r.uniform(0.0, math.log(width)))),) for _ in range(layers)]


def _places(case):
    """Offset and length of each tensor in the arenas, and the arenas' length."""
    at, places = 0, []
    for shape in _shapes(case):
        n = math.prod(shape)
        places.append((at, n))
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return places, at


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _logits(case, rows, gen):
    """Logits as a model gives them (3-D ones without the last position), the tokens, and their log-probabilities."""
    vocab, batch, dtype = case["vocab"], case.get("batch", 0), DTYPES[case["dtype"]]
    shape = (batch, rows // batch + 1, vocab) if batch else (rows, vocab)
    x = torch.empty(shape, device="cuda", dtype=dtype)
    x.normal_(0.0, 2.0, generator=gen)
    if batch:
        x = x[:, :-1]
    tokens = torch.randint(vocab, x.shape[:-1], device="cuda", generator=gen)
    if case.get("banned"):  # columns that the sampler excludes
        x[..., 5::97] = NEG_INF
        tokens = torch.where(tokens % 97 == 5, tokens - 1, tokens)
    lift = torch.empty(tokens.shape, device="cuda").uniform_(0.0, 12.0, generator=gen)
    picked = x.gather(-1, tokens[..., None])
    x.scatter_(-1, tokens[..., None], (picked.float() + lift[..., None]).to(dtype))
    t = case.get("temperature", 1.0)
    parts = zip(x, tokens) if batch else zip(x.split(512), tokens.split(512))
    logp = torch.cat([torch.log_softmax(part.float() / t, -1).gather(-1, k[:, None])[:, 0] for part, k in parts])
    return x, tokens, logp.view(tokens.shape)


def _noise(like, scale, gen):
    return torch.randn(like.shape, device="cuda", generator=gen) * scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen)
    if case["op"] == "preference":
        lengths = _lengths(case)
        rows = sum(lengths) + case["behind"]
        x, tokens, logp = _logits(case, rows, gen)
        mask = torch.zeros(rows, dtype=torch.bool)
        at, offsets = 0, [0]
        for n, prompt in zip(lengths, _prompts(case)):
            mask[at + prompt:at + n] = True
            at += n
            offsets.append(at)
        mask = mask.cuda()
        sums = torch.stack([(logp * mask)[a:b].sum() for a, b in zip(offsets[:-1], offsets[1:])])
        moved = _noise(sums, 5.0, gen)  # how far training has moved each sequence from the reference
        return {"case": case, "logits": x, "tokens": tokens, "mask": mask,
                "offsets": torch.tensor(offsets, device="cuda"), "ref": sums - moved - 5 * moved.sign()}
    x, tokens, logp = _logits(case, case["rows"], gen)
    state = {"case": case, "logits": x, "tokens": tokens, "mask": None}
    if case["masked"]:
        state["mask"] = torch.rand(tokens.shape, device="cuda", generator=gen) >= case["masked"]
    if case["op"] == "policy":
        moved = _noise(logp, 0.2, gen)
        return state | {"old": logp + _noise(logp, 0.15, gen), "ref": logp + moved + 0.2 * moved.sign(),
                        "adv": _noise(logp, 1.0, gen) + 0.5}
    if case["backward"]:
        state |= {"dlogp": _noise(logp, 1.0, gen), "dentropy": _noise(logp, 0.1, gen)}
    return state


def _prepare_adamw(case, gen):
    places, total = _places(case)
    dtype = DTYPES[case["dtype"]]
    inside = torch.zeros(total, dtype=torch.bool)
    for at, n in places:
        inside[at:at + n] = True
    inside = inside.cuda()

    def fill(scale):
        return torch.randn(total, device="cuda", generator=gen) * inside * scale

    arena = {"p": fill(0.02).to(dtype), "g": fill(1e-3).to(dtype)}
    if case["dtype"] == "bf16":  # the 16 bits of the fp32 weight below its bf16 rounding
        low = torch.randint(-32768, 32768, (total,), device="cuda", generator=gen)
        arena["low"] = (low * (arena["p"] != 0)).to(torch.int16)  # with a zero, negative ones would not be a number
    if case["bits"] == 32:
        arena |= {"m": fill(3e-4), "v": fill(1e-3).square()}
    else:
        scales = torch.empty(2, total // BLOCK, device="cuda").uniform_(0.5, 2.0, generator=gen)
        arena |= {"m": fill(100.0).clamp(-448, 448).to(torch.float8_e4m3fn),
                  "v": fill(150.0).abs().clamp(0, 448).to(torch.float8_e4m3fn),
                  "m_scale": scales[0] * 3e-6, "v_scale": scales[1] * 5e-6}
    steps = torch.full((len(places),), float(STEP0), device="cuda")
    return {"case": case, "arena": arena, "steps": steps}


# ---- plain forms --------------------------------------------------------------------------------------------------------
def _rows_plain(x, tokens, temperature):
    """Log-probability of the tokens, entropy, and (probabilities, log-probabilities) of every column."""
    z = x.float() / temperature
    z -= z.amax(-1, keepdim=True)
    p = z.exp()
    total = p.sum(-1, keepdim=True)
    z -= total.log()  # log-probabilities
    p /= total
    logp = z.gather(-1, tokens[..., None])[..., 0]
    entropy = -(p * z.clamp(min=-3e38)).sum(-1)
    return logp, entropy, p, z


def _grad_plain(p, z, tokens, entropy, a, b, temperature, dtype):
    """``(a (onehot - p) - b p (log p + H)) / temperature`` in the type of the logits."""
    grad = z.clamp_(min=-3e38)
    grad += entropy[..., None]
    grad *= -b[..., None]
    grad -= a[..., None]
    grad *= p
    grad.scatter_add_(-1, tokens[..., None], a[..., None])
    return (grad / temperature).to(dtype)


def _logprobs_plain(s):
    case = s["case"]
    t = case["temperature"]
    logp, entropy, p, z = _rows_plain(s["logits"], s["tokens"], t)
    active = torch.ones_like(logp) if s["mask"] is None else s["mask"].float()
    out = {"logp": logp * active, "entropy": entropy * active}
    if case["backward"]:
        out["grad"] = _grad_plain(p, z, s["tokens"], entropy, s["dlogp"] * active, s["dentropy"] * active, t,
                                  s["logits"].dtype)
    return out


def _policy_plain(s):
    case = s["case"]
    t, ent = case["temperature"], case["entropy"]
    logp, entropy, p, z = _rows_plain(s["logits"], s["tokens"], t)
    w = torch.ones_like(logp) if s["mask"] is None else s["mask"].float()
    w = w / w.double().sum().clamp(min=1e-30).float()
    ratio = (logp - s["old"]).exp()
    free, cut = -s["adv"] * ratio, -s["adv"] * ratio.clamp(1 - CLIP, 1 + CLIP_HIGH)
    open_ = ((ratio >= 1 - CLIP) & (ratio <= 1 + CLIP_HIGH)) | (free > cut)
    far = s["ref"] - logp
    surrogate, kl = torch.maximum(free, cut), far.exp() - far - 1
    parts = torch.stack([surrogate, kl, entropy, (cut > free).float()]).double()
    surrogate, kl, ent_mean, clipped = (parts * w.double()).flatten(1).sum(1).unbind()
    scaled = w * LOSS_SCALE[case["dtype"]]
    a = scaled * (torch.where(open_, free, 0.0) + KL_COEF * (1 - far.exp()))
    grad = _grad_plain(p, z, s["tokens"], entropy, a, -ent * scaled, t, s["logits"].dtype)
    loss = surrogate + KL_COEF * kl - ent * ent_mean
    return {"loss": loss.float(), "surrogate": surrogate.float(), "kl": kl.float(), "entropy": ent_mean.float(),
            "clip_fraction": clipped.float(), "logp": logp * (w > 0), "grad": grad}


def _preference_plain(s):
    case = s["case"]
    logp, entropy, p, z = _rows_plain(s["logits"], s["tokens"], 1.0)
    seq = torch.bucketize(torch.arange(len(logp), device="cuda"), s["offsets"][1:], right=True)
    active = s["mask"] & (seq < 2 * case["pairs"])
    seq = seq.clamp(max=2 * case["pairs"] - 1)
    sums = torch.zeros(2 * case["pairs"], dtype=torch.float64, device="cuda")
    sums.index_add_(0, seq, torch.where(active, logp, 0.0).double())
    reward = BETA * (sums - s["ref"].double())
    h = reward[0::2] - reward[1::2]
    loss = ((1 - SMOOTHING) * torch.log1p((-h.abs()).exp()) + SMOOTHING * torch.log1p((-h.abs()).exp())
            + (1 - SMOOTHING) * (-h).clamp(min=0) + SMOOTHING * h.clamp(min=0)).mean()
    dh = (SMOOTHING / (1 + (-h).exp()) - (1 - SMOOTHING) / (1 + h.exp())) / case["pairs"]
    dh = dh * BETA * LOSS_SCALE[case["dtype"]]
    a = torch.where(active, torch.stack([dh, -dh], 1).flatten()[seq], 0.0).float()
    grad = _grad_plain(p, z, s["tokens"], entropy, a, torch.zeros_like(a), 1.0, s["logits"].dtype)
    return {"loss": loss.float(), "sums": sums.float(), "chosen": reward[0::2].float(),
            "rejected": reward[1::2].float(), "grad": grad}


def _mul_high(a, b):
    return (a * b) >> 32 & 0xFFFFFFFF


def _uniform_words(case, steps):
    """Philox4x32-10 words, one for each element of the arenas: key the seed, counter (four elements' index in their
    tensor low and high, tensor, step)."""
    places, total = _places(case)
    start = torch.tensor([at // 4 for at, _ in places], device="cuda")
    count = torch.tensor([b - a for a, b in zip([at // 4 for at, _ in places], [at // 4 for at, _ in places[1:]] +
                                                [total // 4])], device="cuda")
    tensor = torch.repeat_interleave(torch.arange(len(places), device="cuda"), count)
    index = torch.arange(total // 4, device="cuda") - start[tensor]
    c0, c1, c2, c3 = index & 0xFFFFFFFF, index >> 32, tensor, steps.long()[tensor]
    for k in range(10):
        k0, k1 = SEED + k * 0x9E3779B9 & 0xFFFFFFFF, k * 0xBB67AE85 & 0xFFFFFFFF
        c0, c1, c2, c3 = (_mul_high(c2, 0xCD9E8D57) ^ c1 ^ k0, c2 * 0xCD9E8D57 & 0xFFFFFFFF,
                          _mul_high(c0, 0xD2511F53) ^ c3 ^ k1, c0 * 0xD2511F53 & 0xFFFFFFFF)
    return torch.stack([c0, c1, c2, c3], 1).flatten()


def _e4m3_below(y):
    """The largest e4m3 value at most ``y`` and the next one up, for 0 <= y <= 448."""
    step = ((y.clamp(min=2.0 ** -6).view(torch.int32) >> 23) - 3 << 23).view(torch.float32)  # an eighth of its binade
    low = torch.floor(y / step) * step
    return low, low + step


def _block_scale(x):
    top = x.abs().view(-1, BLOCK).amax(1)
    keep = top >= 1e-30
    return torch.where(keep, top / 448, 0.0), torch.where(keep, 448 / top, 0.0)


def _adamw_plain(s):
    case, arena = s["case"], s["arena"]
    places, total = _places(case)
    s["steps"] += 1
    g = arena["g"].float()
    out = dict(arena, steps=s["steps"])
    del out["g"]
    if case["clip"]:
        norm = g.double().square().sum().sqrt()
        g = g * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
        out["norm"] = norm.float()
    bits8 = case["bits"] == 8
    m, v = arena["m"].float(), arena["v"].float()
    if bits8:
        m = (m.view(-1, BLOCK) * arena["m_scale"][:, None]).flatten()
        v = (v.view(-1, BLOCK) * arena["v_scale"][:, None]).flatten().square()
    m = m * BETAS[0] + g * (1 - BETAS[0])
    v = v * BETAS[1] + g * g * (1 - BETAS[1])
    p = arena["p"]
    if "low" in arena:
        p = ((p.view(torch.int16).int() << 16) + arena["low"].int()).view(torch.float32)
    # every tensor has taken the same number of steps
    t = s["steps"][0].double()
    step_size = (LR / (1 - BETAS[0] ** t)).float()
    unbias = (1 / (1 - BETAS[1] ** t).sqrt()).float()
    decay = torch.tensor(1 - LR * DECAY, dtype=torch.float64).float().item()
    r = v.sqrt()
    p = p * decay - step_size * (m / (r * unbias + EPS))
    if "low" in arena:
        bits = p.view(torch.int32)
        high = bits + 0x8000 >> 16
        arena["low"].copy_((bits - (high << 16)).short())
        arena["p"].copy_(high.short().view(torch.bfloat16))
    else:
        arena["p"].copy_(p)
    if not bits8:
        arena["m"].copy_(m)
        arena["v"].copy_(v)
        return out
    word = _uniform_words(case, s["steps"])
    u = ((word & 0xFFFF).float() + 0.5) / 65536
    scale, inverse = _block_scale(m)
    y = (m.abs().view(-1, BLOCK) * inverse[:, None]).flatten().clamp(max=448)
    low, high = _e4m3_below(y)
    code = torch.where((high - low) * u < y - low, high, low).clamp(max=448)
    arena["m"].copy_(torch.copysign(code, m))
    arena["m_scale"].copy_(scale)
    u = ((word >> 16).float() + 0.5) / 65536
    scale, inverse = _block_scale(r)
    y = (r.view(-1, BLOCK) * inverse[:, None]).flatten().clamp(max=448)
    low, high = _e4m3_below(y)
    code = torch.where((high - low) * (high + low) * u < (y - low) * (y + low), high, low).clamp(max=448)
    code = torch.where((r > 0) & (inverse.repeat_interleave(BLOCK) > 0), code.clamp(min=2.0 ** -9), code)
    arena["v"].copy_(code)
    arena["v_scale"].copy_(scale)
    return out


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _adamw_own(s):
    from tt_rsl_rl_b200.ops.adamw import AdamWPlan

    case, arena = s["case"], s["arena"]
    plan = s.get("plan")
    if plan is None:  # kept by a training program from its first step on
        places, _ = _places(case)

        def views(name, shapes=None):
            if name not in arena:
                return None
            if name.endswith("scale"):
                return [arena[name][at // BLOCK:(at + n + BLOCK - 1) // BLOCK] for at, n in places]
            flat = [arena[name][at:at + n] for at, n in places]
            return [x.view(shape) for x, shape in zip(flat, _shapes(case))]

        params = views("p")
        for p, g in zip(params, views("g")):
            p.grad = g
        plan = s["plan"] = AdamWPlan(params, views("m"), views("v"), s["steps"], exp_avg_scales=views("m_scale"),
                                     exp_avg_sq_scales=views("v_scale"), low_bits=views("low"))
    norm = plan.step(lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, max_grad_norm=MAX_NORM if case["clip"] else None,
                     seed=SEED)
    out = dict(arena, steps=s["steps"])
    del out["g"]
    return out if norm is None else out | {"norm": norm}


def _own(s):
    from tt_rsl_rl_b200.ops.token_loss import preference_loss_grad, token_logprobs, token_policy_loss_grad

    case, x, tokens = s["case"], s["logits"], s["tokens"]
    if case["op"] == "logprobs":
        if not case["backward"]:
            logp, entropy = token_logprobs(x, tokens, mask=s["mask"], temperature=case["temperature"])
            return {"logp": logp, "entropy": entropy}
        x = x.detach().requires_grad_()
        logp, entropy = token_logprobs(x, tokens, mask=s["mask"], temperature=case["temperature"])
        grad, = torch.autograd.grad((logp, entropy), x, (s["dlogp"], s["dentropy"]))
        return {"logp": logp, "entropy": entropy, "grad": grad}
    if case["op"] == "policy":
        out, grad = token_policy_loss_grad(x, tokens, s["old"], s["adv"], ref_logp=s["ref"], mask=s["mask"],
                                           clip_param=CLIP, clip_high=CLIP_HIGH, kl_coef=KL_COEF,
                                           entropy_coef=case["entropy"], temperature=case["temperature"],
                                           grad_scale=LOSS_SCALE[case["dtype"]])
        return {"loss": out.loss, "surrogate": out.surrogate, "kl": out.kl, "entropy": out.entropy,
                "clip_fraction": out.clip_fraction, "logp": out.logp, "grad": grad}
    out, grad = preference_loss_grad(x, tokens, s["ref"], offsets=s["offsets"], mask=s["mask"], beta=BETA,
                                     label_smoothing=SMOOTHING, grad_scale=LOSS_SCALE[case["dtype"]])
    return {"loss": out.loss, "sums": out.seq_logps, "chosen": out.chosen_rewards, "rejected": out.rejected_rewards,
            "grad": grad}


def run(state):
    op = state["case"]["op"]
    if own:
        return _adamw_own(state) if op == "adamw" else _own(state)
    return {"logprobs": _logprobs_plain, "policy": _policy_plain, "preference": _preference_plain,
            "adamw": _adamw_plain}[op](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(shape) for shape in _shapes(case))
        weight, grad = 4, BYTES[case["dtype"]]  # fp32 weights, or bf16 ones and the 16 bits below
        states = 8 if case["bits"] == 32 else 2 + 8 / BLOCK
        return {"bytes": n * (2 * weight + grad + 2 * states), "flops": n * 15}
    size = BYTES[case["dtype"]]
    vocab = case["vocab"]
    if case["op"] == "preference":
        rows = sum(_lengths(case)) + case["behind"]
        active = sum(_lengths(case)) - sum(_prompts(case))
        return {"bytes": (active + rows) * vocab * size + rows * 9, "flops": 12 * active * vocab}
    rows = case["rows"]
    active = rows * (1 - case["masked"])
    if case["op"] == "logprobs" and not case["backward"]:
        return {"bytes": active * vocab * size + rows * 16, "flops": 6 * active * vocab}
    return {"bytes": (active + rows) * vocab * size + rows * 32, "flops": 14 * active * vocab}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _adamw_exact(s)
    x, tokens, mask, t = s["logits"], s["tokens"], s["mask"], case.get("temperature", 1.0)
    shape, vocab = tokens.shape, x.shape[-1]
    tokens, rows = tokens.reshape(-1), tokens.numel()
    active = torch.ones(rows, dtype=torch.bool, device="cuda") if mask is None else mask.reshape(-1)
    step = max(1, 2 ** 27 // vocab)
    x = x.reshape(-1, vocab)

    def chunk(at):  # the rows from `at` on in 64 bits, with their log-softmax
        z = x[at:at + step].double().requires_grad_()
        lp = torch.log_softmax(z / t, -1)
        return z, lp, lp.gather(-1, tokens[at:at + step, None])[:, 0]

    def entropy_of(lp):
        return -(lp.exp() * lp.masked_fill(lp == NEG_INF, 0.0)).sum(-1)

    logp, entropy = (torch.zeros(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    with torch.no_grad():
        for at in range(0, rows, step):
            _, lp, logp[at:at + step] = chunk(at)
            entropy[at:at + step] = entropy_of(lp)
    lp0 = logp.clone().requires_grad_()
    en0 = entropy.clone().requires_grad_()
    out = {}
    if case["op"] == "logprobs":
        out = {"logp": (logp * active).view(shape), "entropy": (entropy * active).view(shape)}
        if not case["backward"]:
            return out
        total = ((lp0 * s["dlogp"].reshape(-1) + en0 * s["dentropy"].reshape(-1)) * active).sum()
    elif case["op"] == "policy":
        w = active.double() / active.sum().clamp(min=1)
        old, ref, adv = (s[k].reshape(-1).double() for k in ("old", "ref", "adv"))
        ratio = torch.exp(lp0 - old)
        bounded = torch.clamp(ratio, 1 - CLIP, 1 + CLIP_HIGH)
        gain = torch.minimum(adv * ratio, adv * bounded)
        kl = torch.expm1(ref - lp0) - (ref - lp0)
        total = -(w * gain).sum() + KL_COEF * (w * kl).sum() - case["entropy"] * (w * en0).sum()
        out = {"loss": total, "surrogate": -(w * gain).sum(), "kl": (w * kl).sum(), "entropy": (w * en0).sum(),
               "clip_fraction": (w * (adv * ratio > adv * bounded)).sum(), "logp": (logp * active).view(shape)}
    else:
        ends = s["offsets"].tolist()
        sums = torch.stack([(lp0[a:b] * active[a:b]).sum() for a, b in zip(ends[:-1], ends[1:])])
        reward = BETA * (sums - s["ref"].double())
        h = reward[0::2] - reward[1::2]
        sig = torch.nn.functional.logsigmoid
        total = -((1 - SMOOTHING) * sig(h) + SMOOTHING * sig(-h)).mean()
        out = {"loss": total, "sums": sums, "chosen": reward[0::2], "rejected": reward[1::2]}
    scale = 1.0 if case["op"] == "logprobs" else LOSS_SCALE[case["dtype"]]
    da, db = torch.autograd.grad(total * scale, (lp0, en0), allow_unused=True)
    grad = torch.zeros(rows, vocab, dtype=torch.float64 if rows * vocab < 2 ** 28 else torch.float32, device="cuda")
    for at in range(0, rows, step):
        z, lp, picked = chunk(at)
        weight = da[at:at + step]
        if db is not None and bool(db.any()):
            picked, weight = torch.cat([picked, entropy_of(lp)]), torch.cat([weight, db[at:at + step]])
        keep = active[at:at + step]
        grad[at:at + step] = torch.autograd.grad(picked, z, weight)[0] * keep[:, None]
        del z, lp, picked
    return {k: v.detach() for k, v in out.items()} | {"grad": grad.view(*shape, vocab)}


def _adamw_exact(s):
    case, arena = s["case"], s["arena"]
    out = {"steps": s["steps"].double() + 1}
    g = arena["g"].double()
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, MAX_NORM / (out["norm"].item() + 1e-6))
    m, v = arena["m"].double(), arena["v"].double()
    if case["bits"] == 8:
        m = m * arena["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * arena["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m.lerp_(g, 1 - BETAS[0])
    v = BETAS[1] * v + (1 - BETAS[1]) * g ** 2
    p = arena["p"].double()
    if "low" in arena:
        p = ((arena["p"].view(torch.int16).int() << 16) + arena["low"].int()).view(torch.float32).double()
        out["low"] = None
    t = STEP0 + 1
    hat_m, hat_v = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
    out["p"] = p - LR * DECAY * p - LR * hat_m / (hat_v.sqrt() + EPS)
    if case["bits"] == 32:
        return out | {"m": m, "v": v}
    # the codes are drawn: they have no value of their own, their scales have
    return out | {"m": None, "v": None, "m_scale": m.abs().view(-1, BLOCK).amax(1) / 448,
                  "v_scale": v.sqrt().view(-1, BLOCK).amax(1) / 448}
