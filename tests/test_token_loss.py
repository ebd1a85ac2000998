"""Token-policy operators on the CPU: the PyTorch path against 64-bit definitions, gradients against differences, and
the refusals."""

import pytest
import torch

import token_oracle as oracle
from tt_rsl_rl_b200.ops.token_loss import (preference_loss, preference_loss_grad, token_logprobs, token_policy_loss,
                                           token_policy_loss_grad)


def _case(shape=(5, 7), vocab=11, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(*shape, vocab, generator=g) * 2).to(dtype)
    tokens = torch.randint(vocab, shape, generator=g)
    old = torch.randn(shape, generator=g) * 0.3 - 2
    adv, ref = torch.randn(shape, generator=g), torch.randn(shape, generator=g) * 0.3 - 2
    mask = torch.rand(shape, generator=g) > 0.3
    return logits, tokens, old, adv, ref, mask


@pytest.mark.parametrize("kind", ["k1", "k2", "k3"])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_policy_loss_and_gradient_match_the_definition(kind, reduction):
    logits, tokens, old, adv, ref, mask = _case()
    out, grad = token_policy_loss_grad(logits, tokens, old, adv, ref_logp=ref, mask=mask, clip_high=0.3, kl_coef=0.1,
                                       kl_estimator=kind, entropy_coef=0.02, temperature=0.7, reduction=reduction,
                                       grad_scale=3.0)
    loss, stats, logp, da, db = oracle.policy(logits, tokens, old, adv, ref, mask, lo=0.8, hi=1.3, kl_coef=0.1,
                                              kind=kind, entropy_coef=0.02, temperature=0.7, mean=reduction == "mean")
    assert abs(out.loss - loss) < 1e-5 * (1 + abs(loss))
    for got, want in zip(out[1:5], stats):
        assert abs(got - want) < 1e-5 * (1 + abs(want))
    assert torch.allclose(out.logp.double(), logp, atol=1e-5)
    want, bound = oracle.logits_grad(logits, tokens, mask, 0.7, 3 * da, 3 * db)
    assert ((grad - want).abs() <= bound + oracle.rounding(want, torch.float32)).all()
    auto = logits.clone().requires_grad_()
    (3 * token_policy_loss(auto, tokens, old, adv, ref_logp=ref, mask=mask, clip_high=0.3, kl_coef=0.1,
                           kl_estimator=kind, entropy_coef=0.02, temperature=0.7, reduction=reduction).loss).backward()
    assert torch.allclose(auto.grad, grad, atol=1e-6)


def test_policy_gradient_matches_differences():
    logits, tokens, old, adv, ref, mask = _case((3, 4), 6, seed=3)
    z = logits.double()

    def loss(x):
        return oracle.policy(x, tokens, old, adv, ref, mask, lo=0.8, hi=1.2, kl_coef=0.2, kind="k3", entropy_coef=0.05,
                             temperature=1.3)[0]

    _, grad = token_policy_loss_grad(logits, tokens, old, adv, ref_logp=ref, mask=mask, kl_coef=0.2, entropy_coef=0.05,
                                     temperature=1.3)
    h = 1e-6
    for i in range(3):
        for j in range(4):
            for c in range(6):
                up, down = z.clone(), z.clone()
                up[i, j, c] += h
                down[i, j, c] -= h
                # central differences: h^2 / 6 times a third derivative of order one, and 2^-52 / h of rounding
                assert abs(grad[i, j, c].item() - (loss(up) - loss(down)) / (2 * h)) < 1e-6


def test_masked_rows_hold_anything():
    logits, tokens, old, adv, ref, mask = _case()
    spoiled = logits.clone()
    spoiled[~mask] = float("nan")
    tokens = torch.where(mask, tokens, -100)
    old = torch.where(mask, old, float("inf"))
    a = token_policy_loss_grad(logits, tokens, old, adv, ref_logp=ref, kl_coef=0.1)
    b = token_policy_loss_grad(spoiled, tokens, old, adv, ref_logp=ref, kl_coef=0.1)
    for x, y in zip((*a[0], a[1]), (*b[0], b[1])):
        assert torch.equal(x, y)
    assert (b[1][~mask] == 0).all() and torch.isfinite(b[1]).all()


def test_no_counted_row():
    logits, tokens, old, adv, *_ = _case()
    out, grad = token_policy_loss_grad(logits, tokens, old, adv, mask=torch.zeros(5, 7))
    assert out.loss == 0 and (grad == 0).all()
    logp, entropy = token_logprobs(logits, torch.full_like(tokens, 11))
    assert (logp == 0).all() and (entropy == 0).all()


@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0), ("ipo", 0.0)])
@pytest.mark.parametrize("average", [False, True])
def test_preference_matches_the_definition(kind, smoothing, average):
    logits, tokens, _, _, _, mask = _case((6, 7), seed=1)
    ref = torch.linspace(-20, -12, 6) if not average else torch.linspace(-3, -2, 6)
    out, grad = preference_loss_grad(logits, tokens, ref, mask=mask, beta=0.2, loss_type=kind, label_smoothing=smoothing,
                                     average=average)
    loss, lps, rewards, da = oracle.preference(logits, tokens, ref, [(7 * i, 7 * i + 7) for i in range(6)], mask,
                                               beta=0.2, smoothing=smoothing, kind=kind, average=average)
    assert abs(out.loss - loss) < 1e-5 * (1 + abs(loss))
    assert torch.allclose(out.seq_logps.double(), lps, atol=1e-4)
    assert torch.allclose(torch.stack([out.chosen_rewards, out.rejected_rewards], 1).flatten().double(), rewards,
                          atol=1e-4)
    want, bound = oracle.logits_grad(logits, tokens, mask, 1.0, da, 0 * da)
    assert ((grad - want).abs() <= 2 * bound + 1e-5 * want.abs()).all()
    # packed rows with offsets are the same sequences
    packed, packed_grad = preference_loss_grad(logits.flatten(0, 1), tokens.flatten(), ref, mask=mask.flatten(),
                                               offsets=torch.arange(0, 43, 7), beta=0.2, loss_type=kind,
                                               label_smoothing=smoothing, average=average)
    assert torch.allclose(packed.loss, out.loss) and torch.allclose(packed_grad.view_as(grad), grad, atol=1e-7)


def test_empty_inputs():
    logits, tokens = torch.zeros(0, 5), torch.zeros(0, dtype=torch.long)
    none = torch.zeros(0)
    assert token_logprobs(logits, tokens)[0].shape == (0,)
    out, grad = token_policy_loss_grad(logits, tokens, none, none)
    assert out.loss == 0 and grad.shape == (0, 5)
    out, grad = preference_loss_grad(logits, tokens, none, offsets=torch.zeros(1, dtype=torch.long))
    assert out.loss == 0 and out.chosen_rewards.shape == (0,)


REFUSALS = [
    (TypeError, "logits must be", dict(logits=lambda x: x.double())),
    (ValueError, r"\[rows, V\]", dict(logits=lambda x: x[0, 0])),
    (ValueError, "columns", dict(logits=lambda x: x.transpose(1, 2).contiguous().transpose(1, 2))),
    (TypeError, "tokens must be", dict(tokens=lambda x: x.short())),
    (ValueError, "tokens must have the shape", dict(tokens=lambda x: x[:, 1:])),
    (TypeError, "mask must be", dict(mask=lambda x: x.double())),
    (TypeError, "advantages must be", dict(adv=lambda x: x.half())),
    (ValueError, "old_logp must have the shape", dict(old=lambda x: x.flatten())),
    (ValueError, "temperature", dict(temperature=0.0)),
    (ValueError, "temperature", dict(temperature=float("nan"))),
    (ValueError, "temperature", dict(temperature=1e-7)),
    (ValueError, "kl_estimator", dict(kl_estimator="k4")),
    (ValueError, "reduction", dict(reduction="none")),
    (ValueError, "negative", dict(clip_param=-0.1)),
    (ValueError, "finite", dict(entropy_coef=float("nan"))),
    (ValueError, "needs ref_logp", dict(ref=lambda x: None)),
]


def refuse(device, error, text, change):
    logits, tokens, old, adv, ref, mask = (x.to(device) for x in _case())
    x = {"logits": logits, "tokens": tokens, "old": old, "adv": adv, "ref": ref, "mask": mask.float()}
    kwargs = {"kl_coef": 0.1}
    for key, value in change.items():
        if key in x:
            x[key] = value(x[key])
        else:
            kwargs[key] = value
    with pytest.raises(error, match=text):
        token_policy_loss_grad(x["logits"], x["tokens"], x["old"], x["adv"], ref_logp=x["ref"], mask=x["mask"], **kwargs)
    with pytest.raises(error, match=text):
        token_policy_loss(x["logits"], x["tokens"], x["old"], x["adv"], ref_logp=x["ref"], mask=x["mask"], **kwargs)


@pytest.mark.parametrize("error,text,change", REFUSALS)
def test_policy_refusals(error, text, change):
    refuse("cpu", error, text, change)


def refuse_preference(device):
    logits, tokens, *_ = (x.to(device) for x in _case((4, 7)))
    packed, flat = logits.flatten(0, 1), tokens.flatten()
    off = torch.arange(0, 29, 7, device=device)
    for error, text, args, kwargs in [
        (ValueError, "even", (logits[:3], tokens[:3]), {}),
        (ValueError, "offsets belong", (logits, tokens), {"offsets": off}),
        (ValueError, "need the offsets", (packed, flat), {}),
        (TypeError, "offsets must be", (packed, flat), {"offsets": off.float()}),
        (ValueError, "offsets must be", (packed, flat), {"offsets": off[:, None]}),
        (TypeError, "ref_logps must be", (logits, tokens, torch.zeros(4, device=device).double()), {}),
        (ValueError, "ref_logps must be", (logits, tokens, torch.zeros(3, device=device)), {}),
        (ValueError, "loss_type", (logits, tokens), {"loss_type": "dpo"}),
        (ValueError, "beta", (logits, tokens), {"beta": 0.0}),
        (ValueError, "label_smoothing", (logits, tokens), {"label_smoothing": 0.6}),
        (ValueError, "belongs to", (logits, tokens), {"label_smoothing": 0.1, "loss_type": "ipo"}),
    ]:
        with pytest.raises(error, match=text):
            preference_loss(*args, **kwargs)
        with pytest.raises(error, match=text):
            preference_loss_grad(*args, **kwargs)


def test_preference_refusals():
    refuse_preference("cpu")


def extreme_rows(dtype, top, vocab, seed=0):
    """Eight rows whose largest logits lie within six steps of their type around ``top``: at every column; on every column
    but one; at a tenth of the columns beside far lower ones, -inf and the type's lowest value; all equal; ordinary logits
    with a tenth of the columns at ``top`` where that is low. And the column of each row's largest logit."""
    g = torch.Generator().manual_seed(seed)
    bits = {4: torch.int32, 2: torch.int16}[dtype.itemsize]
    near = torch.full((8, vocab), top, dtype=torch.float64).to(dtype)
    near = (near.view(bits) + torch.randint(-6, 7, near.shape, generator=g).to(bits)).view(dtype)
    x = near.clone()
    x[1, vocab // 2] = near[1].max()
    few = torch.rand(vocab, generator=g) < 0.1
    few[vocab // 3] = True
    x[2] = torch.where(few, near[2], float("-inf"))
    x[3] = torch.where(few, near[3], torch.finfo(dtype).min)
    x[4] = torch.where(few, near[4], (near[4].double() - abs(top) / 2).to(dtype))
    x[5] = x[5, 0]
    ordinary = (torch.randn(2, vocab, generator=g) * 3).to(dtype)
    x[6:] = torch.where(few & (near[6:] < ordinary), near[6:], ordinary)
    return x, x.double().argmax(-1)


# Temperature and largest logit: |largest| / T from ordinary sizes to where fp32 steps are far wider than one, around
# 2^24 / log2(e) = 11,629,080 too (the largest fp32 logits there are a unit of the exponent apart).
RANGES = [(1.0, -1e10), (1.0, 6e9), (1.0, -1e12), (1.0, 1e18), (1.0, -1e19), (1.0, -1e25), (1.0, 11629080.0),
          (1.0, -11629080.0), (1.0, 5e4), (1e-3, 3e6), (1e-3, 16000.0), (1e-3, -11629.08), (1e-6, 5000.0), (1e-6, 6e4),
          (1e-6, 11.62908), (1e-6, -11.62908), (1e6, 1e16), (1e6, -1.162908e13), (1.0, 3e38), (1.0, -3e38), (0.5, -6e4)]


def test_uint8_masks_select():
    """Any value of a byte mask but zero counts a row once."""
    logits, tokens, old, adv, ref, mask = _case((4, 7))
    many = mask.to(torch.uint8) * 3
    many[0, 0] = 255
    mask[0, 0] = True
    for a, b in ((token_policy_loss_grad(logits, tokens, old, adv, ref_logp=ref, mask=m, kl_coef=0.1, reduction="sum")
                  for m in (many, mask)), (preference_loss_grad(logits, tokens, mask=m) for m in (many, mask))):
        for x, y in zip((*a[0], a[1]), (*b[0], b[1])):
            assert torch.equal(x, y)


def only_logits_get_gradients(device):
    """Every other input is a constant of the loss, floating masks and references too."""
    logits, tokens, old, adv, ref, mask = (x.to(device) for x in _case((4, 7)))
    z = logits.clone().requires_grad_()
    rows = [x.clone().requires_grad_() for x in (old, adv, ref, mask.float())]
    seq = torch.zeros(4, device=device, requires_grad=True)
    token_policy_loss(z, tokens, rows[0], rows[1], ref_logp=rows[2], mask=rows[3], kl_coef=0.1, entropy_coef=0.1).loss.backward()
    first, z.grad = z.grad, None
    token_policy_loss(z, tokens, old, adv, ref_logp=ref, mask=mask.float(), kl_coef=0.1, entropy_coef=0.1).loss.backward()
    assert torch.equal(first, z.grad)
    preference_loss(z, tokens, seq, mask=rows[3], average=True).loss.backward()
    assert seq.grad is None and all(x.grad is None for x in rows)
    # without a gradient of the logits there is nothing to differentiate
    assert not token_policy_loss(logits, tokens, rows[0], rows[1]).loss.requires_grad
    assert not preference_loss(logits, tokens, seq).loss.requires_grad


def test_only_logits_get_gradients():
    only_logits_get_gradients("cpu")


def decided_pairs(device):
    """A sequence that its policy excludes (log-probability -inf): as the rejected one its pair is decided, with a loss of
    zero and no gradient; as the chosen one the loss is infinite. Without label smoothing nothing weighs the other side."""
    logits, tokens, *_ = _case((4, 7), seed=5)
    other = preference_loss_grad(logits[2:].to(device), tokens[2:].to(device), beta=0.2)
    banned = logits.clone()
    banned[1, 3, tokens[1, 3]] = float("-inf")
    out, grad = preference_loss_grad(banned.to(device), tokens.to(device), beta=0.2)
    assert out.rejected_rewards[0] == float("-inf")
    # the mean over two pairs, one of them zero: half of the other's loss and gradient, rounded once more
    assert out.loss.item() == pytest.approx(other[0].loss.item() / 2, rel=1e-6)
    assert (grad[:2] == 0).all() and torch.allclose(grad[2:], other[1] / 2, rtol=1e-6, atol=0.0)
    z = banned.clone().to(device).requires_grad_()
    loss = preference_loss(z, tokens.to(device), beta=0.2).loss
    loss.backward()
    assert torch.equal(loss.detach(), out.loss) and torch.isfinite(z.grad).all()
    banned[0, 2, tokens[0, 2]], banned[1] = float("-inf"), logits[1]
    assert preference_loss(banned.to(device), tokens.to(device)).loss == float("inf")
    assert preference_loss(banned.to(device), tokens.to(device), label_smoothing=0.1).loss == float("inf")


def test_decided_pairs():
    decided_pairs("cpu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("temperature,top", RANGES)
def test_large_logits_over_temperature(dtype, temperature, top):
    if dtype == torch.float16 and abs(top) > 6e4:
        return
    x, tokens = extreme_rows(dtype, top, 503)
    logp, entropy = token_logprobs(x, tokens, temperature=temperature)
    _, want, want_h = oracle.rows(x, tokens, torch.ones(8, dtype=torch.bool), temperature)
    assert ((logp.double() - want).abs() <= oracle.logp_bound(want)).all()
    assert ((entropy.double() - want_h).abs() <= 2 * oracle.logp_bound(want_h) + 2e-5).all()


def test_rows_outside_the_sequences_hold_anything():
    logits, tokens, *_ = _case((12,), seed=6)
    spoiled = logits.clone()
    spoiled[:2], spoiled[10], spoiled[11, 3] = float("nan"), float("inf"), float("-inf")
    offsets = torch.tensor([2, 5, 5, 7, 10])
    clean, want = preference_loss_grad(logits, tokens, offsets=offsets)
    out, grad = preference_loss_grad(spoiled, tokens, offsets=offsets)
    assert torch.equal(out.loss, clean.loss) and torch.equal(grad, want)
    assert (grad[:2] == 0).all() and (grad[10:] == 0).all()
    none, grad = preference_loss_grad(spoiled, tokens, offsets=torch.tensor([3]))
    assert none.loss == 0 and (grad == 0).all()


def clipped_ratios(device):
    """A ratio beyond fp32's range (the old policy all but excluded the token) is clipped like any other: no gradient where
    the advantage is positive, an infinite loss where it is not."""
    logits, tokens, old, adv, *_ = (x.to(device) for x in _case((6,), seed=7))
    for far in (-100.0, float("-inf")):
        old[2] = far
        adv[2] = 1.5
        out, grad = token_policy_loss_grad(logits, tokens, old, adv)
        rest = torch.arange(6, device=device) != 2
        other, want = token_policy_loss_grad(logits, tokens, old, adv, mask=rest, reduction="sum")
        assert out.loss.item() == pytest.approx((other.loss.item() - 1.5 * 1.2) / 6, rel=1e-5, abs=1e-6)
        assert torch.allclose(grad, want / 6, rtol=1e-5, atol=1e-7) and (grad[2] == 0).all()
        z = logits.clone().requires_grad_()
        token_policy_loss(z, tokens, old, adv).loss.backward()
        assert torch.allclose(z.grad, grad, rtol=1e-4, atol=1e-6)
        adv[2] = -1.5
        assert token_policy_loss_grad(logits, tokens, old, adv)[0].loss == float("inf")


def test_clipped_ratios():
    clipped_ratios("cpu")


def test_decreasing_offsets_are_refused():
    logits, tokens, *_ = _case((20,), seed=8)
    for offsets in ([0, 10, 5, 20, 20], [5, 3, 20], [0, 10, 30, 15, 20]):
        with pytest.raises(ValueError, match="decrease"):
            preference_loss_grad(logits, tokens, offsets=torch.tensor(offsets))
