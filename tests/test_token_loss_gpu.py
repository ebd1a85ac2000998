"""Token-policy kernels against 64-bit definitions: types, vocabularies, strides, masks, extremes, capture, streams."""

import math

import pytest
import torch

import token_oracle as oracle
from test_token_loss import (RANGES, REFUSALS, clipped_ratios, decided_pairs, extreme_rows, only_logits_get_gradients,
                             refuse, refuse_preference)
from tt_rsl_rl_b200.ops.token_loss import (preference_loss, preference_loss_grad, token_logprobs, token_policy_loss,
                                           token_policy_loss_grad)

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]

def _place(x, how):
    """CPU logits on the device: contiguous, without the last row of each batch entry, with padded rows, or starting one
    element into their storage."""
    if how == "shifted":
        wide = torch.full((*x.shape[:-2], x.shape[-2] + 1, x.shape[-1]), 7.0, dtype=x.dtype, device="cuda")
        wide[..., :-1, :] = x.cuda()
        return wide[..., :-1, :]
    if how == "padded":
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 3), float("nan"), dtype=x.dtype, device="cuda")
        wide[..., :-3] = x.cuda()
        return wide[..., :-3]
    if how == "offset":
        flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")
        flat[1:] = x.cuda().flatten()
        return flat[1:].view(x.shape)
    return x.cuda()


def _make(shape, vocab, dtype, seed=0, dead=False, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*shape, vocab, generator=g) * spread).to(dtype)
    tokens = torch.randint(vocab, shape, generator=g)
    if dead and vocab > 4:
        x[..., 1::3] = float("-inf")
        x[..., 2::3] = torch.finfo(dtype).min
        tokens = tokens // 3 * 3
    mask = torch.rand(shape, generator=g) > 0.25
    mask.view(-1)[0] = True
    return x, tokens, mask, g


def _check_grad(got, x, tokens, counted, temperature, a, b, a_off=None, slack=0.0):
    """``a_off``: how far off a itself may be, per row (it comes from an fp32 log-probability); ``slack``: the same
    relative to a, in units of 3e-5."""
    assert got.dtype == x.dtype and got.shape == x.shape
    want, bound = oracle.logits_grad(x, tokens, counted, temperature, a, b)
    if a_off is not None:  # the column's share: onehot - p, at most 1 at the token and p elsewhere
        p = oracle.rows(x, tokens, counted, temperature)[0].exp()
        share = p.scatter(-1, tokens.clamp(0, p.shape[-1] - 1)[..., None], 1.0)
        bound = bound + torch.where(counted, a_off, 0.0)[..., None] * share / temperature
    got = got.double().cpu()
    far = (got - want).abs() - (want.abs() * 3e-5 * slack + bound * (1 + slack))
    assert (far <= oracle.rounding(want, x.dtype) * 1.01).all(), far.max()
    assert (got[~counted] == 0).all()


SIZES = [((1,), 1), ((3,), 7), ((5,), 8), ((33,), 100), ((4, 9), 1000), ((2, 3), 4099), ((700,), 1024), ((2, 5), 8192),
         ((7,), 20000), ((3, 4), 50001), ((2,), 131072), ((1,), 131075), ((3,), 262144), ((2,), 600001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,vocab", SIZES)
def test_logprobs(dtype, shape, vocab):
    x, tokens, mask, g = _make(shape, vocab, dtype)
    counted = mask
    for how in ("plain", "shifted", "padded", "offset"):
        z = _place(x, how).requires_grad_()
        logp, entropy = token_logprobs(z, tokens.cuda(), mask=mask.cuda(), temperature=0.8)
        _, want, want_h = oracle.rows(x, tokens, counted, 0.8)
        want, want_h = torch.where(counted, want, 0.0), torch.where(counted, want_h, 0.0)
        assert ((logp.detach().double().cpu() - want).abs() <= oracle.logp_bound(want)).all(), how
        # the entropy is ln s minus a mean of |log p|: each within the bound of a log-probability of its size
        assert ((entropy.detach().double().cpu() - want_h).abs() <= 2 * oracle.logp_bound(want_h) + 2e-5).all(), how
        a, b = torch.randn(shape, generator=g), torch.randn(shape, generator=g) * 0.3
        grad, = torch.autograd.grad((logp, entropy), z, (a.cuda(), b.cuda()))
        _check_grad(grad, x, tokens, counted, 0.8, a.double(), b.double())
    one, = torch.autograd.grad(token_logprobs(z, tokens.cuda(), mask=mask.cuda())[0].sum(), z)  # expanded gradient
    _check_grad(one, x, tokens, counted, 1.0, torch.ones(shape).double(), torch.zeros(shape).double())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 3001, 40001])
def test_dead_columns(dtype, vocab):
    """Columns at -inf and at the type's lowest value have probability zero; a row of lowest values is uniform."""
    x, tokens, mask, _ = _make((6,), vocab, dtype, dead=True)
    x[1] = torch.finfo(dtype).min
    x[2, :] = float("-inf")
    x[2, tokens[2]] = -3.0  # one column is left
    logp, entropy = token_logprobs(x.cuda(), tokens.cuda())
    _, want, want_h = oracle.rows(x, tokens, torch.ones(6, dtype=torch.bool), 1.0)
    assert ((logp.double().cpu() - want).abs() <= oracle.logp_bound(want)).all()
    assert ((entropy.double().cpu() - want_h).abs() <= 2 * oracle.logp_bound(want_h) + 2e-5).all()
    old, adv = want.float() + 0.1, torch.linspace(-1, 1, 6)
    out, grad = token_policy_loss_grad(x.cuda(), tokens.cuda(), old.cuda(), adv.cuda(), entropy_coef=0.1,
                                       grad_scale=64.0)
    _, _, _, da, db = oracle.policy(x, tokens, old, adv, None, None, lo=0.8, hi=1.2, kl_coef=0.0, kind="k3",
                                    entropy_coef=0.1, temperature=1.0)
    assert torch.isfinite(out.loss) and torch.isfinite(grad.float()).all()
    _check_grad(grad, x, tokens, torch.ones(6, dtype=torch.bool), 1.0, 64 * da, 64 * db, slack=1.0)


def test_rows_without_a_column_and_nan_logits():
    x, tokens, _, _ = _make((5,), 3000, torch.bfloat16)
    x[1] = float("-inf")
    x[2, 7] = float("nan")
    x[3, 5] = float("inf")
    logp, entropy = token_logprobs(x.cuda(), tokens.cuda())
    want = torch.log_softmax(x.double(), -1).gather(-1, tokens[:, None])[:, 0]
    assert logp.isnan().cpu().tolist() == want.isnan().tolist() == [False, True, True, True, False]
    assert entropy.isnan().cpu().tolist() == [False, True, True, True, False]
    out, grad = token_policy_loss_grad(x.cuda(), tokens.cuda(), logp, torch.ones(5, device="cuda"))
    assert out.loss.isnan()  # a fault in a counted row shows
    keep = torch.tensor([True, False, False, False, True]).cuda()
    out, grad = token_policy_loss_grad(x.cuda(), tokens.cuda(), logp, torch.ones(5, device="cuda"), mask=keep)
    assert torch.isfinite(out.loss) and torch.isfinite(grad.float()).all() and (grad[1:4] == 0).all()


POLICY = [  # kl estimator, kl_coef, entropy_coef, temperature, weights, reduction
    ("k3", 0.04, 0.0, 1.0, "bool", "mean"), ("k1", 0.1, 0.01, 0.7, "float", "sum"), ("k2", 0.1, 0.02, 1.4, None, "mean"),
    ("k3", 0.0, -0.01, 1.0, "uint8", "sum")]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,vocab", SIZES)
@pytest.mark.parametrize("kind,kl_coef,entropy_coef,temperature,kind_w,reduction", POLICY)
def test_policy(dtype, shape, vocab, kind, kl_coef, entropy_coef, temperature, kind_w, reduction):
    x, tokens, mask, g = _make(shape, vocab, dtype, seed=1, dead=kind == "k2")
    mask = {"bool": mask, "uint8": mask.to(torch.uint8) * 3, None: None,
            "float": mask * (0.25 + torch.rand(shape, generator=g))}[kind_w]
    if kind_w == "uint8":
        mask = (mask != 0).to(torch.uint8)
    tokens.view(-1)[-1] = -100 if tokens.numel() > 1 else tokens.view(-1)[-1]
    w = oracle.weights(x, tokens, mask)
    _, logp, _ = oracle.rows(x, tokens, w != 0, temperature)
    old = (logp + 0.2 * torch.randn(shape, generator=g)).float()
    ref = (logp + 0.3 * torch.randn(shape, generator=g)).float()
    # ratios exactly at the clip bounds would be decided by rounding
    ratio = (logp - old.double()).exp()
    old = torch.where(((ratio - 0.8).abs() < 1e-3) | ((ratio - 1.3).abs() < 1e-3), old + 0.01, old)
    adv = torch.randn(shape, generator=g)
    scale = 256.0 if dtype == torch.float16 else 1.0
    kwargs = dict(clip_param=0.2, clip_high=0.3, kl_coef=kl_coef, kl_estimator=kind, entropy_coef=entropy_coef,
                  temperature=temperature, reduction=reduction)
    dev = [t.cuda() for t in (old, adv)]
    extra = dict(ref_logp=ref.cuda(), mask=None if mask is None else mask.cuda())
    loss, stats, want_logp, da, db = oracle.policy(x, tokens, old, adv, ref, mask, lo=0.8, hi=1.3, kl_coef=kl_coef,
                                                   kind=kind, entropy_coef=entropy_coef, temperature=temperature,
                                                   mean=reduction == "mean")
    # a term is a smooth function of logp and H (both within 3e-5 here) with slopes of at most about 2 |A| + 1
    size = (w.abs() * (adv.abs() * 2 + 1)).sum().item() / (abs(w.sum().item()) if reduction == "mean" else 1.0)
    # a = w (-A r or 0, + kl_coef dk/dlogp): logp is off by delta, r by r delta, dk/dlogp by at most (1 + e^d) delta
    delta = oracle.logp_bound(logp) + 2.0 ** -21
    slope = adv.abs().double() * (logp - old.double()).exp() + kl_coef * (1 + (ref.double() - logp).exp())
    a_off = scale * w.abs() * slope * delta / (w.sum().abs() if reduction == "mean" else 1.0)
    for how in ("plain", "shifted", "offset"):
        z = _place(x, how)
        tok = tokens.cuda().int() if how == "shifted" else tokens.cuda()
        out, grad = token_policy_loss_grad(z, tok, *dev, grad_scale=scale, **extra, **kwargs)
        assert abs(out.loss.item() - loss) <= 5e-5 * size + 1e-6 * abs(loss)
        for got, want in zip(out[1:5], stats):
            assert abs(got.item() - want) <= 5e-5 * (w.abs() * (adv.abs() * 2 + 1)).sum() / w.sum().abs() + 1e-6 * abs(want)
        assert ((out.logp.double().cpu() - want_logp).abs() <= oracle.logp_bound(want_logp)).all()
        _check_grad(grad, x, tokens, w != 0, temperature, scale * da, scale * db, a_off)
    z = _place(x, "plain").requires_grad_()
    auto = token_policy_loss(z, tokens.cuda(), *dev, **extra, **kwargs)
    assert abs(auto.loss.item() - loss) <= 5e-5 * size + 1e-6 * abs(loss)
    (auto.loss * scale).backward()
    _check_grad(z.grad, x, tokens, w != 0, temperature, scale * da, scale * db, a_off)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [13, 2048, 50001])
@pytest.mark.parametrize("kind,smoothing,average", [("sigmoid", 0.1, False), ("hinge", 0.0, False), ("ipo", 0.0, True),
                                                    ("sigmoid", 0.0, True)])
def test_preference(dtype, vocab, kind, smoothing, average):
    lengths = [3, 1, 0, 5, 17, 9]
    bounds, at = [], 2  # two rows before the first sequence, three behind the last
    for n in lengths:
        bounds.append((at, at + n))
        at += n
    rows = at + 3
    x, tokens, mask, g = _make((rows,), vocab, dtype, seed=4)
    x[:2], x[-3:] = float("nan"), float("nan")
    mask[:2], mask[-1] = True, True
    offsets = torch.tensor([2] + [b for _, b in bounds])
    clean = torch.where(x.isnan(), 0.0, x)
    lps = oracle.preference(clean, tokens, None, bounds, mask, beta=0.2, average=average)[1]
    ref = (lps + 3 * torch.randn(6, generator=g)).float()
    loss, lps, rewards, da = oracle.preference(clean, tokens, ref, bounds, mask, beta=0.2, smoothing=smoothing,
                                               kind=kind, average=average)
    scale = 64.0 if dtype == torch.float16 else 1.0
    kwargs = dict(mask=mask.cuda(), beta=0.2, label_smoothing=smoothing, loss_type=kind, average=average)
    for how, off in (("plain", offsets), ("offset", offsets.int())):
        out, grad = preference_loss_grad(_place(x, how), tokens.cuda(), ref.cuda(), offsets=off.cuda(), grad_scale=scale,
                                         **kwargs)
        # a sequence of n rows: n bounds of a log-probability (|logp| up to about 25), 17 rows at most
        assert ((out.seq_logps.double().cpu() - lps).abs() <= 17 * 2e-5).all()
        got = torch.stack([out.chosen_rewards, out.rejected_rewards], 1).flatten().double().cpu()
        assert ((got - rewards).abs() <= 17 * 2e-5 * 0.2 + 1e-6 * rewards.abs()).all()
        assert abs(out.loss.item() - loss) <= 2e-3 * (1 + abs(loss)) if kind == "ipo" else 2e-4 * (1 + abs(loss))
        # the coefficient moves with h, which is off by at most 34 * 2e-5 * beta (ipo: divided by beta^2)
        _check_grad(grad, clean, tokens, mask, 1.0, scale * da, 0 * da, slack=40.0)
        assert (grad[:2] == 0).all() and (grad[-3:] == 0).all()
    z = _place(x, "plain").requires_grad_()
    (preference_loss(z, tokens.cuda(), ref.cuda(), offsets=offsets.cuda(), **kwargs).loss * scale).backward()
    _check_grad(z.grad, clean, tokens, mask, 1.0, scale * da, 0 * da, slack=40.0)


def test_preference_batched_and_wild_offsets():
    x, tokens, mask, _ = _make((4, 6), 1001, torch.float32)
    out, grad = preference_loss_grad(_place(x, "shifted"), tokens.cuda(), mask=mask.cuda())
    flat, flat_grad = preference_loss_grad(x.cuda().flatten(0, 1), tokens.cuda().flatten(), mask=mask.cuda().flatten(),
                                           offsets=torch.arange(0, 25, 6).cuda())
    # rows that start elsewhere within 16 bytes are summed in another order: each side is within 3e-5 + |log p| 2^-21 of
    # a p (|log p| < 40 here), and a within 3e-5
    assert (out.loss - flat.loss).abs() <= 3e-5 * flat.loss
    assert ((grad.reshape(24, -1) - flat_grad).abs() <= 2e-4 * flat_grad.abs()).all()
    # offsets beyond the rows are clamped: nothing outside the tensors is touched
    wild, wild_grad = preference_loss_grad(x.cuda().flatten(0, 1), tokens.cuda().flatten(),
                                           offsets=torch.tensor([-5, 6, 12, 18, 10 ** 9]).cuda())
    same, same_grad = preference_loss_grad(x.cuda().flatten(0, 1), tokens.cuda().flatten(),
                                           offsets=torch.arange(0, 25, 6).cuda())
    assert torch.equal(wild.loss, same.loss) and torch.equal(wild_grad, same_grad)


def test_empty_and_uncounted():
    z = torch.zeros(0, 9, device="cuda")
    t, f = torch.zeros(0, dtype=torch.long, device="cuda"), torch.zeros(0, device="cuda")
    assert token_logprobs(z, t)[0].shape == (0,)
    out, grad = token_policy_loss_grad(z, t, f, f)
    assert out.loss.item() == 0 and grad.shape == (0, 9)
    out, grad = preference_loss_grad(z, t, f, offsets=torch.zeros(1, dtype=torch.long, device="cuda"))
    assert out.loss.item() == 0 and out.seq_logps.shape == (0,)
    x, tokens, mask, _ = _make((5,), 700, torch.bfloat16)
    row = torch.ones(5, device="cuda")
    out, grad = token_policy_loss_grad(x.cuda(), tokens.cuda(), row, row, mask=(0 * mask).cuda().bool())
    assert out.loss.item() == 0 and out.entropy.item() == 0 and (grad == 0).all()


def test_offsets_beyond_32_bits():
    vocab, rows = 131072, 16400  # 2.15e9 elements
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    part = (torch.randn(3, vocab, generator=torch.Generator().manual_seed(0)) * 3).bfloat16()
    x[-3:] = part.cuda()
    tokens = torch.arange(rows, device="cuda")
    mask = torch.zeros(rows, dtype=torch.bool, device="cuda")
    mask[-3:] = True
    adv = torch.ones(rows, device="cuda")
    logp, _ = token_logprobs(x, tokens, mask=mask)
    tok, three = tokens[-3:].cpu(), torch.ones(3, dtype=torch.bool)
    _, want, _ = oracle.rows(part, tok, three, 1.0)
    assert ((logp[-3:].double().cpu() - want).abs() <= oracle.logp_bound(want)).all()
    out, grad = token_policy_loss_grad(x, tokens, logp, adv, mask=mask)
    _, _, _, da, db = oracle.policy(part, tok, logp[-3:].cpu(), torch.ones(3), None, None, lo=0.8, hi=1.2, kl_coef=0.0,
                                    kind="k3", entropy_coef=0.0, temperature=1.0)
    _check_grad(grad[-3:], part, tok, three, 1.0, da, db, slack=1.0)
    assert not grad[:-3].any()


def _inputs(seed, rows=300, vocab=5000):
    x, tokens, mask, g = _make((rows,), vocab, torch.bfloat16, seed=seed)
    old, adv = torch.randn(rows, generator=g) - 9, torch.randn(rows, generator=g)
    return [t.cuda() for t in (x, tokens, old, adv, mask)]


def _both(x, tokens, old, adv, mask):
    a, ga = token_policy_loss_grad(x, tokens, old, adv, ref_logp=old, mask=mask, kl_coef=0.1, entropy_coef=0.01)
    b, gb = preference_loss_grad(x, tokens, offsets=torch.arange(0, len(x) + 1, 50, device=x.device), mask=mask)
    return [*a, ga, *b, gb]


def test_capture_and_streams():
    """Two captured graphs replayed on two streams at once, and an eager call on a third, give the eager results."""
    inputs = [_inputs(s) for s in (1, 2, 3)]
    want = [[t.clone() for t in _both(*i)] for i in inputs]
    graphs, outs = [], []
    for i in inputs[:2]:
        _both(*i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_both(*i))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = _both(*inputs[2])
    torch.cuda.synchronize()
    for got, expected in zip((*outs, eager), want):
        assert all(torch.equal(a, b) for a, b in zip(got, expected))
    # a replay reads new inputs
    inputs[0][0].copy_(inputs[1][0])
    graphs[0].replay()
    fresh = _both(*inputs[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], fresh))


def test_autograd_forms_refuse_capture():
    x, tokens, old, adv, mask = _inputs(4, 8, 100)
    z = x.requires_grad_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: token_logprobs(z, tokens), lambda: token_policy_loss(z, tokens, old, adv),
                     lambda: preference_loss(z, tokens, offsets=tokens)):
            with pytest.raises(RuntimeError, match="capture"):
                call()


def test_autograd_twice_and_same_as_grad_form():
    x, tokens, old, adv, mask = _inputs(5)
    z = x.clone().requires_grad_()
    loss = token_policy_loss(z, tokens, old, adv, mask=mask).loss
    loss.backward(retain_graph=True)
    first = z.grad.clone()
    loss.backward()
    assert torch.equal(z.grad, first + first)
    _, grad = token_policy_loss_grad(x, tokens, old, adv, mask=mask)
    # both round the same value of the same fp32 accuracy to bfloat16
    assert (grad.float() - first.float()).abs().max() <= first.float().abs().max() * 2.0 ** -7
    with torch.no_grad():
        assert token_policy_loss(z, tokens, old, adv, mask=mask).loss.item() == pytest.approx(loss.item(), abs=1e-6)


def test_differentiable_once():
    x, tokens, old, adv, mask = _inputs(8, 8, 100)
    z = x.float().requires_grad_()
    for value in (token_logprobs(z, tokens)[0].sum(), token_policy_loss(z, tokens, old, adv).loss,
                  preference_loss(z, tokens, offsets=torch.tensor([0, 4, 8], device="cuda")).loss):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(value, z, create_graph=True)


def test_gradients_reach_leaves_through_views():
    """The means and log-probabilities of a loss carry no gradient; only one of two outputs may be used."""
    x, tokens, old, adv, mask = _inputs(9, 8, 100)
    z = x.float().requires_grad_()
    out = token_policy_loss(z, tokens, old, adv, mask=mask)
    assert out.loss.requires_grad and not any(t.requires_grad for t in out[1:])
    for pick in (0, 1):
        z.grad = None
        token_logprobs(z, tokens)[pick].sum().backward()
        assert torch.isfinite(z.grad).all() and z.grad.abs().sum() > 0
    pref = preference_loss(z.view(2, 4, 100), tokens.view(2, 4))
    assert pref.loss.requires_grad and not any(t.requires_grad for t in pref[1:])


@pytest.mark.parametrize("estimator", ["k1", "k2", "k3"])
def test_infinite_divergence_without_weight(estimator):
    """A reference that excludes a token makes the divergence infinite; with kl_coef 0 the loss does not see it."""
    x, tokens, old, adv, mask = _inputs(10)
    ref = old.clone()
    ref[mask.nonzero()[0]] = float("-inf")
    args = (x, tokens, old, adv)
    plain, grad = token_policy_loss_grad(*args, mask=mask)
    out, with_ref = token_policy_loss_grad(*args, ref_logp=ref, mask=mask, kl_estimator=estimator)
    assert not torch.isfinite(out.kl) and torch.equal(out.loss, plain.loss) and torch.equal(with_ref, grad)
    z = x.clone().requires_grad_()
    loss = token_policy_loss(z, tokens, old, adv, ref_logp=ref, mask=mask, kl_estimator=estimator).loss
    loss.backward()
    assert torch.equal(loss.detach(), plain.loss) and torch.isfinite(z.grad).all()


def test_scale_on_the_device():
    x, tokens, old, adv, mask = _inputs(6)
    _, one = token_policy_loss_grad(x, tokens, old, adv, grad_scale=8.0)
    _, two = token_policy_loss_grad(x, tokens, old, adv, grad_scale=torch.tensor(8.0, device="cuda"))
    assert torch.equal(one, two)
    with pytest.raises(ValueError, match="scale"):
        token_policy_loss_grad(x, tokens, old, adv, grad_scale=torch.tensor(8.0))


@pytest.mark.parametrize("error,text,change", REFUSALS)
def test_policy_refusals(error, text, change):
    refuse("cuda", error, text, change)


def test_preference_refusals():
    refuse_preference("cuda")
    x, tokens, old, adv, mask = _inputs(7, 8, 100)
    with pytest.raises(ValueError, match="device"):
        token_logprobs(x, tokens.cpu())


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_weights_only_select(dtype):
    """A float mask decides which rows count; neither the log-probabilities nor their gradients are weighted by it."""
    x, tokens, mask, g = _make((40,), 1001, dtype, seed=11)
    w = torch.where(mask, torch.linspace(-2.0, 3.0, 40), 0.0)
    a, b = torch.randn(40, generator=g), torch.randn(40, generator=g) * 0.3
    for how in ("plain", "offset"):
        z = _place(x, how).requires_grad_()
        logp, entropy = token_logprobs(z, tokens.cuda(), mask=w.cuda())
        _, want, _ = oracle.rows(x, tokens, mask, 1.0)
        want = torch.where(mask, want, 0.0)
        assert ((logp.detach().double().cpu() - want).abs() <= oracle.logp_bound(want)).all()
        grad, = torch.autograd.grad((logp, entropy), z, (a.cuda(), b.cuda()))
        _check_grad(grad, x, tokens, mask, 1.0, a.double(), b.double())


def _check_far_grad(got, x, tokens, temperature, a, b, slack=0.0):
    """``_check_grad`` where probabilities reach below 2^-126 (all rows count). A p is 2^q times a number in [1/2, 2], and
    2^q below 2^-126 is flushed to zero: that takes p (|a| + |b| (|log p| + H)) / T off an element with p below 2^-125."""
    counted = torch.ones(tokens.shape, dtype=torch.bool)
    want, bound = oracle.logits_grad(x, tokens, counted, temperature, a, b)
    log_p, _, entropy = oracle.rows(x, tokens, counted, temperature)
    safe = torch.where(log_p == float("-inf"), 0.0, log_p)
    size = log_p.exp() * (a.abs()[:, None] + b.abs()[:, None] * (safe.abs() + entropy[:, None])) / temperature
    bound = bound * (1 + slack) + want.abs() * 3e-5 * slack + torch.where(log_p < -125 * math.log(2.0), size, 0.0)
    assert got.dtype == x.dtype and got.shape == x.shape
    far = (got.double().cpu() - want).abs() - bound
    assert (far <= oracle.rounding(want, x.dtype) * 1.01).all(), far.max()


def check_extreme(dtype, vocab, temperature, top):
    """Log-probabilities, entropies, gradients and the policy loss of ``extreme_rows``."""
    if dtype == torch.float16 and abs(top) > 6e4:
        return
    x, best = extreme_rows(dtype, top, vocab)
    counted = torch.ones(8, dtype=torch.bool)
    any_token = torch.randint(vocab, (8,), generator=torch.Generator().manual_seed(1))
    any_token = torch.where(x.gather(1, any_token[:, None])[:, 0] > -3e38 / 4, any_token, best)
    g = torch.Generator().manual_seed(2)
    a, b = torch.randn(8, generator=g), torch.randn(8, generator=g) * 0.3
    for tokens in (best, any_token):
        z = _place(x, "offset").requires_grad_()
        logp, entropy = token_logprobs(z, tokens.cuda(), temperature=temperature)
        _, want, want_h = oracle.rows(x, tokens, counted, temperature)
        assert ((logp.detach().double().cpu() - want).abs() <= oracle.logp_bound(want)).all()
        assert ((entropy.detach().double().cpu() - want_h).abs() <= 2 * oracle.logp_bound(want_h) + 2e-5).all()
        # a small temperature multiplies the gradient: kept inside fp16's range
        scale = min(1.0, temperature * 1e3)
        grad, = torch.autograd.grad((logp, entropy), z, (scale * a.cuda(), scale * b.cuda()))
        _check_far_grad(grad, x, tokens, temperature, scale * a.double(), scale * b.double())
    # log p of the largest column is above -13 here: old_logp and the ratio are ordinary numbers
    _, want, _ = oracle.rows(x, best, counted, temperature)
    old, adv = want.float() + 0.1, torch.linspace(-1, 1, 8)
    for entropy_coef in (0.0, 0.1):
        out, grad = token_policy_loss_grad(x.cuda(), best.cuda(), old.cuda(), adv.cuda(), entropy_coef=entropy_coef,
                                           temperature=temperature, grad_scale=scale)
        loss, _, _, da, db = oracle.policy(x, best, old, adv, None, None, lo=0.8, hi=1.2, kl_coef=0.0, kind="k3",
                                           entropy_coef=entropy_coef, temperature=temperature)
        # logp and H within 3e-5, slopes of at most 2 |A| + 1
        assert abs(out.loss.item() - loss) <= 1e-4
        _check_far_grad(grad, x, best, temperature, scale * da, scale * db, slack=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [37, 5000, 131075])
@pytest.mark.parametrize("temperature,top", [(1.0, 2000.0), (1.0, 5e4), (1.0, -5e4), (0.5, -6e4), (1e-3, 30.0)])
def test_large_logits(dtype, vocab, temperature, top):
    """Logits far from zero are as exact as others: the shift of the exponents is one number for all of a row's columns."""
    check_extreme(dtype, vocab, temperature, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [37, 5000, 131075])
@pytest.mark.parametrize("temperature,top", RANGES)
def test_large_logits_over_temperature(dtype, vocab, temperature, top):
    """Finite logits give finite results whatever their size over the temperature (the spacing of fp32 numbers as large
    as |z| / T is far above one here, so the sums have to be of differences)."""
    check_extreme(dtype, vocab, temperature, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [0.5, 0.8, 1.0, 2.0])
def test_token_at_the_lowest_value(dtype, temperature):
    """A token whose column was masked with its type's lowest value: its log-probability is that value over T, or -inf
    where this leaves fp32's range; never NaN."""
    x, tokens, _, _ = _make((4,), 501, dtype, seed=12)
    x[1, tokens[1]] = x[2, tokens[2]] = torch.finfo(dtype).min
    logp, entropy = token_logprobs(x.cuda(), tokens.cuda(), temperature=temperature)
    _, want, want_h = oracle.rows(x, tokens, torch.ones(4, dtype=torch.bool), temperature)
    inf = want < -torch.finfo(torch.float32).max
    assert inf.tolist() == [False, temperature < 1, temperature < 1, False]
    assert torch.equal(logp.cpu()[inf], torch.full((int(inf.sum()),), float("-inf")))
    assert ((logp.double().cpu() - want).abs() <= oracle.logp_bound(want))[~inf].all()
    assert ((entropy.double().cpu() - want_h).abs() <= 2 * oracle.logp_bound(want_h) + 2e-5).all()
    old = torch.where(want < -100, -5.0, want).float()  # the ratio of an excluded token is zero
    out, grad = token_policy_loss_grad(x.cuda(), tokens.cuda(), old.cuda(), torch.ones(4, device="cuda"),
                                       temperature=temperature)
    assert out.loss.item() == pytest.approx(-0.5, abs=1e-4) and torch.isfinite(grad.float()).all()


@pytest.mark.parametrize("shape", [(0,), (0, 5), (3, 0)])
def test_backward_without_rows(shape):
    z = torch.zeros(*shape, 9, device="cuda", requires_grad=True)
    t, f = torch.zeros(shape, dtype=torch.long, device="cuda"), torch.zeros(shape, device="cuda")
    losses = [token_policy_loss(z, t, f, f, ref_logp=f, kl_coef=0.1, entropy_coef=c).loss for c in (0.0, 0.1)]
    losses.append(sum(x.sum() for x in token_logprobs(z, t)))
    if shape != (3, 0):  # three sequences are no pairs
        losses.append(preference_loss(z, t, offsets=None if len(shape) == 2 else t.new_zeros(1)).loss)
    for loss in losses:
        grad, = torch.autograd.grad(loss, z)
        assert loss.item() == 0 and grad.shape == z.shape


def test_uint8_masks_select():
    x, tokens, old, adv, mask = _inputs(13)
    for call in (lambda m: token_policy_loss_grad(x, tokens, old, adv, mask=m, reduction="sum"),
                 lambda m: preference_loss_grad(x.view(6, 50, -1), tokens.view(6, 50), mask=m.view(6, 50))):
        a, b = call(mask.to(torch.uint8) * 3), call(mask)
        assert all(torch.equal(p, q) for p, q in zip((*a[0], a[1]), (*b[0], b[1])))


def test_only_logits_get_gradients():
    only_logits_get_gradients("cuda")


def test_forward_mode_is_refused():
    """The kernels have no forward-mode derivative: a tangent of the logits is refused, not dropped."""
    x, tokens, old, adv, mask = _inputs(14, 8, 100)
    z = x.float()
    forms = (lambda q: token_logprobs(q, tokens)[0], lambda q: token_policy_loss(q, tokens, old, adv).loss,
             lambda q: token_policy_loss_grad(q, tokens, old, adv)[0].loss,
             lambda q: preference_loss(q.view(2, 4, -1), tokens.view(2, 4)).loss,
             lambda q: preference_loss_grad(q.view(2, 4, -1), tokens.view(2, 4))[0].loss)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(z, torch.ones_like(z))
        for form in forms:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                form(dual)
            form(z)


def test_decided_pairs():
    decided_pairs("cuda")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,smoothing,average", [("sigmoid", 0.0, False), ("sigmoid", 0.1, False), ("sigmoid", 0.3, True),
                                                    ("hinge", 0.0, False), ("hinge", 0.0, True), ("ipo", 0.0, False),
                                                    ("ipo", 0.0, True)])
def test_preference_losses(dtype, kind, smoothing, average):
    """Each loss's value in all of its forms, for pairs on both sides of its border."""
    x, tokens, mask, _ = _make((8, 9), 301, dtype, seed=15)
    bounds = [(9 * i, 9 * i + 9) for i in range(8)]
    lps = oracle.preference(x, tokens, None, bounds, mask, beta=0.2, average=average)[1]
    h = torch.tensor([-6.0, -0.4, 0.7, 9.0])  # differences of rewards
    ref = lps.float()
    ref[0::2] -= h / 0.2
    loss = oracle.preference(x, tokens, ref, bounds, mask, beta=0.2, smoothing=smoothing, kind=kind, average=average)[0]
    kwargs = dict(mask=mask.cuda(), beta=0.2, label_smoothing=smoothing, loss_type=kind, average=average)
    # a sequence's log-probability is off by at most 9 bounds of a row's (|logp| < 25: 1.6e-5 each), h by twice beta times
    # that (6e-5) and its own rounding in fp32 (2^-21); the slopes by h are at most 1 (sigmoid, hinge) and
    # 2 (|h| + 0.5) / beta^2 = 475 (ipo), and the value is rounded
    tol = (6e-5 + 2.0 ** -21) * (475 if kind == "ipo" else 1) + 2.0 ** -22 * abs(loss)
    forms = [preference_loss_grad(x.cuda(), tokens.cuda(), ref.cuda(), **kwargs)[0].loss,
             preference_loss(x.cuda(), tokens.cuda(), ref.cuda(), **kwargs).loss,
             preference_loss(x.cuda().requires_grad_(), tokens.cuda(), ref.cuda(), **kwargs).loss,
             preference_loss(x.cuda().flatten(0, 1), tokens.cuda().flatten(), ref.cuda(),
                             offsets=torch.arange(0, 73, 9).cuda(), **(kwargs | {"mask": mask.cuda().flatten()})).loss]
    for got in forms:
        assert abs(got.item() - loss) <= tol


def test_clipped_ratios():
    clipped_ratios("cuda")


def test_decreasing_offsets_give_nan():
    """Two sequences may not share a row: the kernel says so, since the host does not wait for the offsets."""
    x, tokens, mask, _ = _make((4000,), 40, torch.float32, seed=16)
    mask = mask.cuda()
    many = torch.arange(0, 4001, 2)
    many[1990] = many[1988] - 1
    for offsets in ([0, 10, 5, 20, 20], [5, 3, 20], many.tolist(), [0, 10, 5000, 3999, 4000]):
        out, grad = preference_loss_grad(x.cuda(), tokens.cuda(), offsets=torch.tensor(offsets).cuda(), mask=mask)
        assert out.loss.isnan() and all(t.isnan().all() for t in out[1:4])
        assert grad[mask].isnan().all() and (grad[~mask] == 0).all()
        z = x.cuda().requires_grad_()
        preference_loss(z, tokens.cuda(), offsets=torch.tensor(offsets).cuda().int(), mask=mask).loss.backward()
        assert z.grad[mask].isnan().all()
