"""AdamW over many tensors on the CPU: the update against 64 bits, the 8-bit codes, the optimizer form, refusals."""

import copy

import numpy as np
import pytest
import torch

import token_oracle as oracle
from tt_rsl_rl_b200.ops.adamw import BLOCK, CODES, AdamW, AdamW8bit, AdamWPlan
from tt_rsl_rl_b200.utils.utils import resolve_optimizer

HYPER = {"lr": 1e-2, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 0.1}
SHAPES = [(3, 5), (1,), (257,), (0,), (16, 32), (1023,)]


def make_plan(dtype, bits, device="cpu", shapes=SHAPES, seed=0, offset=0):
    """Parameters with gradients and the tensors of their plan. ``offset`` shifts every tensor by that many elements in
    its storage."""
    g = torch.Generator().manual_seed(seed)

    def rand(shape, scale, dt=torch.float32):
        n = int(torch.tensor(shape).prod())
        flat = torch.zeros(n + offset, dtype=dt, device=device)
        flat[offset:] = (torch.randn(n, generator=g) * scale).to(dt).to(device)
        return flat[offset:].view(shape)

    params = [rand(s, 0.5, dtype) for s in shapes]
    for p in params:
        p.grad = rand(p.shape, 0.1, dtype)
    steps = torch.tensor([float(3 + i) for i in range(len(shapes))], device=device)
    kwargs = {}
    if bits == 32:
        m, v = [rand(s, 0.05) for s in shapes], [rand(s, 0.1).square_() for s in shapes]
    else:
        blocks = [-(-p.numel() // BLOCK) for p in params]
        m = [rand(s, 100.0).clamp_(-448, 448).to(CODES) for s in shapes]
        v = [rand(s, 100.0).abs_().clamp_(0, 448).to(CODES) for s in shapes]
        if offset:  # .to() made new storage: shift it again
            m, v = ([torch.cat([x.new_zeros(offset, dtype=torch.uint8), x.flatten().view(torch.uint8)])[offset:]
                     .view(CODES).view(x.shape) for x in xs] for xs in (m, v))
        kwargs = {"exp_avg_scales": [torch.full((b,), 1e-3, device=device) for b in blocks],
                  "exp_avg_sq_scales": [torch.full((b,), 2e-3, device=device) for b in blocks]}
    if dtype == torch.bfloat16:
        kwargs["low_bits"] = [torch.randint(-2 ** 15, 2 ** 15, s, generator=g).to(torch.int16).to(device) for s in shapes]
    return params, m, v, steps, kwargs


def whole(p, low):
    """The float32 weight of a bfloat16 parameter."""
    return ((p.view(torch.int16).int() << 16) + low.int()).view(torch.float32)


def state_values(m, v, kwargs, i):
    if "exp_avg_scales" not in kwargs:
        return m[i].clone(), v[i].clone()
    n = m[i].numel()
    ms, vs = (kwargs[k][i].repeat_interleave(BLOCK)[:n].view(m[i].shape) for k in ("exp_avg_scales", "exp_avg_sq_scales"))
    return m[i].float() * ms, (v[i].float() * vs).square()


def check_step(dtype, bits, max_norm, device="cpu", offset=0, maximize=False):
    """One step against 64 bits. Bounds: each of the few fp32 operations is off by 2^-24 of its result, so moments and
    weights by 2^-21 of the sizes that they are made of; bfloat16 parameters hold the rounding of the weight."""
    params, m, v, steps, kwargs = make_plan(dtype, bits, device, offset=offset)
    before = [(p.clone() if dtype == torch.float32 else whole(p, low)) for p, low in
              zip(params, kwargs.get("low_bits", params))]
    old = [state_values(m, v, kwargs, i) for i in range(len(params))]
    norm = AdamWPlan(params, m, v, steps, **kwargs).step(max_grad_norm=max_norm, maximize=maximize, seed=5, **HYPER)
    clip = 1.0
    if max_norm:
        want = torch.cat([p.grad.flatten().double() for p in params]).norm()
        assert abs(norm.item() - want.item()) <= 2.0 ** -23 * want.item()
        clip = min(1.0, max_norm / (want.item() + 1e-6))
    else:
        assert norm is None
    assert steps.tolist() == [4.0 + i for i in range(len(params))]
    for i, p in enumerate(params):
        wp, wm, wv = oracle.adamw(before[i], p.grad, *old[i], 4 + i, clip=-clip if maximize else clip, **HYPER)
        got = p if dtype == torch.float32 else whole(p, kwargs["low_bits"][i])
        size = wp.abs() + before[i].abs() + (wp - before[i]).abs() * 4
        assert ((got.double() - wp).abs() <= size * 2.0 ** -21 + 1e-9).all()
        if dtype == torch.bfloat16:
            assert ((p.double() - got.double()).abs() <= got.double().abs() * 2.0 ** -8 + 1e-38).all()
        if bits == 32:
            gm = old[i][0].abs() + p.grad.abs()
            assert ((m[i] - wm).abs() <= gm * 2.0 ** -21).all()
            assert ((v[i] - wv).abs() <= wv * 2.0 ** -21).all()
        else:
            gm, gv = state_values(m, v, kwargs, i)
            rep = lambda x: x.repeat_interleave(BLOCK)[:p.numel()].view(p.shape)  # noqa: E731
            ms, vs = rep(kwargs["exp_avg_scales"][i]), rep(kwargs["exp_avg_sq_scales"][i])
            # a code is one of the two neighbours: an eighth of the binade above 2^-6, 2^-9 below, in units of the scale
            assert ((gm - wm).abs() <= wm.abs() / 8 * (1 + 1e-5) + ms * 2.0 ** -9).all()
            root = wv.sqrt()
            assert ((gv.double().sqrt() - root).abs() <= root / 8 * (1 + 1e-5) + vs * 2.0 ** -9).all()
            assert (gv[root > 0] > 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e4])
def test_step_matches_64_bits(dtype, bits, max_norm):
    check_step(dtype, bits, max_norm)


def test_maximize():
    check_step(torch.float32, 32, 0.5, maximize=True)


def rounding_statistics(device):
    """4096 draws of the same block: the mean of the stored moments is the moment. An element's stored value has a
    standard deviation of at most half the distance of two codes (d), the mean of n draws of d / (2 sqrt(n)); five of
    those leave 512 means outside with a chance below 1e-3."""
    n, draws = 256, 4096
    one = torch.Generator().manual_seed(2)
    grad = torch.randn(n, generator=one).to(device)
    grad[0] = 40.0  # most codes of the block are far below its largest
    p = torch.zeros(n * draws, device=device)
    p.grad = grad.repeat(draws)
    m, v = torch.zeros(n * draws, device=device).to(CODES), torch.zeros(n * draws, device=device).to(CODES)
    ms, vs = torch.zeros(draws, device=device), torch.zeros(draws, device=device)
    AdamWPlan([p], [m], [v], torch.zeros(1, device=device), exp_avg_scales=[ms], exp_avg_sq_scales=[vs]).step(seed=3, **HYPER)
    m_all = (m.float().view(draws, n) * ms[:, None]).double()
    v_all = (v.float().view(draws, n) * vs[:, None]).double().square()
    want_m, want_v = 0.1 * grad.double(), 0.01 * grad.double().square()
    for got, want, gap in ((m_all, want_m, want_m.abs() / 8 + ms[0].double() * 2.0 ** -9),
                           (v_all, want_v, want_v * (2 / 8 + 1 / 64) + 2 * want_v.sqrt() * vs[0].double() * 2.0 ** -9
                            + (vs[0].double() * 2.0 ** -9) ** 2)):
        far = (got.mean(0) - want).abs()
        # 2^-16: the resolution of the random numbers, in distances of codes
        assert (far <= gap * (5 / (2 * draws ** 0.5) + 2.0 ** -16) + want.abs() * 1e-5).all()
        assert got.std(0)[1:].gt(0).float().mean() > 0.9  # the draws differ


def test_codes_are_right_on_average():
    rounding_statistics("cpu")


def zeros_written(device):
    """Weights set to zero (of either sign) from outside meet lower bits of another weight."""
    p = torch.randn(4096, device=device).bfloat16()
    p.grad = torch.randn(4096, device=device).bfloat16()
    opt = AdamW([p], lr=1e-3, weight_decay=0.0)
    opt.step()
    low = opt.state[p]["low_bits"]
    assert (low < 0).any() and (low > 0).any()
    p[:2048] = 0.0
    p[1024:2048] *= -1.0
    p.grad = torch.zeros_like(p)
    opt.step()
    assert torch.isfinite(p).all() and (p[:2048].abs() < 2e-3).all()


def test_zeros_written_from_outside():
    zeros_written("cpu")


def test_optimizer_follows_torch():
    torch.manual_seed(0)
    a = torch.nn.Sequential(torch.nn.Linear(7, 9), torch.nn.Tanh(), torch.nn.Linear(9, 2))
    b = copy.deepcopy(a)
    mine, theirs = AdamW(a.parameters(), **HYPER), torch.optim.AdamW(b.parameters(), **HYPER)
    for i in range(5):
        x = torch.randn(4, 7)
        for model, opt in ((a, mine), (b, theirs)):
            opt.zero_grad()
            model(x).square().sum().backward()
            if i == 2:
                next(model.parameters()).grad = None  # a parameter without gradient keeps its step count
            opt.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.allclose(p, q, atol=1e-6)
    again = AdamW(a.parameters(), **HYPER)
    again.load_state_dict(theirs.state_dict())
    x = torch.randn(4, 7)
    for model, opt in ((a, again), (b, theirs)):
        opt.zero_grad()
        model(x).square().sum().backward()
        opt.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.allclose(p, q, atol=1e-6)
    back = torch.optim.AdamW(b.parameters(), **HYPER)
    back.load_state_dict(again.state_dict())


def resume(device, dtype, bits):
    """A resumed optimizer takes the step that the original takes, bit for bit."""
    torch.manual_seed(1)
    p = torch.randn(300, 3, device=device, dtype=dtype).requires_grad_()
    q = p.detach().clone().requires_grad_()
    first = AdamW([p], state_bits=bits, max_grad_norm=1.0, **HYPER)
    grads = [torch.randn_like(p) for _ in range(4)]
    for g in grads[:3]:
        p.grad = g
        first.step()
    with torch.no_grad():
        q.copy_(p)
    second = AdamW([q], state_bits=bits, max_grad_norm=1.0, **HYPER)
    second.load_state_dict(copy.deepcopy(first.state_dict()))
    for param, opt in ((p, first), (q, second)):
        param.grad = grads[3].clone()
        opt.step()
    assert torch.equal(p, q) and torch.equal(first.grad_norm, second.grad_norm)
    for key, x in first.state[p].items():
        y = second.state[q][key]
        assert x.dtype == y.dtype and torch.equal(x.float(), y.float()), key


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_resume(dtype, bits):
    resume("cpu", dtype, bits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_of_another_layout(dtype):
    """32-bit states are laid out anew; the scales of 8-bit ones belong to an order in memory, so those are refused, and
    so are states of another shape."""
    torch.manual_seed(2)
    values, grads = torch.randn(2, 3, 20, 7).to(dtype), [torch.randn(2, 3, 20, 7).to(dtype) for _ in range(2)]
    p = values.contiguous(memory_format=torch.channels_last).requires_grad_()
    q = values.clone().requires_grad_()
    for bits in (32, 8):
        first, second = AdamW([p], state_bits=bits, **HYPER), AdamW([q], state_bits=bits, **HYPER)
        p.grad = grads[0]
        first.step()
        with torch.no_grad():
            q.copy_(p)
        second.load_state_dict(first.state_dict())
        p.grad, q.grad = grads[1], grads[1]
        if bits == 8:
            with pytest.raises(ValueError, match="order in memory"):
                second.step()
            continue
        first.step()
        second.step()
        assert torch.equal(p, q)
        if dtype == torch.bfloat16:
            assert torch.equal(first.state[p]["low_bits"], second.state[q]["low_bits"])
    row = torch.ones(7).requires_grad_()
    third = AdamW([row])
    wide = AdamW([torch.ones(1).requires_grad_()])
    wide.param_groups[0]["params"][0].grad = torch.ones(1)
    wide.step()
    third.load_state_dict(wide.state_dict())
    row.grad = torch.ones(7)
    with pytest.raises(ValueError, match="shape"):
        third.step()


def test_states_of_another_update():
    """What AdamW's step would leave out is refused when it is loaded; groups of older dictionaries lack settings."""
    p = torch.ones(5).requires_grad_()
    p.grad = torch.ones(5)
    theirs = torch.optim.AdamW([p], amsgrad=True)
    theirs.step()
    with pytest.raises(ValueError, match="amsgrad"):
        AdamW([p]).load_state_dict(theirs.state_dict())
    theirs = torch.optim.Adam([p], weight_decay=0.1)
    theirs.step()
    with pytest.raises(ValueError, match="decoupled"):
        AdamW([p]).load_state_dict(theirs.state_dict())
    theirs = torch.optim.Adam([p])
    theirs.step()
    state = theirs.state_dict()
    del state["param_groups"][0]["maximize"]
    ours = AdamW([p])
    ours.load_state_dict(state)
    q = p.detach().clone().requires_grad_()
    q.grad = p.grad.clone()
    again = torch.optim.Adam([q])
    again.load_state_dict(theirs.state_dict())
    ours.step()
    again.step()
    assert torch.allclose(p, q, atol=1e-6)


def test_groups_share_the_norm():
    a, b = torch.ones(3).requires_grad_(), torch.ones(4, dtype=torch.bfloat16).requires_grad_()
    opt = AdamW([{"params": [a], "lr": 0.0}, {"params": [b]}], lr=0.1, max_grad_norm=1.0, weight_decay=0.0)
    a.grad, b.grad = torch.full((3,), 2.0), torch.full((4,), 1.0, dtype=torch.bfloat16)
    opt.step()
    assert abs(opt.grad_norm - 4.0) < 1e-6
    assert (a == 1).all() and (b < 1).all()


def refuse_plans(device):
    def plan(change=lambda *a: None, dtype=torch.float32, bits=32):
        params, m, v, steps, kwargs = make_plan(dtype, bits, device, shapes=[(4, 6), (300,)])
        x = {"params": params, "m": m, "v": v, "steps": steps, **kwargs}
        change(x)
        return AdamWPlan(x.pop("params"), x.pop("m"), x.pop("v"), x.pop("steps"), **x)

    for error, text, change, kwargs in [
        (ValueError, "no parameters", lambda x: x.update(params=[], m=[], v=[]), {}),
        (ValueError, "one exp_avg", lambda x: x.update(m=x["m"][:1]), {}),
        (TypeError, "parameters must be", lambda x: x.update(params=[p.half() for p in x["params"]]), {}),
        (TypeError, "states must be", lambda x: x.update(m=[p.double() for p in x["m"]]), {}),
        (TypeError, "exp_avg_sq 0", lambda x: x.update(v=[p.double() for p in x["v"]]), {}),
        (TypeError, "share a type", lambda x: x.update(params=[x["params"][0], x["params"][1].bfloat16()]), {}),
        (ValueError, "shape and strides", lambda x: x["m"].__setitem__(0, x["m"][0].t().contiguous().t()), {}),
        (ValueError, "gaps or overlaps", lambda x: x["params"].__setitem__(0, torch.zeros(4, 12, device=device)[:, ::2]), {}),
        (ValueError, "steps must be", lambda x: x.update(steps=x["steps"][:1]), {}),
        (ValueError, "need their scales", lambda x: x.pop("exp_avg_scales"), {"bits": 8}),
        (ValueError, "scales", lambda x: x["exp_avg_scales"].__setitem__(1, torch.zeros(1, device=device)), {"bits": 8}),
        (ValueError, "low_bits", lambda x: x.pop("low_bits"), {"dtype": torch.bfloat16}),
        (ValueError, "share memory", lambda x: x.update(params=[x["params"][0]] * 2, m=[x["m"][0], x["m"][0].clone()],
                                                        v=[x["v"][0], x["v"][0].clone()]), {}),
        (ValueError, "share memory", lambda x: x["v"].__setitem__(1, x["m"][1]), {}),
    ]:
        with pytest.raises(error, match=text):
            plan(change, **kwargs)
    good = plan()
    for text, kwargs in [("lr", {"lr": -1.0}), ("betas", {"lr": 0.1, "betas": (0.9, 1.0)}), ("eps", {"lr": 0.1, "eps": -1}),
                         ("weight_decay", {"lr": 0.1, "weight_decay": -1}), ("max_grad_norm", {"lr": 0.1, "max_grad_norm": 0.0}),
                         ("seed", {"lr": 0.1, "seed": -1})]:
        with pytest.raises(ValueError, match=text):
            good.step(**kwargs)


def test_refusals():
    refuse_plans("cpu")
    p = torch.zeros(3).requires_grad_()
    with pytest.raises(ValueError, match="state_bits"):
        AdamW([p], state_bits=4)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        q = torch.zeros(3, dtype=torch.float64).requires_grad_()
        q.grad = torch.zeros_like(q)
        AdamW([q]).step()
    opt = AdamW8bit([p])
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="does not belong to 8-bit"):
        other = AdamW([p])
        other.step()
        opt.load_state_dict(other.state_dict())
        opt.step()


def test_names_resolve():
    assert resolve_optimizer("adamw_fused") is AdamW and resolve_optimizer("AdamW_8bit") is AdamW8bit
    assert resolve_optimizer("adamw") is torch.optim.AdamW


def test_hooks_of_loading():
    """A hook before loading changes what is loaded, one behind it what was; types stay those of the states."""
    p, q = (torch.ones(300, dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    first, second = AdamW([p]), AdamW([q])
    p.grad = torch.full_like(p, 0.5)
    first.step()

    def before(_, state):
        state = copy.deepcopy(state)
        state["state"][0]["exp_avg"].mul_(2.0)
        return state

    second.register_load_state_dict_pre_hook(before)
    second.register_load_state_dict_post_hook(lambda opt: opt.state[q]["exp_avg_sq"].zero_())
    second.load_state_dict(first.state_dict())
    assert second.state[q]["exp_avg"].dtype == torch.float32
    assert torch.equal(second.state[q]["exp_avg"], 2 * first.state[p]["exp_avg"])
    assert (second.state[q]["exp_avg_sq"] == 0).all() and (first.state[p]["exp_avg_sq"] > 0).all()
    refused = torch.optim.AdamW([p], amsgrad=True)
    refused.register_load_state_dict_pre_hook(lambda *_: None)
    third = AdamW([q])
    third.register_load_state_dict_pre_hook(lambda _, state: {**state, "param_groups": [
        {**g, "amsgrad": False} for g in state["param_groups"]]})
    third.load_state_dict({"state": {}, "param_groups": refused.state_dict()["param_groups"]})


def test_codes_without_scales_are_refused():
    """8-bit codes mean nothing without their scales: they are not taken as zero."""
    p = torch.ones(300).requires_grad_()
    p.grad = torch.ones(300)
    first = AdamW8bit([p])
    first.step()
    for key in ("exp_avg_scale", "exp_avg_sq_scale"):
        state = copy.deepcopy(first.state_dict())
        del state["state"][0][key]
        second = AdamW8bit([p])
        second.load_state_dict(state)
        with pytest.raises(ValueError, match=key):
            second.step()


def test_roots_are_rounded():
    """Roots and quotients are correctly rounded, as the kernels' roots are (those of PyTorch's CPU operations may be a step
    off)."""
    gen = torch.Generator().manual_seed(6)
    m, v = torch.randn(1 << 20, generator=gen), torch.rand(1 << 20, generator=gen) * 10
    p = torch.zeros(1 << 20)
    p.grad = torch.zeros(1 << 20)
    one = np.float32
    want = -(m.numpy() * one(0.5) / (np.sqrt(v.numpy() * one(0.75)) * one(2.0) + one(1e-8)))
    # lr / (1 - b1) = 1, 1 / sqrt(1 - b2) = 2
    AdamWPlan([p], [m], [v], torch.zeros(1)).step(lr=0.5, betas=(0.5, 0.75), eps=1e-8, weight_decay=0.0)
    assert (p.numpy() == want).all()


def spikes(device):
    """A finite gradient whose square leaves fp32's range makes its block's second moment infinite: the block's weights
    stay where they are, the other blocks do not see it."""
    ends = []
    for spike in (1.0, 1e25):
        p = torch.ones(600, device=device).requires_grad_()
        opt = AdamW8bit([p], weight_decay=0.0)
        for step in range(3):
            p.grad = torch.linspace(-1, 1, 600, device=device)
            p.grad[3] = spike if step == 0 else 1.0
            opt.step()
            if step == 0:
                held = p.detach()[:256].clone()
        assert opt.state[p]["exp_avg_sq_scale"].isinf().tolist() == [spike > 1, False, False]
        ends.append((held, p.detach().clone()))
    assert torch.equal(ends[0][1][256:], ends[1][1][256:])
    assert torch.equal(ends[1][1][:256], ends[1][0]) and torch.isfinite(ends[1][0]).all()


def test_spikes():
    spikes("cpu")
