"""The AdamW kernels: 64-bit definition, bit-exactness with the CPU path, odd tensors, many tensors, capture."""

import copy

import numpy as np
import pytest
import torch

from test_adamw import (HYPER, SHAPES, check_step, make_plan, refuse_plans, resume, rounding_statistics, spikes, whole,
                        zeros_written)
from tt_rsl_rl_b200.ops.adamw import CODES, AdamW, AdamW8bit, AdamWPlan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e4])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_step_matches_64_bits(dtype, bits, max_norm, offset):
    check_step(dtype, bits, max_norm, "cuda", offset=offset)


def _bytes(x):
    return x.detach().cpu().contiguous().view(-1).view(torch.uint8)


def _same_weight(a, b, before):
    """Moments, codes and scales come from the same correctly rounded operations on both sides. In the weight's update
    the CPU's loops may contract a product and a sum. An intermediate that differs by one unit in the last place moves
    the rounding of each later operation by at most one unit: denominator, quotient, product and difference, so four
    units (2^-23 each) of numbers no larger than the weight before and after together."""
    size = b.cpu().double().abs() + before.cpu().double().abs()
    return ((a.cpu().double() - b.cpu().double()).abs() <= size * 4 * 2.0 ** -23).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_same_states_as_on_the_cpu(dtype, bits):
    shapes = SHAPES + [(70000,), (513, 129)]
    sides = []
    for device in ("cpu", "cuda"):
        params, m, v, steps, kwargs = make_plan(dtype, bits, device, shapes=shapes)
        before = [p.float() for p in params] if dtype == torch.float32 else [
            whole(p, x) for p, x in zip(params, kwargs["low_bits"])]
        before = [p.clone() for p in before]
        norm = AdamWPlan(params, m, v, steps, first_stream=9, **kwargs).step(max_grad_norm=1.0, seed=2 ** 40 + 3, **HYPER)
        low = kwargs.pop("low_bits", None)
        weights = params if low is None else [whole(p, x) for p, x in zip(params, low)]
        sides.append(([norm, steps, *m, *v, *(t for k in sorted(kwargs) for t in kwargs[k])], weights))
    assert all(torch.equal(_bytes(a), _bytes(b)) for a, b in zip(sides[0][0], sides[1][0]))
    assert all(_same_weight(a, b, c) for a, b, c in zip(sides[1][1], sides[0][1], before))


def test_codes_are_right_on_average():
    rounding_statistics("cuda")


@pytest.mark.parametrize("count", [39, 41, 400, 401, 1203])
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(count, bits):
    """Lists over one launch's table, tensors without a gradient among them."""
    shapes = [(1 + (37 * i) % 700,) for i in range(count)]
    params, m, v, steps, kwargs = make_plan(torch.float32, bits, "cuda", shapes=shapes)
    for p in params[::7]:
        p.grad = None
    clones = [copy.deepcopy([p.detach().cpu(), None if p.grad is None else p.grad.cpu()]) for p in params]
    cpu = {k: [t.cpu() for t in kwargs[k]] for k in kwargs}
    others = [p for p, _ in clones]
    before = [p.clone() for p in others]
    for p, g in clones:
        p.grad = g
    cpu_m, cpu_v, cpu_steps = [t.cpu() for t in m], [t.cpu() for t in v], steps.cpu()
    norm = AdamWPlan(params, m, v, steps, **kwargs).step(max_grad_norm=0.1, **HYPER)
    want = AdamWPlan(others, cpu_m, cpu_v, cpu_steps, **cpu).step(max_grad_norm=0.1, **HYPER)
    assert torch.equal(norm.cpu(), want) and torch.equal(steps.cpu(), cpu_steps)
    assert all(torch.equal(_bytes(a), _bytes(b)) for a, b in zip((*m, *v), (*cpu_m, *cpu_v)))
    assert all(_same_weight(a, b, c) for a, b, c in zip(params, others, before))


def test_strided_parameters_and_gradients():
    p = torch.randn(6, 10, device="cuda").t().requires_grad_()
    q = p.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
    g = torch.randn(10, 6, device="cuda")
    p.grad, q.grad = g, g.clone()  # the first gradient's order differs from its parameter's
    opts = [AdamW([x], **HYPER) for x in (p, q)]
    for opt in opts:
        opt.step()
    assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_resume(dtype, bits):
    resume("cuda", dtype, bits)


def test_written_bfloat16_parameters_win():
    p = torch.randn(500, device="cuda", dtype=torch.bfloat16).requires_grad_()
    opt = AdamW([p], lr=1e-4, weight_decay=0.0)
    for _ in range(3):
        p.grad = torch.randn_like(p)
        opt.step()
    new = torch.randn(500, device="cuda", dtype=torch.bfloat16) + 3
    with torch.no_grad():
        p.copy_(new)
    p.grad = torch.zeros_like(p)
    opt.step()
    # one step moves by at most lr / (1 - b1), and the kept bits are at most half a bfloat16 step
    assert ((p - new).abs().float() <= new.abs().float() * 2.0 ** -7 + 2e-3).all()


def test_zeros_written_from_outside():
    zeros_written("cuda")


def test_versions_tell_autograd():
    w = torch.randn(8, device="cuda").requires_grad_()
    y = (w * w).sum()
    opt = AdamW([w])
    w.grad = torch.ones_like(w)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_not_finite_gradients():
    for bits in (32, 8):
        p = torch.ones(600, device="cuda").requires_grad_()
        p.grad = torch.ones(600, device="cuda")
        p.grad[3] = float("nan")
        opt = AdamW([p], state_bits=bits)
        opt.step()
        assert p.isnan().sum() == 1 and p[3].isnan()
        values = opt.state[p]["exp_avg"].float()
        if bits == 8:  # the block of the NaN is lost, the others are not
            scale = opt.state[p]["exp_avg_scale"]
            assert scale.isnan().tolist() == [True, False, False]
            values = values * scale.repeat_interleave(256)[:600]
            assert torch.isfinite(values[256:]).all()
        p.grad = torch.ones(600, device="cuda") * float("inf")
        opt2 = AdamW([torch.nn.Parameter(torch.ones(600, device="cuda"))], state_bits=bits, max_grad_norm=1.0)
        opt2.param_groups[0]["params"][0].grad = p.grad
        opt2.step()
        assert opt2.grad_norm.isinf()


def test_zero_gradients_leave_zero_states():
    p = torch.ones(300, device="cuda").requires_grad_()
    p.grad = torch.zeros_like(p)
    opt = AdamW8bit([p], weight_decay=0.0)
    opt.step()
    assert (p == 1).all() and (opt.state[p]["exp_avg"].float() == 0).all()
    assert (opt.state[p]["exp_avg_sq_scale"] == 0).all()


def test_capture_reads_rate_and_steps_from_the_device():
    params = [torch.randn(n, device="cuda") for n in (5, 1000, 70000)]
    grads = [torch.randn_like(p) for p in params]
    results = []
    for captured in (False, True):
        ps = [p.clone().requires_grad_() for p in params]
        for p, g in zip(ps, grads):
            p.grad = g.clone()
        lr = torch.tensor(1e-2, device="cuda")
        opt = AdamW(ps, lr=lr, state_bits=8, max_grad_norm=1.0)
        opt.step()
        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        for k in range(3):
            lr.fill_(1e-2 / (k + 1))
            graph.replay() if captured else opt.step()
        torch.cuda.synchronize()
        results.append([*ps, *(opt.state[p]["exp_avg"] for p in ps), opt.grad_norm, opt.state[ps[0]]["step"]])
    for a, b in zip(*results):
        assert torch.equal(_bytes(a), _bytes(b))
    assert results[0][-1].item() == 4


def test_first_step_is_not_captured():
    p = torch.ones(4, device="cuda").requires_grad_()
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before capturing"):
            opt.step()


def test_refusals():
    refuse_plans("cuda")
    p = torch.ones(4, device="cuda").requires_grad_()
    with pytest.raises(ValueError, match="share a device"):
        q = torch.ones(4).requires_grad_()
        AdamW([p, q]).step()
    plan = AdamWPlan([p], [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")], torch.zeros(1, device="cuda"))
    p.grad = torch.ones_like(p)
    p.data = torch.ones(5, device="cuda")
    with pytest.raises(ValueError):
        plan.step(lr=0.1)
    assert CODES == torch.float8_e4m3fn




def _norm_of(grads, max_norm=1.0):
    """Norm that a clipped step returns, and the step's optimizer."""
    params = [torch.nn.Parameter(torch.zeros_like(g, device="cuda")) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g.cuda()
    opt = AdamW(params, max_grad_norm=max_norm, weight_decay=0.0, betas=(0.5, 0.5))
    opt.step()
    return opt.grad_norm.item(), opt


@pytest.mark.parametrize("dtype,seed", [(torch.float32, 71), (torch.float32, 155), (torch.float32, 198),
                                        (torch.bfloat16, 18), (torch.bfloat16, 224), (torch.bfloat16, 297)])
def test_norm_of_growing_gradients(dtype, seed):
    """Sums whose terms grow: every square is larger than the sum before it. The errors of its sixteen sums (2^-25 each) are
    added up in fp32: 256 times 2^-49, so the sum is right to 2^-41 and the norm is the rounded one (half a step: 2^-24)
    whatever the order. The seeds are some where error terms that assume the larger number first lead to a neighbour."""
    rng = np.random.default_rng(seed)
    chain = (1 + rng.random(16)) * 2.0 ** (np.arange(16) * rng.choice([0.5, 1.0, 2.0, 4.0]))
    # runs of 2,048 elements in which each lane meets the sixteen numbers one after another
    g = torch.tensor(chain, dtype=torch.float32).to(dtype).repeat_interleave(128).repeat(7104)
    want = g.double().norm().item()
    assert abs(_norm_of([g])[0] - want) <= want * (2.0 ** -24 + 2.0 ** -42)
    back = g.flip(0)
    assert abs(_norm_of([back])[0] - want) <= want * (2.0 ** -24 + 2.0 ** -42)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-36, 1e-25, 1e-20, 1e-12, 1e18, 1e20, 1e25, 1e30])
@pytest.mark.parametrize("mixed", [False, True])
def test_norm_beyond_the_range_of_squares(dtype, size, mixed):
    """Gradients whose squares leave fp32's range: the norm is the 64-bit one rounded, and the step clips with it."""
    gen = torch.Generator().manual_seed(3)
    grads = [(torch.randn(n, generator=gen) * size).to(dtype) for n in (5, 3000, 70001, 256)]
    if mixed:
        grads[1][::2] = 1.0
    want = torch.cat(grads).double().norm().item()
    norm, opt = _norm_of(grads)
    assert abs(norm - want) <= want * (2.0 ** -24 + 2.0 ** -42)
    clip = min(1.0, 1.0 / (want + 1e-6))
    for group in opt.param_groups:
        for p, g in zip(group["params"], grads):
            m = opt.state[p]["exp_avg"].double().cpu()
            # clip, its product with g and the product with 0.5: half a step each, and subnormal numbers' spacing
            assert ((m - 0.5 * clip * g.double()).abs() <= m.abs() * 2.0 ** -22 + 2.0 ** -148).all()


def _quotients(m, v, eps):
    """``-m' / (2 sqrt(v') + eps)`` as the step forms it, with m' = m / 2 and v' = 0.75 v, and as fp32 operations of
    NumPy, each rounded correctly."""
    p = torch.nn.Parameter(torch.zeros(len(m), device="cuda"))
    p.grad = torch.zeros(len(m), device="cuda")
    plan = AdamWPlan([p], [m.cuda()], [v.cuda()], torch.zeros(1, device="cuda"))
    plan.step(lr=0.5, betas=(0.5, 0.75), eps=eps, weight_decay=0.0)  # lr / (1 - b1) = 1, 1 / sqrt(1 - b2) = 2
    one = np.float32
    with np.errstate(over="ignore"):
        root = np.sqrt(v.numpy() * one(0.75))
        return p.detach().cpu().numpy(), -(m.numpy() * one(0.5) / (root * one(2.0) + one(eps)))


@pytest.mark.parametrize("eps", [1e-8, 1e-20])
def test_roots_and_quotients_are_rounded(eps):
    """After the last Newton step the quotient is rounded from a value within 2^-21 of a step of the true one, the root
    likewise: each is the rounded one but where the true one lies that close to the middle of two numbers (a chance of
    about 2^-20 a number), and then it is the neighbour. A root that is off by a step moves the quotient by two at most."""
    gen = torch.Generator().manual_seed(4)
    n = 1 << 22
    v = torch.exp((torch.rand(n, generator=gen) * 60 - 40) * 0.6931)  # 2^-40 to 2^20
    m = torch.exp((torch.rand(n, generator=gen) * 60 - 30) * 0.6931) * (1 - 2 * (torch.rand(n, generator=gen) < 0.5).float())
    got, want = _quotients(m, v, eps)
    off = np.abs(got.view(np.int32).astype(np.int64) - want.view(np.int32).astype(np.int64))
    assert off.max() <= 3 and (off > 0).mean() <= 1e-4


def test_quotients_beyond_the_range_are_infinite():
    m = torch.tensor([1e29, -1e29, 1e29, 1e25, 3e17, 0.0])
    v = torch.tensor([1e-30, 1e-30, 1e20, 1e-38, 1e-38, 0.0])
    got, want = _quotients(m, v, 1e-20)
    assert not np.isnan(want).any() and np.isinf(want[:2]).all()
    assert ((got == want) | (np.abs(got - want) <= np.abs(want) * 3 * 2.0 ** -23)).all()


def test_spikes():
    spikes("cuda")
