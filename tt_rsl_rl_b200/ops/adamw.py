"""AdamW over many tensors at once (``csrc/adamw_kernels.cu``), with 32-bit or 8-bit states.

The update is ``torch.optim.AdamW``'s (decoupled weight decay); the states of ``state_bits=32`` have its names and
values. bfloat16 parameters are the upper half of a float32 weight whose lower 16 bits the optimizer keeps
(``low_bits``), so a step is never lost to rounding: the pair is 4 bytes, the parameter alone is what the model reads.
A finite parameter written from outside (a loaded checkpoint) is taken over by the next step, to within half of a
bfloat16 step.

8-bit states hold, for each 256 consecutive elements of a tensor, a float32 scale and e4m3 codes: of the first moment
and of the *root* of the second, whose range a code covers better. One step moves a moving average by far less than the
distance between two codes, so a code is rounded up or down at random with the probabilities that make the stored first
and second moments right on average (Philox4x32-10, keyed by ``seed``; counted by element, tensor and step, so equal
seeds give equal steps on every rank). A root never rounds down to zero, which would leave ``m / eps`` as a step. Blocks
whose largest moment is below 1e-30 are stored as zero; a NaN or infinity makes its block's scale NaN or infinite. A finite
gradient whose square is beyond float32 (1.8e19 and more, unless it is clipped) makes its block's second moment infinite, so
the block's weights stay where they are.

The gradients' norm is right to float32's rounding over their whole range, whatever the order and split of the tensors. The
learning rate may be a tensor on the device; a captured step (after one eager one) reads it at every replay, and
advances the step counts, which are on the device too. On CPU tensors the same arithmetic runs as PyTorch operations.
"""

from __future__ import annotations

import math

import torch

from . import ext

BLOCK = 256  # consecutive elements that share a scale
CODES = torch.float8_e4m3fn
TINY = 1e-30


def _check_hyper(lr, betas, eps, weight_decay, max_grad_norm, seed) -> None:
    if not isinstance(lr, torch.Tensor) and not (lr >= 0.0 and math.isfinite(lr)):
        raise ValueError(f"lr must be finite and not negative, got {lr}")
    if not all(0.0 <= b < 1.0 for b in betas):
        raise ValueError(f"betas must lie in [0, 1), got {tuple(betas)}")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    if not (weight_decay >= 0.0 and math.isfinite(weight_decay)):
        raise ValueError(f"weight_decay must be finite and not negative, got {weight_decay}")
    if max_grad_norm is not None and not max_grad_norm > 0.0:
        raise ValueError(f"max_grad_norm must be positive, got {max_grad_norm}")
    if not 0 <= seed < 2 ** 63:
        raise ValueError(f"seed must lie in [0, 2^63), got {seed}")


class AdamWPlan:
    """The tensors of a step: parameters of one type (float32 or bfloat16) on one device with their states.

    ``exp_avgs`` and ``exp_avg_sqs`` have the parameters' shapes and strides, in float32, or in float8_e4m3fn (codes of
    the first moment and of the root of the second) with ``exp_avg_scales`` / ``exp_avg_sq_scales`` of one float32 per
    256 elements in memory order. ``steps``: float32 ``[parameters]``. ``low_bits`` (int16, bfloat16 parameters only):
    the float32 weight's bits minus its bfloat16 rounding's. ``first_stream`` numbers the parameters' random streams.
    :meth:`step` updates all of them in place, whatever their number, in two launches per 400 tensors."""

    def __init__(self, params, exp_avgs, exp_avg_sqs, steps: torch.Tensor, *, exp_avg_scales=None,
                 exp_avg_sq_scales=None, low_bits=None, first_stream: int = 0) -> None:
        self.params = list(params)
        tensors = (self.params, list(exp_avgs), list(exp_avg_sqs), steps, list(exp_avg_scales or ()),
                   list(exp_avg_sq_scales or ()), list(low_bits or ()))
        if not self.params:
            raise ValueError("AdamWPlan: no parameters")
        self.device = self.params[0].device
        if self.device.type == "cuda":
            self._native = ext().AdamWPlan(*tensors, first_stream)
        else:
            self._native = None
            _check_plan_cpu(*tensors)
            self._tensors, self._first_stream = tensors, first_stream

    def step(self, *, lr, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
             max_grad_norm: float | None = None, maximize: bool = False, seed: int = 0) -> torch.Tensor | None:
        """One step of every parameter whose ``.grad`` is set. With ``max_grad_norm`` the gradients count as scaled by
        ``min(1, max_grad_norm / (norm + 1e-6))`` (``.grad`` keeps its values) and their norm is returned."""
        _check_hyper(lr, betas, eps, weight_decay, max_grad_norm, seed)
        return _step([self], [(lr, *betas, eps, weight_decay, maximize, seed)], max_grad_norm)


def _step(plans: list[AdamWPlan], settings: list[tuple], max_grad_norm: float | None) -> torch.Tensor | None:
    if plans[0]._native is None:
        return _step_torch(plans, settings, max_grad_norm)
    rows = []
    for lr, *rest in settings:
        tensor = isinstance(lr, torch.Tensor)
        on_device = tensor and lr.is_cuda
        rows.append((0.0 if on_device else float(lr), lr if on_device else None, *rest))
    return ext().adamw_step([p._native for p in plans], rows, max_grad_norm or 0.0)


# ---- the same step as PyTorch operations (CPU tensors) --------------------------------------------------------------------
def _check_plan_cpu(params, m, v, steps, m_scales, v_scales, low) -> None:
    n, dtype, state = len(params), params[0].dtype, m[0].dtype if m else None
    if len(m) != n or len(v) != n:
        raise ValueError("AdamWPlan: one exp_avg and one exp_avg_sq per parameter")
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"AdamWPlan: parameters must be float32 or bfloat16, got {dtype}")
    if state not in (torch.float32, CODES):
        raise TypeError(f"AdamWPlan: states must be float32 or float8_e4m3fn, got {state}")
    if state == CODES and not (len(m_scales) == len(v_scales) == n):
        raise ValueError("AdamWPlan: 8-bit states need their scales (exp_avg_scales, exp_avg_sq_scales)")
    if state != CODES and (m_scales or v_scales):
        raise ValueError("AdamWPlan: float32 states have no scales")
    if len(low) != (n if dtype == torch.bfloat16 else 0):
        raise ValueError("AdamWPlan: low_bits belong to bfloat16 parameters, one each")
    if steps.dtype != torch.float32 or steps.numel() != n or not steps.is_contiguous():
        raise ValueError("AdamWPlan: steps must be a contiguous float32 tensor, one element per parameter")
    for i, p in enumerate(params):
        if p.dtype != dtype or p.device != params[0].device:
            raise TypeError("AdamWPlan: parameters of one plan share a type and a device")
        if not _dense(p):
            raise ValueError(f"AdamWPlan: parameter {i} has gaps or overlaps in memory (strides {p.stride()})")
        for name, s, want in (("exp_avg", m[i], state), ("exp_avg_sq", v[i], state),
                              *((("low_bits", low[i], torch.int16),) if low else ())):
            if s.dtype != want:
                raise TypeError(f"AdamWPlan: {name} {i} must be {want}, got {s.dtype}")
            if s.shape != p.shape or s.stride() != p.stride():
                raise ValueError(f"AdamWPlan: {name} {i} must have the parameter's device, shape and strides")
    apart = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                   for t in (*params, *m, *v, *m_scales, *v_scales, *low) if t.numel())
    if any(b[0] < a[1] for a, b in zip(apart, apart[1:])):
        raise ValueError("AdamWPlan: two tensors share memory")
    for i, p in enumerate(params):
        for s in (m_scales[i], v_scales[i]) if m_scales else ():
            if s.dtype != torch.float32 or s.numel() != -(-p.numel() // BLOCK) or not s.is_contiguous():
                raise ValueError(f"AdamWPlan: scales {i} must hold one float32 per {BLOCK} elements of the parameter")


def _dense(p: torch.Tensor) -> bool:
    span = 1
    for size, stride in sorted(((n, s) for n, s in zip(p.shape, p.stride()) if n != 1), key=lambda x: x[1]):
        if stride != span:
            return p.numel() == 0
        span *= size
    return True


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether tensors of one shape walk memory in the same order (strides of single elements do not matter)."""
    return all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _flat(x: torch.Tensor) -> torch.Tensor:
    """A dense tensor's elements in memory order (a view)."""
    return x.as_strided((x.numel(),), (1,))


def _philox(index4: torch.Tensor, stream: int, step: int, seed: int) -> torch.Tensor:
    """Philox4x32-10 (Salmon et al., SC 2011): four 32-bit words per counter (index low, index high, stream, step)."""
    low = 0xFFFFFFFF
    c = [index4 & low, index4 >> 32, torch.full_like(index4, stream & low), torch.full_like(index4, step & low)]
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32 & low) ^ c[1] ^ k0, b & low, (a >> 32 & low) ^ c[3] ^ k1, a & low]
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return torch.stack(c, 1).flatten()


def _e4m3_below(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The largest e4m3 value at most ``y`` (in [0, 448]) and its successor."""
    exponent = y.clamp(min=2.0 ** -6).view(torch.int32) >> 23
    spacing = (exponent - 3 << 23).view(torch.float32)
    below = torch.floor(y / spacing) * spacing
    return below, below + spacing


def _store_codes(x: torch.Tensor, rnd: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, squared: bool) -> None:
    blocks = len(scales)
    padded = torch.zeros(blocks * BLOCK)
    padded[:len(x)] = x
    top = padded.abs().view(blocks, BLOCK).amax(1)
    on = ~(top < TINY)
    inverse = torch.where(on, 448.0 / top, 0.0).repeat_interleave(BLOCK)[:len(x)]
    y = (x.abs() * inverse).nan_to_num(nan=448.0).clamp(max=448.0)
    below, above = _e4m3_below(y)
    u = (rnd.float() + 0.5) / 65536.0
    if squared:
        up = (above - below) * (above + below) * u < (y - below) * (y + below)
    else:
        up = (above - below) * u < y - below
    value = torch.where(up, above, below)
    if squared:
        value = torch.where((x > 0) & on.repeat_interleave(BLOCK)[:len(x)], value.clamp(min=2.0 ** -9), value)
    codes.copy_(torch.copysign(value, x) if not squared else value)
    scales.copy_(torch.where(on, top * (1.0 / 448.0), 0.0))


def _join(p: torch.Tensor, low: torch.Tensor) -> torch.Tensor:
    """The float32 weight of a bfloat16 one and its lower bits, unless those (of another weight) would carry it across
    zero."""
    b = p.view(torch.int16).int() << 16
    w = b + low.int()
    return torch.where((w ^ b) < 0, b, w).view(torch.float32)


def _step_torch(plans, settings, max_grad_norm):
    norm, clip = None, torch.ones(())
    with torch.no_grad():
        if max_grad_norm is not None:
            squares = [p.grad.double().square().sum() for plan in plans for p in plan.params if p.grad is not None]
            root = torch.stack(squares).sum().sqrt() if squares else torch.zeros((), dtype=torch.float64)
            norm, clip = root.float(), (max_grad_norm / (root + 1e-6)).clamp(max=1.0).float()
        for plan, (lr, b1, b2, eps, decay, maximize, seed) in zip(plans, settings):
            params, m, v, steps, m_scales, v_scales, low = plan._tensors
            lr = float(lr)
            for i, p in enumerate(params):
                if p.grad is None:
                    continue
                if p.grad.dtype != p.dtype or p.grad.layout != torch.strided:
                    raise TypeError(f"AdamW: the gradient of parameter {i} must be a strided {p.dtype} tensor")
                steps[i] += 1.0
                grad = torch.empty_like(p, memory_format=torch.preserve_format).copy_(p.grad)
                g = _flat(grad).float() * (-clip if maximize else clip)
                w, mi, vi = _flat(p), _flat(m[i]), _flat(v[i])
                x = w if w.dtype == torch.float32 else _join(w, _flat(low[i]))
                m0, v0 = mi.float(), vi.float()
                if m_scales:
                    m0 = m0 * m_scales[i].repeat_interleave(BLOCK)[:len(x)]
                    v0 = (v0 * v_scales[i].repeat_interleave(BLOCK)[:len(x)]).square()
                m1 = m0 * b1 + g * (1 - b1)
                v1 = v0 * b2 + g * g * (1 - b2)
                t = float(steps[i])
                step_size, unbias, keep = torch.tensor([lr / (1 - b1 ** t), (1 - b2 ** t) ** -0.5, 1 - lr * decay])
                root = v1.double().sqrt().float()  # rounded correctly, which an fp32 root here may not be
                x = x * keep - step_size * (m1 / (root * unbias + eps))
                if low:
                    bits = x.view(torch.int32)
                    high = torch.where(x.isnan(), 0x7fc0, bits + 0x8000 >> 16)
                    _flat(low[i]).copy_(torch.where(x.isnan(), 0, bits - (high << 16)))
                    w.copy_(high.to(torch.int16).view(torch.bfloat16))
                else:
                    w.copy_(x)
                if m_scales:
                    groups = torch.arange(-(-len(x) // 4))
                    words = _philox(groups, plan._first_stream + i, int(t), seed)[:len(x)]
                    _store_codes(m1, words & 0xFFFF, mi, m_scales[i], False)
                    _store_codes(root, words >> 16, vi, v_scales[i], True)
                else:
                    mi.copy_(m1)
                    vi.copy_(v1)
    return norm


# ---- torch.optim form ---------------------------------------------------------------------------------------------------
class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW``'s update as a :class:`AdamWPlan` step over all parameters.

    ``state_bits``: 32 or 8. ``max_grad_norm``: clip the global gradient norm inside the step (``grad_norm`` holds the
    norm afterwards). Parameters are float32 or bfloat16, all on one device. In a 32-bit optimizer, state dictionaries
    of ``torch.optim.AdamW`` load. The tensors of ``state`` and the lists of parameters are bound at the first step:
    write states in place or load a state dictionary, add parameters with ``add_param_group``."""

    def __init__(self, params, lr: float | torch.Tensor = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, max_grad_norm: float | None = None,
                 maximize: bool = False, seed: int = 0) -> None:
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        _check_hyper(lr, betas, eps, weight_decay, max_grad_norm, seed)
        self.state_bits, self.max_grad_norm, self.seed = state_bits, max_grad_norm, seed
        self.grad_norm: torch.Tensor | None = None
        self._plans: list[tuple[dict, AdamWPlan]] | None = None
        super().__init__(params, {"lr": lr, "betas": tuple(betas), "eps": eps, "weight_decay": weight_decay,
                                  "maximize": maximize})

    def __getstate__(self):
        return super().__getstate__() | {"state_bits": self.state_bits, "max_grad_norm": self.max_grad_norm,
                                         "seed": self.seed}

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("maximize", False)
        self._plans, self.grad_norm = None, None

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        self._plans = None

    def load_state_dict(self, state_dict) -> None:
        """The base class casts states to the parameter's type; codes, scales and float32 moments keep theirs here: as the
        last hook before loading leaves them, and before the first one behind it."""
        loaded = {}

        def check(_, state):
            for group in state["param_groups"]:
                if group.get("amsgrad"):
                    raise ValueError("AdamW: the loaded state is of an update with amsgrad, which this one has not")
                if not group.get("decoupled_weight_decay", True) and group.get("weight_decay", 0.0) != 0.0:
                    raise ValueError("AdamW: the loaded state is of an update whose weight decay is not decoupled")
            loaded.update(state)

        def keep_types(_):
            saved = [i for group in loaded["param_groups"] for i in group["params"]]
            own = [p for group in self.param_groups for p in group["params"]]
            for index, p in zip(saved, own):
                for key, value in loaded["state"].get(index, {}).items():
                    if isinstance(value, torch.Tensor):
                        self.state[p][key] = value.detach().to(device=p.device, copy=True)

        hooks = (self.register_load_state_dict_pre_hook(check),
                 self.register_load_state_dict_post_hook(keep_types, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
        self._plans = None

    def _state_of(self, p: torch.Tensor) -> dict:
        """The parameter's state, made or completed."""
        state = self.state[p]
        dtype = torch.float32 if self.state_bits == 32 else CODES
        for key in ("exp_avg", "exp_avg_sq"):
            x = state.get(key)
            if x is None:
                state[key] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format).to(dtype)
                continue
            if (x.dtype == CODES) != (self.state_bits == 8) or not x.is_floating_point():
                raise ValueError(f"the loaded {key} is {x.dtype}: it does not belong to {self.state_bits}-bit states")
            if x.shape != p.shape:
                raise ValueError(f"the loaded {key} has the shape {tuple(x.shape)}, its parameter {tuple(p.shape)}")
            if self.state_bits == 8 and state.get(f"{key}_scale") is None:
                raise ValueError(f"the loaded {key} has no {key}_scale: 8-bit codes mean nothing without their scales")
            if self.state_bits == 8 and not _same_order(x, p):
                raise ValueError(f"the loaded {key} has strides {x.stride()}, its parameter {p.stride()}: the scales of "
                                 "8-bit states follow the order in memory")
            if x.dtype != dtype or x.stride() != p.stride():
                like = torch.empty_like(p, dtype=dtype, memory_format=torch.preserve_format)
                state[key] = like.copy_(x)
        if self.state_bits == 8:
            for key in ("exp_avg_scale", "exp_avg_sq_scale"):
                if state.get(key) is None:
                    state[key] = torch.zeros(-(-p.numel() // BLOCK), device=p.device)
        if p.dtype == torch.bfloat16:
            low = state.get("low_bits")
            if low is None or (low.dtype == torch.int16 and low.shape == p.shape and low.stride() != p.stride()):
                like = torch.zeros_like(p, dtype=torch.int16, memory_format=torch.preserve_format)
                state["low_bits"] = like if low is None else like.copy_(low)
        return state

    def _build(self) -> list[tuple[dict, AdamWPlan]]:
        plans, stream, devices = [], 0, set()
        for group in self.param_groups:
            for dtype in (torch.float32, torch.bfloat16):
                params = [p for p in group["params"] if p.dtype == dtype]
                if not params:
                    continue
                devices.update(p.device for p in params)
                states = [self._state_of(p) for p in params]
                steps = torch.tensor([float(s.get("step", 0.0)) for s in states], device=params[0].device)
                for s, step in zip(states, steps):
                    s["step"] = step
                many = {k: [s[k] for s in states] if k in states[0] else None
                        for k in ("exp_avg_scale", "exp_avg_sq_scale", "low_bits")}
                plans.append((group, AdamWPlan(params, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                                               steps, exp_avg_scales=many["exp_avg_scale"],
                                               exp_avg_sq_scales=many["exp_avg_sq_scale"], low_bits=many["low_bits"],
                                               first_stream=stream)))
                stream += len(params)
            odd = [p.dtype for p in group["params"] if p.dtype not in (torch.float32, torch.bfloat16)]
            if odd:
                raise TypeError(f"AdamW parameters must be float32 or bfloat16, got {odd[0]}")
        if len(devices) > 1:
            raise ValueError(f"AdamW parameters must share a device, got {sorted(map(str, devices))}")
        return plans

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._plans is None:
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: run one step before capturing one (it creates the states)")
            self._plans = self._build()
        settings = []
        for group, _ in self._plans:
            _check_hyper(group["lr"], group["betas"], group["eps"], group["weight_decay"], self.max_grad_norm, self.seed)
            settings.append((group["lr"], *group["betas"], group["eps"], group["weight_decay"], group["maximize"],
                             self.seed))
        self.grad_norm = _step([plan for _, plan in self._plans], settings, self.max_grad_norm)
        return loss


class AdamW8bit(AdamW):
    """:class:`AdamW` with 8-bit states."""

    def __init__(self, params, lr: float | torch.Tensor = 1e-3, **kwargs) -> None:
        super().__init__(params, lr, state_bits=8, **kwargs)
