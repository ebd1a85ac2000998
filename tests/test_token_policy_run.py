"""The token-policy operators as they are used together: score, loss with gradient, optimizer step; and the optimizers
by their configuration names."""

import pytest
import torch

import token_oracle as oracle
from helpers import ppo_cfg, small_env
from tt_rsl_rl_b200.ops.adamw import AdamW
from tt_rsl_rl_b200.ops.token_loss import preference_loss, token_logprobs, token_policy_loss, token_policy_loss_grad
from tt_rsl_rl_b200.runners import OnPolicyRunner


class TinyPolicy(torch.nn.Module):
    """Logits of the next token from the current one."""

    def __init__(self, vocab, width):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, width)
        self.head = torch.nn.Linear(width, vocab)

    def forward(self, tokens):
        return self.head(torch.tanh(self.embed(tokens)))


def train(device, dtype, bits, steps=3):
    """Policy-loss steps on padded responses: each parameter's gradient is the chain rule's on the 64-bit gradient of the
    logits, in both forms of the loss; every step moves the weights and leaves them finite."""
    torch.manual_seed(0)
    vocab, batch, length = 53, 4, 9
    model = TinyPolicy(vocab, 16).to(device, dtype)
    reference = TinyPolicy(vocab, 16).to(device, dtype)
    tokens = torch.randint(vocab, (batch, length), device=device)
    mask = torch.arange(1, length, device=device)[None] >= torch.tensor([[1], [3], [5], [8]], device=device)
    optimizer = AdamW(model.parameters(), lr=1e-3, state_bits=bits, max_grad_norm=1.0)
    with torch.no_grad():
        old, entropy = token_logprobs(model(tokens)[:, :-1], tokens[:, 1:], mask=mask)
        ref, _ = token_logprobs(reference(tokens)[:, :-1], tokens[:, 1:], mask=mask)
    assert (old[~mask] == 0).all() and (entropy[mask] > 0).all()
    adv = torch.randn(batch, length - 1, device=device)
    kwargs = dict(ref_logp=ref, mask=mask, kl_coef=0.05, entropy_coef=0.01)
    for step in range(steps):
        logits = model(tokens)[:, :-1]
        out, grad = token_policy_loss_grad(logits, tokens[:, 1:], old, adv, **kwargs)
        optimizer.zero_grad()
        logits.backward(grad)
        by_hand = [p.grad.clone() for p in model.parameters()]
        cpu = [t.detach().cpu() for t in (logits, tokens[:, 1:], old, adv, ref, mask)]
        _, _, _, da, db = oracle.policy(*cpu, lo=0.8, hi=1.2, kl_coef=0.05, kind="k3", entropy_coef=0.01,
                                        temperature=1.0)
        want, _ = oracle.logits_grad(cpu[0], cpu[1], cpu[5], 1.0, da, db)
        # 36 rows of products: each gradient of the logits is off by half a step of its type and 1e-4 (the coefficients of
        # fp32 log-probabilities, on the first step exp(0) - 1 among them), the sums of the chain rule by a step of it more
        eps = torch.finfo(dtype).eps
        assert ((grad.cpu().double() - want).abs() <= want.abs() * (eps / 2 + 1e-4) + 1e-6).all()
        full = torch.zeros(batch, length, vocab, dtype=torch.float64)
        full[:, :-1] = want
        bias = full.sum((0, 1))
        assert ((model.head.bias.grad.cpu().double() - bias).abs() <= full.abs().sum((0, 1)) * (4 * eps + 1e-4) + 1e-5).all()
        optimizer.zero_grad()
        loss = token_policy_loss(model(tokens)[:, :-1], tokens[:, 1:], old, adv, **kwargs).loss
        loss.backward()
        for p, g in zip(model.parameters(), by_hand):
            scale = g.abs().max() + 1e-6
            assert ((p.grad - g).abs() <= scale * (4 * eps + 1e-4)).all()  # the same values by other kernels
        before = [p.detach().clone() for p in model.parameters()]
        optimizer.step()
        assert torch.isfinite(optimizer.grad_norm) and all(torch.isfinite(p).all() for p in model.parameters())
        assert any(not torch.equal(p, q) for p, q in zip(model.parameters(), before))
        assert out.clip_fraction >= 0 and torch.isfinite(out.loss)
    # a preference step on the same model
    optimizer.zero_grad()
    pref = preference_loss(model(tokens)[:, :-1], tokens[:, 1:], old.sum(1), mask=mask)
    pref.loss.backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    assert pref.chosen_rewards.shape == (2,)
    optimizer.step()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(dtype, bits):
    train("cpu", dtype, bits)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps_gpu(dtype, bits):
    train("cuda", dtype, bits)


@pytest.mark.gpu
def test_captured_training_step():
    """Loss, gradient and optimizer step as one graph, replayed, equal the eager steps."""
    torch.manual_seed(0)
    vocab, rows = 3001, 40
    tokens = torch.randint(vocab, (rows,), device="cuda")
    adv = torch.randn(rows, device="cuda")
    start = torch.randn(rows, vocab, device="cuda", dtype=torch.bfloat16)
    old, _ = token_logprobs(start, tokens)
    results = []
    for captured in (False, True):
        logits = start.clone().requires_grad_()
        opt = AdamW([logits], lr=1e-2, state_bits=8, max_grad_norm=1.0)

        def step():
            _, logits.grad = token_policy_loss_grad(logits, tokens, old, adv, entropy_coef=0.01)
            opt.step()

        step()
        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        for _ in range(3):
            graph.replay() if captured else step()
        torch.cuda.synchronize()
        results.append((logits.detach().clone(), opt.state[logits]["low_bits"].clone()))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def ppo_iterations(device, name):
    torch.manual_seed(0)
    cfg = ppo_cfg(optimizer=name)
    runner = OnPolicyRunner(small_env(device=device), cfg, log_dir=None, device=device)
    before = [p.detach().clone() for p in runner.alg.actor.parameters()]
    runner.learn(2)
    assert runner.alg.engine is None  # the fused engines step Adam
    assert all(torch.isfinite(p).all() for p in runner.alg.actor.parameters())
    assert any(not torch.equal(p, q) for p, q in zip(runner.alg.actor.parameters(), before))
    saved = runner.alg.save()
    other = OnPolicyRunner(small_env(device=device), ppo_cfg(optimizer=name), log_dir=None, device=device)
    other.alg.load(saved, None, True)
    other.learn(1)
    return runner


@pytest.mark.parametrize("name", ["adamw_fused", "adamw_8bit"])
def test_ppo_with_the_optimizer(name):
    ppo_iterations("cpu", name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["adamw_fused", "adamw_8bit"])
def test_ppo_with_the_optimizer_gpu(name):
    ppo_iterations("cuda:0", name)
