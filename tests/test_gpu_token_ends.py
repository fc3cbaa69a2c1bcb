"""The operators at the token ends together, as a rollout and a training step use them: tokens drawn from the logits of a
tied model, embedded again, and the training step on them with its gradients joined in one fp32 buffer."""

import pytest
import torch

from areal_amd.functional import (
    embed_tokens,
    fused_lm_head_logprobs_entropy,
    gather_kept_logprobs_entropy,
    ppo_actor_loss_fn,
    sample_tokens,
)
from oracle import token_ends as O

pytestmark = pytest.mark.gpu


def test_rollout_then_training_step(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    V, H, B, steps, tau, scale = 2048, 128, 6, 5, 0.8, 2.0
    master = (torch.randn(V, H, generator=g, device=dev) * 0.3).requires_grad_(True)
    mix = torch.randn(H, H, generator=g, device=dev) * H**-0.5

    def model(ids):  # tied: the same weight at both ends
        return torch.tanh(embed_tokens(ids, master, scale, out_dtype=torch.bfloat16).float() @ mix)

    ids, tokens, old, kepts = torch.randint(0, V, (B,), generator=g, device=dev), [], [], []
    inputs = []
    with torch.no_grad():
        for _ in range(steps):
            logits = model(ids) @ master.t()
            u = torch.rand(B, generator=g, device=dev)
            got = sample_tokens(logits, u, temperature=tau, top_p=0.9, top_k=100, return_kept=True)
            want, lp, _, kept = O.sample(logits.cpu(), u.cpu(), tau, 100, 0.9)
            assert torch.equal(got.tokens.cpu(), want) and torch.equal(got.kept.cpu(), O.pack_bits(kept))
            inputs.append(ids)
            tokens.append(got.tokens)
            old.append(got.logprobs)
            kepts.append(got.kept)
            ids = got.tokens
    inputs, labels, old, kept = torch.cat(inputs), torch.cat(tokens), torch.cat(old), torch.cat(kepts)

    # the trainer's log-probabilities under the kept sets: those of the rollout, so that every ratio is 1
    logits = model(inputs) @ master.t()
    lp, ent = gather_kept_logprobs_entropy(logits, labels, kept, tau)
    # exponents up to ~10 / 0.8 in base 2, off by a few 2^-24 of that each
    torch.testing.assert_close(lp.detach(), old, rtol=1e-6, atol=1e-5)
    n = B * steps
    adv = torch.randn(n, generator=g, device=dev)
    loss, stat = ppo_actor_loss_fn(lp, old, old, adv, 0.2, torch.ones(n, dtype=torch.bool, device=dev))
    assert (stat["importance_weight"] - 1).abs().max() < 1e-4
    (dlogits,) = torch.autograd.grad(loss, logits, retain_graph=True)
    mask = torch.zeros(n, V, dtype=torch.bool)
    for j in range(32):
        mask[:, j::32] = (kept.cpu() >> j & 1).bool()
    want = O.kept_backward(logits.detach().cpu(), labels.cpu(), mask, -adv.cpu() / n, torch.zeros(n), tau)
    torch.testing.assert_close(dlogits.cpu().double(), want, rtol=1e-3, atol=1e-6)  # (ratios of 1 to 1e-5 in the weights)
    loss.backward()
    assert torch.isfinite(master.grad).all()


def test_tied_gradients_in_one_buffer(dev):
    """The lm_head's dWeight and the embedding's gradient, both added to the master's fp32 .grad."""
    g = torch.Generator(device=dev).manual_seed(1)
    V, H, T = 1536, 128, 200
    master = (torch.randn(V, H, generator=g, device=dev) * 0.2).bfloat16().float().requires_grad_(True)
    ids = torch.randint(0, V, (T,), generator=g, device=dev)
    labels = torch.randint(0, V, (T,), generator=g, device=dev)
    up = torch.randn(T, generator=g, device=dev)
    accum = torch.zeros(V, H, device=dev)
    compute = master.detach().bfloat16()
    hidden = embed_tokens(ids, master, out_dtype=torch.bfloat16, weight_grad_accum=accum)
    out = fused_lm_head_logprobs_entropy(hidden, compute, labels, weight_grad_accum=accum)
    (out.logprobs * up).sum().backward()
    assert master.grad is None
    # plain form in fp32
    w = master.detach().cpu().requires_grad_(True)
    lp = torch.log_softmax(w[ids.cpu()] @ w.t(), -1)[torch.arange(T), labels.cpu()]
    (lp * up.cpu()).sum().backward()
    # dlogits, hidden states and dHidden are bf16 on the way: 2^-8 of their size each
    assert (accum.cpu() - w.grad).norm() / w.grad.norm() < 3 * 2.0**-8
