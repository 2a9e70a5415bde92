"""Decoder.score and Decoder.divergence: given transcripts judged by the decode plan itself,
and the decoder's tail tuned against them (final norm and token table)."""

from __future__ import annotations

import importlib

import pytest
import torch

import training_reference as ref
from conftest import PACKAGE

pytestmark = pytest.mark.gpu

STREAMS, STEPS = 3, 6


@pytest.fixture(scope="module")
def dec(lffw):
    return importlib.import_module(PACKAGE + ".decoder")


@pytest.fixture(scope="module")
def training(cuda):
    return importlib.import_module(PACKAGE + ".training")


@pytest.fixture(scope="module")
def plan(cuda, dec):
    config = dec.DecoderConfig(layers=2)
    g = torch.Generator(device=cuda).manual_seed(4)
    ck = dec.add_synthetic_decoder({}, config, seed=31, device=cuda)
    weights = dec.DecoderWeights.from_checkpoint(ck, config)
    cross_kv = torch.randn((4, STREAMS, config.heads, config.audio_positions, 64), generator=g, device=cuda).half()
    scales = dec.calibrate(weights, cross_kv, STREAMS, steps=3)
    return dec.Decoder(weights, scales, cross_kv, STREAMS)


@pytest.fixture(scope="module")
def greedy(plan):
    """(tokens [streams, steps], states [steps, streams, d]) of a greedy decode."""
    plan.reset()
    tokens, states = [], []
    for _ in range(STEPS):
        plan.step()
        tokens.append(plan.tokens.clone())
        states.append(plan.states.clone())
    return torch.stack(tokens, 1), torch.stack(states)


def test_states_are_the_decode_s(plan, greedy, native):
    tokens, states = greedy
    assert torch.equal(plan.final_states(tokens), states)
    assert torch.equal(plan.lengths, torch.full_like(plan.lengths, STEPS))
    assert native.device_error() == 0


def test_score(plan, greedy, training, fp8):
    tokens, states = greedy
    table = plan.weights.token_table
    x = states.view(-1, states.shape[2])
    labels = tokens.t().reshape(-1)
    targets = ref.label_targets(labels, table.shape[0], -100)
    e_loss, e_lse, _ = ref.vocab_loss(x, table, targets)
    bound, _ = ref.loss_bounds(x, table, targets, e_loss, e_lse)
    losses = plan.score(tokens)
    assert losses.shape == tokens.shape
    assert ref.worst(losses.t().reshape(-1), e_loss, bound) <= 1
    # The greedy choice has the largest probability of its position: no other token costs less.
    other = plan.score(torch.where(tokens == 5, 6, 5).to(torch.int32))
    assert (losses[:, 0] <= other[:, 0]).all()
    # Padding costs nothing, and does not change what comes before it.
    padded = tokens.clone()
    padded[1, 3:] = -100
    again = plan.score(padded)
    assert not again[1, 3:].any() and torch.equal(again[1, :3], losses[1, :3])
    assert torch.equal(again[[0, 2]], losses[[0, 2]])
    assert training.token_error() == 0 and fp8.decoder_error() == 0


def test_divergence(plan, greedy, training):
    tokens, states = greedy
    table = plan.weights.token_table
    x = states.view(-1, states.shape[2])
    z = x.double() @ table.double().t()
    # Against its own best logits: what the left-out tail of the distribution weighs.
    best = z.topk(100, dim=1)
    shape = (STEPS, STREAMS, 100)
    t_tokens = best.indices.to(torch.int32).view(shape).transpose(0, 1).contiguous()
    t_logits = best.values.float().view(shape).transpose(0, 1).contiguous()
    got = plan.divergence(tokens, t_tokens, t_logits, temperature=1.0)
    tail = torch.logsumexp(z, 1) - torch.logsumexp(best.values, 1)
    targets = ref.teacher_targets(best.indices, best.values.float(), table.shape[0], 1.0)
    e_loss, e_lse, _ = ref.vocab_loss(x, table, targets)
    bound, _ = ref.loss_bounds(x, table, targets, e_loss, e_lse, 1.0, 100)
    assert ref.worst(got.t().reshape(-1), e_loss, bound) <= 1
    assert ((got.t().reshape(-1).double() - tail).abs() <= bound + 2.0 ** -18).all()
    padded = tokens.clone()
    padded[2] = -100
    assert not plan.divergence(padded, t_tokens, t_logits)[2].any()


def test_refusals(plan, greedy):
    tokens, _ = greedy
    for bad in (tokens.long(), tokens[:2], tokens.cpu(), tokens[:, :0], tokens.repeat(1, 100)):
        with pytest.raises(ValueError):
            plan.score(bad)
    with pytest.raises(ValueError):
        plan.divergence(tokens, torch.zeros((STREAMS, STEPS + 1, 2), dtype=torch.int32, device="cuda"),
                        torch.zeros((STREAMS, STEPS + 1, 2), device="cuda"))


def test_refuses_teachers_of_other_ranks(plan, greedy):
    tokens, _ = greedy
    with pytest.raises(ValueError):
        plan.divergence(tokens, tokens, torch.zeros_like(tokens, dtype=torch.float32))
    with pytest.raises(ValueError):
        plan.divergence(tokens, tokens.unsqueeze(2), torch.zeros((STREAMS, STEPS, 2), device="cuda"))


def test_tokens_outside_the_vocabulary(plan, greedy, training, fp8):
    """They are reported, cost nothing, and change neither what comes before them nor other streams."""
    tokens, _ = greedy
    losses = plan.score(tokens)
    bad = tokens.clone()
    bad[1, 2], bad[2, STEPS - 1] = plan.config.vocab, -5
    got = plan.score(bad)
    assert fp8.decoder_error() == 1 and training.token_error() == 1
    assert got[1, 2] == 0 and got[2, STEPS - 1] == 0
    assert torch.equal(got[0], losses[0]) and torch.equal(got[1, :2], losses[1, :2])
    assert torch.equal(got[2, :-1], losses[2, :-1])


def test_tuning_the_tail(plan, greedy, training):
    """The tail's parameters against the transcripts: the summed score's gradients by autograd
    agree with its change under a step, and the tuned parts are the decoder's own."""
    tokens, _ = greedy
    w = plan.weights
    labels = tokens.t().reshape(-1).long()
    g = torch.Generator(device="cuda").manual_seed(8)
    stream_rows = (torch.randn((STEPS * STREAMS, plan.config.d_model), generator=g, device="cuda") * 2).half()
    gamma, beta = (t.clone().requires_grad_() for t in w.ln_post)
    table = w.token_table.clone().requires_grad_()
    _, states = training.layer_norm(stream_rows, gamma, beta)
    training.cross_entropy(states, table, labels).sum().backward()
    for leaf in (gamma, beta, table):
        assert torch.isfinite(leaf.grad).all() and leaf.grad.any()

    # The exact function's gradients of gamma and beta; what separates them is the 16-bit states
    # (half a step each, times the logits' gradient) and their 16-bit gradient.
    _, y, mean, rstd = ref.layer_norm(stream_rows, w.ln_post[0], w.ln_post[1], 1e-5)
    hat = (stream_rows.double() - mean) * rstd
    p = torch.softmax(y @ w.token_table.double().t(), 1)
    p[torch.arange(p.shape[0]), labels] -= 1
    dy = p @ w.token_table.double()
    # |d dy| <= |table|_2^2-ish of the state's rounding: bounded by the row norms of the table.
    norms = w.token_table.double().square().sum(1)
    spread = 2 * norms.max().sqrt() * (ref.rounding(y.abs(), torch.float16).square().sum(1).sqrt() * norms.max().sqrt())
    off = spread.unsqueeze(1) + 2.0 ** -10 * (p.abs() @ w.token_table.double().abs())
    for grad, exact, bound in ((beta.grad, dy.sum(0), off.sum(0)), (gamma.grad, (dy * hat).sum(0), (off * hat.abs()).sum(0))):
        assert ((grad.double() - exact).abs() <= bound + 2.0 ** -12).all()
