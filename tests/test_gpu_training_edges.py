"""Edges of the scoring and training operators: weights of exactly zero, logits that pass fp32's
range in one order of summation, loss gradients near the end of fp32's range, several pieces of
the vocabulary, column sums over very many rows, and the whole tail against 64 bits."""

from __future__ import annotations

import importlib

import pytest
import torch

import training_reference as ref
from conftest import PACKAGE

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def training(cuda):
    module = importlib.import_module(PACKAGE + ".training")
    module.token_error()
    yield module
    assert module.token_error() == 0
    assert importlib.import_module(PACKAGE + "._native").device_error() == 0


def operands(n, d, vocab, dtype, seed=0, scale=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed + n * 7 + d * 3 + vocab)
    x = torch.randn((n, d), generator=g, device="cuda").to(dtype)
    w = (torch.randn((vocab, d), generator=g, device="cuda") * scale).to(dtype)
    return g, x, w, torch.randn(n, generator=g, device="cuda")


# ---- a teacher's weights of zero ------------------------------------------------------


@pytest.mark.parametrize("n", [20, 300])
@pytest.mark.parametrize("masked", [40, 300])
def test_zero_weights_at_logits_of_minus_infinity(training, n, masked):
    """A teacher's entry whose probability is exactly 0 says nothing about its token, whose logit
    may be -infinity; a token there with a weight, once or repeated, costs an infinite loss."""
    d, vocab = 64, 1200
    g, x, w, dloss = operands(n, d, vocab, torch.bfloat16)
    x[:, 0], w[:, 0] = 0.0, 0.0
    tokens = torch.randint(masked, vocab, (n, 6), generator=g, device="cuda", dtype=torch.int32)
    logits = torch.randn((n, 6), generator=g, device="cuda")
    tokens[:, 2] = torch.randint(masked, (n,), generator=g, device="cuda", dtype=torch.int32)
    logits[:, 2] = -1e4  # exp(-1e4) is 0 in fp32, and in 64 bits
    left_out = tokens.clone()
    left_out[:, 2] = -1
    big = x.clone()
    big[:, 0], w[:masked, 0] = 1e20, -1e20
    losses, lse = training.distillation_forward(big, w, tokens, logits)
    targets = ref.teacher_targets(left_out - masked, logits, vocab - masked, 1.0)
    e_loss, e_lse, _ = ref.vocab_loss(x, w[masked:], targets)
    b_loss, b_lse = ref.loss_bounds(x, w[masked:], targets, e_loss, e_lse, 1.0, 6)
    assert ref.worst(lse, e_lse, b_lse) <= 1 and ref.worst(losses, e_loss, b_loss) <= 1
    without, lse_without = training.distillation_forward(big, w, left_out, logits)
    assert torch.equal(losses, without) and torch.equal(lse, lse_without)
    grads = training.distillation_backward(big, w, tokens, logits, lse, dloss)
    for a, b in zip(grads, training.distillation_backward(big, w, left_out, logits, lse, dloss)):
        assert torch.equal(a, b)
    # The same token twice and three times, among the masked ones, with weights above zero.
    tokens[::2, 3:5] = tokens[::2, 2:3]
    losses, lse = training.distillation_forward(big, w, tokens, logits)
    assert losses[::2].isposinf().all() and ref.worst(lse, e_lse, b_lse) <= 1
    assert torch.equal(losses[1::2], without[1::2])


# ---- sums that pass fp32's range on their way -------------------------------------------


@pytest.mark.parametrize("n", [20, 200, 1500])
def test_label_logits_whose_partial_sums_overflow(training, n):
    """Products of 1.5 x 2^127 that cancel: two negative ones in the first sixteen columns, their
    opposites 128 columns on.  A sum in the order of the columns passes -2^128 on its way, one of
    pairs 128 apart does not; where it is the label's logit, its loss and lse are those of the
    finite sum."""
    d, vocab = 256, 900
    g, x, w, _ = operands(n, d, vocab, torch.bfloat16)
    hot = [0, 8, 128, 136]
    x[:, hot], w[:, hot] = 0.0, 0.0
    labels = torch.full((n,), 333, device="cuda")
    labels[1::3] = torch.randint(vocab, (len(labels[1::3]),), generator=g, device="cuda")
    labels[2::7] = -100
    other = labels != 333
    w[333, :16], w[333, 128:144] = 0.0, 0.0  # next to them, small products would be lost
    targets = ref.label_targets(labels, vocab, -100)
    e_loss, e_lse, _ = ref.vocab_loss(x, w, targets)
    b_loss, b_lse = ref.loss_bounds(x, w, targets, e_loss, e_lse)
    x[~other] = x[~other].index_fill(1, torch.tensor(hot, device="cuda"), 1.5 * 2.0 ** 63)
    w[333, hot] = torch.tensor([-1.0, -1.0, 1.0, 1.0], device="cuda").bfloat16() * 2.0 ** 64
    losses, lse = training.cross_entropy_forward(x, w, labels)
    assert ref.worst(lse, e_lse, b_lse) <= 1 and ref.worst(losses, e_loss, b_loss) <= 1


# ---- loss gradients near the end of fp32's range -----------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("teacher,temperature,exponent", [(False, 1.0, 90), (False, 1.0, 112), (False, 1.0, 127),
                                                          (True, 1.0, 112), (True, 64.0, 110), (True, 64.0, 127),
                                                          (True, 2.0 ** -6, 127)])
@pytest.mark.parametrize("n", [20, 200, 300])
def test_loss_gradients_near_the_end_of_the_range(training, n, teacher, temperature, exponent, dtype):
    """Whatever the loss scale, the logits' gradient is held within its type: gradients that the
    results' type holds are exact to their rounding, others are infinite with their sign, and a
    column of zeros stays zero."""
    d, vocab, k = 64, 300, 3
    g, x, w, _ = operands(n, d, vocab, dtype)
    x[:, 7], w[:, 5] = 0.0, 0.0
    dloss = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, -1.0, 1.0) * 1.9 * 2.0 ** exponent
    if teacher:
        tokens = torch.randint(vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
        logits = torch.randn((n, k), generator=g, device="cuda")
        targets = ref.teacher_targets(tokens, logits, vocab, temperature)
        _, lse = training.distillation_forward(x, w, tokens, logits, temperature=temperature)
        dx, dw = training.distillation_backward(x, w, tokens, logits, lse, dloss, temperature=temperature)
    else:
        labels = torch.randint(vocab, (n,), generator=g, device="cuda")
        targets = ref.label_targets(labels, vocab, -100)
        _, lse = training.cross_entropy_forward(x, w, labels)
        dx, dw = training.cross_entropy_backward(x, w, labels, lse, dloss)
    assert not dx[:, 5].any() and not dw[:, 7].any()
    _, e_lse, grad = ref.vocab_loss(x, w, targets, temperature)
    full = grad * dloss.double().unsqueeze(1)
    e_dx, e_dw = full @ w.double(), full.t() @ x.double()
    bounds = ref.grad_bounds(x, w, grad, dloss, e_lse, e_dx, e_dw, temperature, targets[0], k if teacher else 1)
    top = torch.finfo(dtype).max
    for got, want, bound in zip((dx, dw), (e_dx, e_dw), bounds):
        got = got.double()
        inside = want.abs() + bound < top
        assert ((got - want).abs() <= bound)[inside].all()
        beyond = want.abs() - bound > top * (1 + torch.finfo(dtype).eps)
        assert torch.equal(got[beyond], torch.copysign(torch.full_like(want[beyond], torch.inf), want[beyond]))
        assert not torch.isnan(got).any()


# ---- norms whose rows one warp owns -------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [8, 64, 136, 256])
def test_norms_of_one_warp_rows(training, cols, dtype):
    """Rows that a single warp owns, in rings that are refilled many times (few stages of many
    groups): the residual's gradient, which no sum uses, is read before its stage is."""
    rows = 60001
    g = torch.Generator(device="cuda").manual_seed(cols)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    x, r, dy, dsum = (normal(rows, cols).to(dtype) for _ in range(4))
    gamma, beta = 1 + 0.2 * normal(cols), 0.3 * normal(cols)
    total, y, stats = training.layer_norm_forward(x, gamma, beta, residual=r)
    dx, dgamma, dbeta = training.layer_norm_backward(dy, total, gamma, stats, dsum=dsum)
    e_total, e_y, mean, rstd = ref.layer_norm(x, gamma, beta, 1e-5, r)
    assert torch.equal(total, e_total)
    assert ref.worst(y, e_y, ref.layer_norm_bound(total, gamma, beta, e_y, mean, rstd)) <= 1
    e = ref.layer_norm_grads(dy, total, gamma, mean, rstd, dsum)
    b = ref.layer_norm_grad_bounds(dy, total, gamma, mean, rstd, e[0], dsum)
    for got, want, bound in zip((dx, dgamma, dbeta), e, b):
        assert ref.worst(got, want, bound) <= 1
    for _ in range(20):
        again = training.layer_norm_backward(dy, total, gamma, stats, dsum=dsum)
        assert all(torch.equal(a, b) for a, b in zip(again, (dx, dgamma, dbeta)))
