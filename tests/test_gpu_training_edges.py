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


# ---- several pieces of the vocabulary ------------------------------------------------------


@pytest.mark.parametrize("teacher,dtype", [(False, torch.float16), (True, torch.bfloat16), (True, torch.float16)])
def test_pieces_with_several_column_tiles(training, teacher, dtype):
    """So many rows that the vocabulary takes two pieces, with two tiles across the width, entries
    at both sides of the border of the pieces, and each gradient alone."""
    n, d, vocab, k = 9000, 328, 30011, 5
    piece = 15104  # 512 MB of 9000 16-bit rows are 29696 columns; two equal pieces, rounded up to 256
    g, x, w, dloss = operands(n, d, vocab, dtype, scale=0.05)
    at_border = torch.tensor([0, piece - 1, piece, vocab - 1, 255, 256, piece + 255, piece + 256], device="cuda")
    if teacher:
        tokens = torch.randint(vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
        tokens[:, 0] = at_border[torch.arange(n, device="cuda") % 8].int()
        tokens[torch.rand((n, k), generator=g, device="cuda") < 0.1] = -1
        tokens[::9] = -1
        logits = torch.randn((n, k), generator=g, device="cuda")
        targets, temperature = ref.teacher_targets(tokens, logits, vocab, 1.5), 1.5
        losses, lse = training.distillation_forward(x, w, tokens, logits, temperature=1.5)
        backward = lambda **want: training.distillation_backward(x, w, tokens, logits, lse, dloss, temperature=1.5, **want)
    else:
        labels = torch.randint(vocab, (n,), generator=g, device="cuda")
        labels[:800] = at_border.repeat(100)
        labels[::9] = -100
        targets, temperature = ref.label_targets(labels, vocab, -100), 1.0
        losses, lse = training.cross_entropy_forward(x, w, labels)
        backward = lambda **want: training.cross_entropy_backward(x, w, labels, lse, dloss, **want)
    e_loss, e_lse, grad = ref.vocab_loss(x, w, targets, temperature)
    b_loss, b_lse = ref.loss_bounds(x, w, targets, e_loss, e_lse, temperature, k if teacher else 1)
    assert ref.worst(lse, e_lse, b_lse) <= 1 and ref.worst(losses, e_loss, b_loss) <= 1
    full = grad * dloss.double().unsqueeze(1)
    e_dx, e_dw = full @ w.double(), full.t() @ x.double()
    del full
    b_dx, b_dw = ref.grad_bounds(x, w, grad, dloss, e_lse, e_dx, e_dw, temperature, targets[0], k if teacher else 1)
    dx, dw = backward()
    assert ref.worst(dx, e_dx, b_dx) <= 1 and ref.worst(dw, e_dw, b_dw) <= 1
    assert not dx[::9].any()
    assert torch.equal(backward(want_dx=False)[1], dw)
    alone = backward(want_dweight=False)[0]
    assert ref.worst(alone, e_dx, b_dx) <= 1 and not alone[::9].any()


# ---- the gain of the logits' gradient ------------------------------------------------------


@pytest.mark.parametrize("teacher", [False, True])
@pytest.mark.parametrize("n", [200, 300])
def test_gain_keeps_the_steps_fine(training, n, teacher):
    """Loss gradients from 1 to 1.12 lie just above a power of two, where a 16-bit type's steps are
    coarsest.  Unsure rows (p near 1/1000) leave the targets' elements of dz there, and dx and dW
    mostly those times a row of 16-bit numbers.

    In shares of 2^-8: rounding v uniformly to steps of 2 at [1, 2) leaves 1/sqrt(3)/v.  As it is, v
    is 1.06 on average, 0.545; a quarter-octave gain of 1.68 takes it to 1.78, 0.324.  The results'
    own rounding, over mantissas spread evenly in their logarithm (mean square 1.5 / log 2), leaves
    1/sqrt(3)/1.471 = 0.392.  Together 0.671 and 0.509, which is 1.71 and 1.30 times the latter, with
    some 0.05 of sampling (the same roundings of 64-bit products: 1.55 to 1.66 and 1.24 to 1.27)."""
    d, vocab = 512, 1000
    g, x, w, _ = operands(n, d, vocab, torch.bfloat16, scale=0.05)
    dloss = 1.0 + 0.12 * torch.rand(n, generator=g, device="cuda")
    labels = torch.randperm(vocab, generator=g, device="cuda")[:n]
    targets = ref.label_targets(labels, vocab, -100)
    if teacher:
        tokens, logits = labels.int().unsqueeze(1), torch.zeros((n, 1), device="cuda")
        _, lse = training.distillation_forward(x, w, tokens, logits)
        dx, dw = training.distillation_backward(x, w, tokens, logits, lse, dloss)
    else:
        _, lse = training.cross_entropy_forward(x, w, labels)
        dx, dw = training.cross_entropy_backward(x, w, labels, lse, dloss)
    _, _, grad = ref.vocab_loss(x, w, targets)
    full = grad * dloss.double().unsqueeze(1)
    for got, want in ((dx, full @ w.double()), (dw[labels], (full.t() @ x.double())[labels])):
        once = (want.to(torch.bfloat16).double() - want).norm()
        assert float((got.double() - want).norm() / once) < 1.4


# ---- the sums over the rows of a norm --------------------------------------------------------


def test_column_sums_of_very_many_rows(training):
    """2^31 elements and more, with a gradient in the first 100 and the last 700 rows only: every
    other row adds exact zeros, so each of these must be in the sums once, and nothing else."""
    rows, cols = (1 << 31) // 1280 + 1000, 1280
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((rows, cols), generator=g, device="cuda", dtype=torch.bfloat16)
    dy = torch.zeros_like(x)
    where = torch.cat([torch.arange(100), torch.arange(rows - 700, rows)]).cuda()
    dy[where] = torch.randn((800, cols), generator=g, device="cuda", dtype=torch.bfloat16)
    gamma, beta = torch.rand(cols, generator=g, device="cuda") + 0.5, torch.randn(cols, generator=g, device="cuda")
    total, _, stats = training.layer_norm_forward(x, gamma, beta)
    _, dgamma, dbeta = training.layer_norm_backward(dy, total, gamma, stats, want_dx=False)
    _, _, mean, rstd = ref.layer_norm(x[where], gamma, beta, 1e-5)
    e_dx, e_dg, e_db = ref.layer_norm_grads(dy[where], x[where], gamma, mean, rstd)
    _, b_dg, b_db = ref.layer_norm_grad_bounds(dy[where], x[where], gamma, mean, rstd, e_dx)
    assert ref.worst(dgamma, e_dg, b_dg) <= 1 and ref.worst(dbeta, e_db, b_db) <= 1
    # A row that is lost or taken twice moves each sum by its own term, of size 0.6 to 0.8: the bounds,
    # 802 x 2^-24 x 800 x 0.8 = 0.031 and less, lie well below that.
    assert b_dg.max() < 0.05 and b_db.max() < 0.05


# ---- the tail of a decoder ---------------------------------------------------------------------


def test_tail_against_64_bits(training):
    """Final norm and token loss of the decoder's own parameters: every gradient against 64 bits
    from the 16-bit states that the norm returned, with bounds well below the gradients, and the
    summed score's change under a step of gamma and beta."""
    dec = importlib.import_module(PACKAGE + ".decoder")
    config = dec.DecoderConfig(layers=1)
    weights = dec.DecoderWeights.from_checkpoint(
        dec.add_synthetic_decoder({}, config, seed=31, device=torch.device("cuda:0")), config)
    n, d, vocab = 18, config.d_model, config.vocab
    g = torch.Generator(device="cuda").manual_seed(8)
    rows = (torch.randn((n, d), generator=g, device="cuda") * 2).half()
    labels = torch.randint(vocab, (n,), generator=g, device="cuda")
    gamma, beta = (t.clone().requires_grad_() for t in weights.ln_post)
    table = weights.token_table.clone().requires_grad_()
    leaf = rows.clone().requires_grad_()
    _, states = training.layer_norm(leaf, gamma, beta)
    training.cross_entropy(states, table, labels).sum().backward()

    y, w = states.detach(), weights.token_table
    targets = ref.label_targets(labels, vocab, -100)
    ones = torch.ones(n, device="cuda")
    _, lse, grad = ref.vocab_loss(y, w, targets)
    e_dy, e_dw = grad @ w.double(), grad.t() @ y.double()
    b_dy, b_dw = ref.grad_bounds(y, w, grad, ones, lse, e_dy, e_dw, 1.0, targets[0], 1, 2)
    assert ref.worst(table.grad, e_dw, b_dw) <= 1
    _, _, mean, rstd = ref.layer_norm(rows, *weights.ln_post, 1e-5)
    e_dx, e_dg, e_db = ref.layer_norm_grads(e_dy, rows, weights.ln_post[0], mean, rstd)
    # The norm's backward is given dy within b_dy of e_dy: its own bounds at that size, and b_dy
    # carried through it.
    size = e_dy.abs() + b_dy
    hat = ((rows.double() - mean) * rstd).abs()
    b_dx, b_dg, b_db = ref.layer_norm_grad_bounds(size, rows, weights.ln_post[0], mean, rstd, e_dx)
    off = b_dy * weights.ln_post[0].double().abs()
    carried = rstd * (off + off.mean(1, keepdim=True) + hat * (off * hat).mean(1, keepdim=True))
    checks = ((beta.grad, e_db, b_db + b_dy.sum(0)), (gamma.grad, e_dg, b_dg + (b_dy * hat).sum(0)),
              (leaf.grad, e_dx, b_dx + carried * 1.01), (table.grad, e_dw, b_dw))
    for got, want, bound in checks:
        assert ref.worst(got, want, bound) <= 1
        assert bound.norm() < 0.25 * want.norm()

    # A step up the gradient of gamma and beta, and one down: half the score's difference is the
    # gradient times the step but for the exact function's third-order term (in 64 bits), the
    # states' roundings (half a step each, times dy) and the losses' own errors.
    scale = 0.05 / max(gamma.grad.abs().max(), beta.grad.abs().max())
    dg, db = gamma.grad * scale, beta.grad * scale

    def score(sign):
        _, s, _ = training.layer_norm_forward(rows, weights.ln_post[0] + sign * dg, weights.ln_post[1] + sign * db)
        losses, _ = training.cross_entropy_forward(s, w, labels)
        return losses.double().sum(), s

    def exact(sign):
        s = ref.layer_norm(rows, weights.ln_post[0] + sign * dg, weights.ln_post[1] + sign * db, 1e-5)[1]
        z = s @ w.double().t()
        return (torch.logsumexp(z, 1) - z[torch.arange(n), labels]).sum()

    (up, s), (down, _) = score(1), score(-1)
    slope, e_slope = (up - down) / 2, (exact(1) - exact(-1)) / 2
    predicted = (gamma.grad.double() * dg).sum() + (beta.grad.double() * db).sum()
    e_predicted = (e_dg * dg).sum() + (e_db * db).sum()
    e_loss, e_lse, _ = ref.vocab_loss(s, w, targets)
    noise = (ref.rounding(s.double().abs() + 0.1, torch.float16) * (e_dy.abs() + 0.1 * w.double().abs().amax(0))).sum() \
        + ref.loss_bounds(s, w, targets, e_loss, e_lse)[0].sum()
    room = (checks[0][2] * db.abs()).sum() + (checks[1][2] * dg.abs()).sum()
    assert (slope - predicted).abs() <= (e_slope - e_predicted).abs() + noise + room
    assert noise + room < 0.5 * predicted  # the step is seen
