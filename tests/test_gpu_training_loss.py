"""Cross entropy and distillation over the vocabulary, with gradients, against 64 bits
(bounds in training_reference)."""

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


def compare(forward, backward, x, w, dloss, targets, temperature=1.0, entries=1):
    losses, lse = forward()
    e_loss, e_lse, g = ref.vocab_loss(x, w, targets, temperature)
    b_loss, b_lse = ref.loss_bounds(x, w, targets, e_loss, e_lse, temperature, entries)
    assert ref.worst(lse, e_lse, b_lse) <= 1
    assert ref.worst(losses, e_loss, b_loss) <= 1
    dx, dw = backward(lse)
    full = g * dloss.double().unsqueeze(1)
    e_dx, e_dw = full @ w.double(), full.t() @ x.double()
    b_dx, b_dw = ref.grad_bounds(x, w, g, dloss, e_lse, e_dx, e_dw, temperature, targets[0], entries)
    assert ref.worst(dx, e_dx, b_dx) <= 1
    assert ref.worst(dw, e_dw, b_dw) <= 1
    return losses, lse, dx, dw


SHAPES = [(1, 8, 1), (1, 64, 2), (5, 72, 130), (128, 384, 513), (129, 384, 512), (20, 1280, 1003), (257, 136, 1999),
          (300, 512, 2049), (640, 264, 777), (1025, 768, 1500)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,vocab", SHAPES)
def test_cross_entropy(training, n, d, vocab, dtype):
    g, x, w, dloss = operands(n, d, vocab, dtype)
    labels = torch.randint(vocab, (n,), generator=g, device="cuda")
    labels[torch.rand(n, generator=g, device="cuda") < 0.2] = -100
    labels = labels if n % 2 else labels.to(torch.int32)  # both label types
    compare(lambda: training.cross_entropy_forward(x, w, labels),
            lambda lse: training.cross_entropy_backward(x, w, labels, lse, dloss),
            x, w, dloss, ref.label_targets(labels, vocab, -100))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,temperature", [(1, 1.0), (5, 2.0), (33, 1.5), (256, 4.0)])
@pytest.mark.parametrize("n,d,vocab", [(1, 64, 300), (7, 512, 1001), (131, 136, 777), (300, 384, 1300)])
def test_distillation(training, n, d, vocab, k, temperature, dtype):
    g, x, w, dloss = operands(n, d, vocab, dtype, seed=k)
    # Tokens in no order, some twice, some left out, logits of every accepted type.
    tokens = torch.randint(vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
    tokens[torch.rand((n, k), generator=g, device="cuda") < 0.1] = -1
    logits = torch.randn((n, k), generator=g, device="cuda") * 4
    logits = logits.to([torch.float32, torch.float16, torch.bfloat16][k % 3])
    logits[torch.rand((n, k), generator=g, device="cuda") < 0.05] = -torch.inf
    compare(lambda: training.distillation_forward(x, w, tokens, logits, temperature=temperature),
            lambda lse: training.distillation_backward(x, w, tokens, logits, lse, dloss, temperature=temperature),
            x, w, dloss, ref.teacher_targets(tokens, logits, vocab, temperature), temperature, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,vocab", [(3, 65536, 40), (300, 8200, 1030), (20000, 8, 3), (40, 8, 300001),
                                       (2000, 4096, 1)])
def test_extreme_shapes(training, n, d, vocab, dtype):
    g, x, w, dloss = operands(n, d, vocab, dtype, scale=d ** -0.5)
    labels = torch.randint(vocab, (n,), generator=g, device="cuda")
    labels[torch.rand(n, generator=g, device="cuda") < 0.2] = -100
    compare(lambda: training.cross_entropy_forward(x, w, labels),
            lambda lse: training.cross_entropy_backward(x, w, labels, lse, dloss),
            x, w, dloss, ref.label_targets(labels, vocab, -100))
    tokens = torch.randint(vocab, (n, 33), generator=g, device="cuda", dtype=torch.int32)
    logits = torch.randn((n, 33), generator=g, device="cuda")
    compare(lambda: training.distillation_forward(x, w, tokens, logits),
            lambda lse: training.distillation_backward(x, w, tokens, logits, lse, dloss),
            x, w, dloss, ref.teacher_targets(tokens, logits, vocab, 1.0), 1.0, 33)


def test_pieces_and_splits(training):
    """Enough rows that the vocabulary takes several pieces of G, whose dx adds up in fp32; the
    last piece is narrower than the others and ends inside a tile."""
    n, d, vocab = 9000, 72, 30011
    g, x, w, dloss = operands(n, d, vocab, torch.bfloat16)
    labels = torch.randint(vocab, (n,), generator=g, device="cuda")
    labels[:7] = torch.tensor([0, vocab - 1, 14847, 14848, 255, 256, -100])
    losses, lse = training.cross_entropy_forward(x, w, labels)
    dx, dw = training.cross_entropy_backward(x, w, labels, lse, dloss)
    part = slice(0, 600)  # dx row by row; dw against the sum over all rows, by columns
    targets = ref.label_targets(labels[part], vocab, -100)
    e_loss, e_lse, grad = ref.vocab_loss(x[part], w, targets)
    b_loss, b_lse = ref.loss_bounds(x[part], w, targets, e_loss, e_lse)
    assert ref.worst(losses[part], e_loss, b_loss) <= 1 and ref.worst(lse[part], e_lse, b_lse) <= 1
    full = grad * dloss[part].double().unsqueeze(1)
    e_dx = full @ w.double()
    b_dx, _ = ref.grad_bounds(x[part], w, grad, dloss[part], e_lse, e_dx, full.t() @ x[part].double())
    assert ref.worst(dx[part], e_dx, b_dx) <= 1
    z = x.double() @ w.double().t()
    p = torch.softmax(z, 1)
    t, valid, _ = ref.label_targets(labels, vocab, -100)
    grad = (p - t) * valid.unsqueeze(1)
    e_dw = (grad * dloss.double().unsqueeze(1)).t() @ x.double()
    _, b_dw = ref.grad_bounds(x, w, grad, dloss, torch.logsumexp(z, 1), dx.double(), e_dw)
    assert ref.worst(dw, e_dw, b_dw) <= 1


def test_largest_vocabulary_few_rows(training):
    n, d, vocab = 20, 384, 51866
    g, x, w, dloss = operands(n, d, vocab, torch.float16)
    labels = torch.randint(vocab, (n,), generator=g, device="cuda", dtype=torch.int32)
    labels[:2] = torch.tensor([0, vocab - 1])
    compare(lambda: training.cross_entropy_forward(x, w, labels),
            lambda lse: training.cross_entropy_backward(x, w, labels, lse, dloss),
            x, w, dloss, ref.label_targets(labels, vocab, -100))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [60, 500])
def test_ignored_rows_reach_nothing(training, n, dtype):
    """Rows without a target may hold anything: NaN and infinities in their states (and in the
    losses' gradients) change no other row and no gradient."""
    d, vocab = 128, 900
    g, x, w, dloss = operands(n, d, vocab, dtype)
    labels = torch.randint(vocab, (n,), generator=g, device="cuda")
    out = torch.rand(n, generator=g, device="cuda") < 0.4
    labels[out] = 50257
    bad, bad_dloss = x.clone(), dloss.clone()
    bad[out] = torch.tensor([float("nan"), float("inf"), -float("inf"), 65504.0] * (d // 4), device="cuda").to(dtype)
    bad_dloss[out] = float("nan")
    losses, lse = training.cross_entropy_forward(x, w, labels, ignore_index=50257)
    losses_b, lse_b = training.cross_entropy_forward(bad, w, labels, ignore_index=50257)
    assert not losses[out].any() and torch.equal(losses, losses_b) and torch.equal(lse[~out], lse_b[~out])
    dx, dw = training.cross_entropy_backward(x, w, labels, lse, dloss, ignore_index=50257)
    dx_b, dw_b = training.cross_entropy_backward(bad, w, labels, lse_b, bad_dloss, ignore_index=50257)
    assert not dx[out].any() and torch.equal(dx, dx_b) and torch.equal(dw, dw_b)


@pytest.mark.parametrize("teacher", [False, True])
@pytest.mark.parametrize("n", [60, 200, 500])
def test_large_gradients_of_ignored_rows(training, n, teacher):
    """A finite but huge loss gradient at a row without a target scales nothing: neither fp16's
    range nor its precision is spent on it."""
    d, vocab, k = 128, 900, 40
    g, x, w, dloss = operands(n, d, vocab, torch.float16)
    labels = torch.randint(vocab, (n,), generator=g, device="cuda")
    tokens = torch.randint(vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
    logits = torch.randn((n, k), generator=g, device="cuda")
    logits[:, :33] = -torch.inf  # the entries that count come late
    out = torch.rand(n, generator=g, device="cuda") < 0.4
    labels[out], tokens[out] = -100, -1
    huge = torch.where(out, 1e30, dloss)
    if teacher:
        losses, lse = training.distillation_forward(x, w, tokens, logits)
        grads = [training.distillation_backward(x, w, tokens, logits, lse, g) for g in (dloss, huge)]
    else:
        losses, lse = training.cross_entropy_forward(x, w, labels)
        grads = [training.cross_entropy_backward(x, w, labels, lse, g) for g in (dloss, huge)]
    assert not losses[out].any() and not grads[0][0][out].any()
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


@pytest.mark.parametrize("n", [20, 300])
@pytest.mark.parametrize("masked", [40, 300, 777])
def test_logits_of_minus_infinity(training, n, masked):
    """bf16 reaches products past fp32: columns whose logit is -infinity, a whole tile of them
    too, count as probability 0, whatever their place; a label there has an infinite loss."""
    d, vocab = 64, 1200
    g, x, w, dloss = operands(n, d, vocab, torch.bfloat16)
    x[:, 0], w[:, 0] = 0.0, 0.0
    labels = torch.randint(masked, vocab, (n,), generator=g, device="cuda")
    e_loss, e_lse, grad = ref.vocab_loss(x, w[masked:], ref.label_targets(labels - masked, vocab - masked, -100))
    targets = ref.label_targets(labels - masked, vocab - masked, -100)
    b_loss, b_lse = ref.loss_bounds(x, w[masked:], targets, e_loss, e_lse)
    full = grad * dloss.double().unsqueeze(1)
    e_dx, e_dw = full @ w[masked:].double(), full.t() @ x.double()
    b_dx, b_dw = ref.grad_bounds(x, w[masked:], grad, dloss, e_lse, e_dx, e_dw)
    big = x.clone()
    big[:, 0], w[:masked, 0] = 1e20, -1e20
    losses, lse = training.cross_entropy_forward(big, w, labels)
    assert ref.worst(lse, e_lse, b_lse) <= 1 and ref.worst(losses, e_loss, b_loss) <= 1
    dx, dw = training.cross_entropy_backward(big, w, labels, lse, dloss)
    assert ref.worst(dx, e_dx, b_dx) <= 1 and ref.worst(dw[masked:, 1:], e_dw[:, 1:], b_dw[:, 1:]) <= 1
    assert not dw[:masked].any()
    labels[::2] = masked // 2
    losses, lse_there = training.cross_entropy_forward(big, w, labels)
    assert losses[::2].isposinf().all() and ref.worst(lse_there, e_lse, b_lse) <= 1


@pytest.mark.parametrize("n,valid", [(700, 0), (700, 1), (700, 31), (700, 33), (700, 64), (700, 65), (700, 255),
                                     (700, 256), (700, 257), (700, 699), (100, 1), (100, 63), (100, 70), (300, 290)])
def test_counts_of_valid_rows(training, n, valid):
    """The valid rows move together for the gradients: their count around the ends of K blocks,
    warps and tiles, with NaN in all others (and in memory that the workspace gets)."""
    d, vocab = 136, 777
    g, x, w, dloss = operands(n, d, vocab, torch.bfloat16)
    labels = torch.full((n,), -100, dtype=torch.int64, device="cuda")
    keep = torch.randperm(n, generator=g, device="cuda")[:valid]
    labels[keep] = torch.randint(vocab, (valid,), generator=g, device="cuda")
    out = labels < 0
    x[out] = float("nan")
    losses, lse = training.cross_entropy_forward(x, w, labels)
    poison = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]
    del poison  # cached by the allocator: the workspace's memory starts as NaN
    dx, dw = training.cross_entropy_backward(x, w, labels, lse, dloss)
    clean = torch.where(out.unsqueeze(1), 0.0, x).to(x.dtype)
    targets = ref.label_targets(labels, vocab, -100)
    _, e_lse, grad = ref.vocab_loss(clean, w, targets)
    dloss = torch.where(out, 0.0, dloss)
    full = grad * dloss.double().unsqueeze(1)
    e_dx, e_dw = full @ w.double(), full.t() @ clean.double()
    b_dx, b_dw = ref.grad_bounds(clean, w, grad, dloss, e_lse, e_dx, e_dw)
    assert not dx[out].any()
    assert ref.worst(dx, e_dx, b_dx) <= 1 and ref.worst(dw, e_dw, b_dw) <= 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,valid", [(1, 1), (7, 7), (8, 8), (8, 3), (9, 9), (16, 16), (17, 17), (33, 20), (100, 97),
                                     (128, 128), (129, 128), (257, 1), (300, 9), (300, 33), (700, 64), (700, 128)])
@pytest.mark.parametrize("teacher", [False, True])
def test_few_rows_are_rounded_once(training, n, valid, teacher, dtype):
    """With up to 128 rows that have a target (a teacher up to 256 rows: rows at all) the logits'
    gradient is held in two parts, so that only the results are rounded to 16 bits."""
    d, vocab, k = 72, 500, 3
    g, x, w, dloss = operands(n, d, vocab, dtype, seed=valid)
    out = torch.ones(n, dtype=torch.bool, device="cuda")
    out[torch.randperm(n, generator=g, device="cuda")[:valid]] = False
    x[out], dloss[out] = float("nan"), float("nan")
    if teacher:
        tokens = torch.randint(vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
        tokens[out] = -1
        logits = torch.randn((n, k), generator=g, device="cuda")
        targets = ref.teacher_targets(tokens, logits, vocab, 1.0)
        _, lse = training.distillation_forward(x, w, tokens, logits)
        backward = lambda: training.distillation_backward(x, w, tokens, logits, lse, dloss)
    else:
        labels = torch.randint(vocab, (n,), generator=g, device="cuda")
        labels[out] = -100
        targets = ref.label_targets(labels, vocab, -100)
        _, lse = training.cross_entropy_forward(x, w, labels)
        backward = lambda: training.cross_entropy_backward(x, w, labels, lse, dloss)
    poison = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]
    del poison  # the workspace's memory starts as NaN
    dx, dw = backward()
    clean = torch.where(out.unsqueeze(1), 0.0, x).to(dtype)
    dloss = torch.where(out, 0.0, dloss)
    _, e_lse, grad = ref.vocab_loss(clean, w, targets)
    full = grad * dloss.double().unsqueeze(1)
    e_dx, e_dw = full @ w.double(), full.t() @ clean.double()
    parts = 1 if teacher and 128 < n <= 256 else 2
    b_dx, b_dw = ref.grad_bounds(clean, w, grad, dloss, e_lse, e_dx, e_dw, 1.0, targets[0], k if teacher else 1, parts)
    assert ref.worst(dx, e_dx, b_dx) <= 1 and ref.worst(dw, e_dw, b_dw) <= 1
    assert not dx[out].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,k", [(40, 1, 216), (300, 2, 256), (70, 5, 250), (280, 40, 64)])
def test_tokens_that_occur_many_times(training, n, vocab, k, dtype):
    """Few different tokens in many entries: their probabilities add up before they meet the
    softmax (with one token in all, the gradient is that of 1 - 1)."""
    g, x, w, dloss = operands(n, 64, vocab, dtype, seed=3)
    tokens = torch.randint(vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
    logits = torch.randn((n, k), generator=g, device="cuda") * 3
    compare(lambda: training.distillation_forward(x, w, tokens, logits, temperature=0.5),
            lambda lse: training.distillation_backward(x, w, tokens, logits, lse, dloss, temperature=0.5),
            x, w, dloss, ref.teacher_targets(tokens, logits, vocab, 0.5), 0.5, k)


@pytest.mark.parametrize("n,valid", [(700, 0), (700, 1), (700, 63), (700, 65), (700, 256), (700, 257), (700, 700),
                                     (257, 200), (256, 100), (100, 0), (100, 33)])
@pytest.mark.parametrize("k", [3, 40, 200])
def test_counts_of_valid_rows_with_a_teacher(training, n, valid, k):
    """The same with a teacher, whose rows move above 256 rows: entries left out of every row
    somewhere, whole rows of them, NaN in the states and gradients of those."""
    d, vocab, temperature = 72, 600, 1.5
    g, x, w, dloss = operands(n, d, vocab, torch.float16, seed=k)
    tokens = torch.randint(vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
    tokens[torch.rand((n, k), generator=g, device="cuda") < 0.2] = -1
    logits = (torch.randn((n, k), generator=g, device="cuda") * 3).half()
    out = torch.ones(n, dtype=torch.bool, device="cuda")
    out[torch.randperm(n, generator=g, device="cuda")[:valid]] = False
    tokens[out] = -1
    x[out], dloss[out] = float("nan"), float("nan")
    losses, lse = training.distillation_forward(x, w, tokens, logits, temperature=temperature)
    poison = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]
    del poison  # cached by the allocator: the workspace's memory starts as NaN
    dx, dw = training.distillation_backward(x, w, tokens, logits, lse, dloss, temperature=temperature)
    targets = ref.teacher_targets(tokens, logits, vocab, temperature)
    out |= ~targets[1]  # and rows whose entries were all left out by chance
    clean = torch.where(out.unsqueeze(1), 0.0, x).to(x.dtype)
    e_loss, e_lse, grad = ref.vocab_loss(clean, w, targets, temperature)
    b_loss, _ = ref.loss_bounds(clean, w, targets, e_loss, e_lse, temperature, k)
    assert ref.worst(losses, e_loss, b_loss) <= 1 and not losses[out].any() and not dx[out].any()
    dloss = torch.where(out, 0.0, dloss)
    full = grad * dloss.double().unsqueeze(1)
    e_dx, e_dw = full @ w.double(), full.t() @ clean.double()
    b_dx, b_dw = ref.grad_bounds(clean, w, grad, dloss, e_lse, e_dx, e_dw, temperature)
    assert ref.worst(dx, e_dx, b_dx) <= 1 and ref.worst(dw, e_dw, b_dw) <= 1


def test_rows_without_teacher_entries(training):
    n, d, vocab, k = 40, 64, 500, 4
    g, x, w, dloss = operands(n, d, vocab, torch.float16)
    tokens = torch.randint(vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
    logits = torch.randn((n, k), generator=g, device="cuda")
    tokens[3] = -1
    logits[5] = -torch.inf
    logits[6, :3] = -torch.inf  # one entry left: t = 1
    logits[7] = torch.finfo(torch.float32).min  # the lowest value masks nothing: equal shares
    tokens[8, 0] = -1
    logits[8, 0] = float("nan")  # a left-out entry may hold anything
    x[3] = float("nan")
    targets = ref.teacher_targets(tokens, logits, vocab, 1.0)
    losses, lse = training.distillation_forward(x, w, tokens, logits)
    dx, dw = training.distillation_backward(x, w, tokens, logits, lse, dloss)
    assert losses[3] == 0 and losses[5] == 0 and not dx[[3, 5]].any()
    clean = x.clone()
    clean[3] = 0
    e_loss, e_lse, grad = ref.vocab_loss(clean, w, targets)
    b_loss, _ = ref.loss_bounds(clean, w, targets, e_loss, e_lse, 1.0, k)
    assert ref.worst(losses, e_loss, b_loss) <= 1
    full = grad * dloss.double().unsqueeze(1)
    e_dx, e_dw = full @ w.double(), full.t() @ clean.double()
    b_dx, b_dw = ref.grad_bounds(clean, w, grad, dloss, e_lse, e_dx, e_dw)
    assert ref.worst(dx, e_dx, b_dx) <= 1 and ref.worst(dw, e_dw, b_dw) <= 1


@pytest.mark.parametrize("n", [50, 400])
def test_ignored_token_of_the_vocabulary(training, n):
    """ignore_index may be a token: its rows are ignored, its column of the softmax stays."""
    g, x, w, dloss = operands(n, 64, 300, torch.float16)
    labels = torch.randint(8, (n,), generator=g, device="cuda")
    compare(lambda: training.cross_entropy_forward(x, w, labels, ignore_index=5),
            lambda lse: training.cross_entropy_backward(x, w, labels, lse, dloss, ignore_index=5),
            x, w, dloss, ref.label_targets(labels, 300, 5))


@pytest.mark.parametrize("temperature", [2.0 ** -6, 2.0 ** 6])
def test_extreme_temperatures(training, temperature):
    """Both ends of the range, with logits that leave fp32's range when divided by it."""
    n, d, vocab, k = 70, 64, 500, 6
    g, x, w, dloss = operands(n, d, vocab, torch.bfloat16, scale=0.02)
    tokens = torch.randint(vocab, (n, k), generator=g, device="cuda", dtype=torch.int32)
    logits = torch.randn((n, k), generator=g, device="cuda")
    logits[:10] = torch.finfo(torch.float32).min
    logits[20, 2] = torch.finfo(torch.float32).max
    clipped = torch.where(logits.abs() > 1e30, logits.sign() * 1e30, logits)  # the same softmax in 64 bits
    compare(lambda: training.distillation_forward(x, w, tokens, logits, temperature=temperature),
            lambda lse: training.distillation_backward(x, w, tokens, logits, lse, dloss, temperature=temperature),
            x, w, dloss, ref.teacher_targets(tokens, clipped, vocab, temperature), temperature, k)


def test_offsets_past_32_bits(training):
    """A table of more than 2^31 elements: tokens at both of its ends."""
    n, d, vocab = 5, 1280, 1_700_000
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn((vocab, d), generator=g, device="cuda", dtype=torch.bfloat16)
    w *= 0.02
    x = torch.randn((n, d), generator=g, device="cuda").to(torch.bfloat16)
    labels = torch.tensor([0, vocab - 1, 1_677_721, 1_677_722, 5], device="cuda")
    dloss = torch.tensor([1.0, 2.0, 0.5, 1.5, -1.0], device="cuda")
    losses, lse = training.cross_entropy_forward(x, w, labels)
    dx, dw = training.cross_entropy_backward(x, w, labels, lse, dloss)
    z = torch.cat([x.double() @ part.double().t() for part in w.split(200_000)], 1)
    e_lse = torch.logsumexp(z, 1)
    rows = torch.arange(n, device="cuda")
    off = ref.logit_bound(x, w[:1000]) * 1.5 + 2.0 ** -16  # rows of the table are alike
    assert ((lse - e_lse).abs() <= off).all() and ((losses - (e_lse - z[rows, labels])).abs() <= 2 * off).all()
    p = (z - e_lse.unsqueeze(1)).exp()
    p[rows, labels] -= 1
    p *= dloss.double().unsqueeze(1)
    e_dx = sum(part @ rows_.double() for part, rows_ in zip(p.split(200_000, 1), w.split(200_000)))
    # G's half step and the logits' error, over the products' magnitudes; one rounding at the end.
    share = 2.0 ** -9 + torch.expm1(3 * off).max() + vocab * 2 * ref.U32
    mag = sum(part.abs() @ rows_.double().abs() for part, rows_ in zip(p.split(200_000, 1), w.split(200_000)))
    assert ((dx.double() - e_dx).abs() <= share * mag + ref.rounding(e_dx.abs(), torch.bfloat16)).all()
    for part in (slice(0, 1000), slice(1_677_700, 1_678_700), slice(vocab - 1000, vocab)):
        e_dw = p[:, part].t() @ x.double()
        mag = p[:, part].abs().t() @ x.double().abs()
        assert ((dw[part].double() - e_dw).abs() <= share * mag + ref.rounding(e_dw.abs(), torch.bfloat16) + 1e-9).all()


def test_all_rows_ignored(training):
    g, x, w, dloss = operands(33, 64, 200, torch.bfloat16)
    labels = torch.full((33,), -100, device="cuda")
    losses, lse = training.cross_entropy_forward(x, w, labels)
    dx, dw = training.cross_entropy_backward(x, w, labels, lse, dloss)
    assert not losses.any() and not dx.any() and not dw.any()


def test_tokens_outside_the_vocabulary(training):
    """Treated as ignored, and reported."""
    g, x, w, dloss = operands(10, 64, 200, torch.float16)
    labels = torch.randint(200, (10,), generator=g, device="cuda")
    assert training.token_error() == 0
    for bad in (200, 2 ** 31, -5):
        wrong, ignored = labels.clone(), labels.clone()
        wrong[4], ignored[4] = bad, -100
        losses, lse = training.cross_entropy_forward(x, w, wrong)
        assert training.token_error() == 1 and training.token_error() == 0
        assert torch.equal(losses, training.cross_entropy_forward(x, w, ignored)[0])
        got = training.cross_entropy_backward(x, w, wrong, lse, dloss)
        assert training.token_error() == 1
        for a, b in zip(got, training.cross_entropy_backward(x, w, ignored, lse, dloss)):
            assert torch.equal(a, b)
    tokens = torch.randint(200, (10, 3), generator=g, device="cuda", dtype=torch.int32)
    logits = torch.randn((10, 3), generator=g, device="cuda")
    wrong, left_out = tokens.clone(), tokens.clone()
    wrong[2, 1], left_out[2, 1] = 200, -1
    assert torch.equal(training.distillation_forward(x, w, wrong, logits)[0],
                       training.distillation_forward(x, w, left_out, logits)[0])
    assert training.token_error() == 1


@pytest.mark.parametrize("scale", [2.0 ** -30, 1.0, 2.0 ** 12])
def test_gradient_scales(training, scale):
    """G is held in 16 bits whatever the loss scale: the gradients scale with dloss exactly (by
    powers of two), as long as the outputs' type holds them."""
    g, x, w, dloss = operands(300, 128, 1000, torch.bfloat16)
    labels = torch.randint(1000, (300,), generator=g, device="cuda")
    _, lse = training.cross_entropy_forward(x, w, labels)
    dx, dw = training.cross_entropy_backward(x, w, labels, lse, dloss)
    dx_s, dw_s = training.cross_entropy_backward(x, w, labels, lse, dloss * scale)
    assert torch.equal(dx_s.float(), dx.float() * scale) and torch.equal(dw_s.float(), dw.float() * scale)


def test_zero_gradient(training):
    g, x, w, _ = operands(50, 64, 300, torch.float16)
    labels = torch.randint(300, (50,), generator=g, device="cuda")
    _, lse = training.cross_entropy_forward(x, w, labels)
    dx, dw = training.cross_entropy_backward(x, w, labels, lse, torch.zeros(50, device="cuda"))
    assert not dx.any() and not dw.any()


def test_subsets_of_the_gradients(training):
    """dweight alone has the same bits; dx alone may sum its products in other parts (its tiles
    then have the GPU to themselves): fp32 sums of vocab terms apart, rounded once each."""
    for n in (40, 700):
        vocab = 1111
        g, x, w, dloss = operands(n, 256, vocab, torch.float16)
        labels = torch.randint(vocab, (n,), generator=g, device="cuda")
        _, lse = training.cross_entropy_forward(x, w, labels)
        dx, dw = training.cross_entropy_backward(x, w, labels, lse, dloss)
        none, dw1 = training.cross_entropy_backward(x, w, labels, lse, dloss, want_dx=False)
        assert none is None and torch.equal(dw1, dw)
        dx1, none = training.cross_entropy_backward(x, w, labels, lse, dloss, want_dweight=False)
        assert none is None
        p = torch.softmax(x.double() @ w.double().t(), 1)
        p[torch.arange(n), labels] -= 1
        mag = (p * dloss.double().unsqueeze(1)).abs() @ w.double().abs()
        bound = 2 * ((vocab + 160) * 2 * ref.U32 * mag + ref.rounding(dx.double().abs() + 2.0 ** -11, torch.float16))
        assert ((dx1.double() - dx.double()).abs() <= bound).all()


def test_repeatable(training):
    g, x, w, dloss = operands(1500, 512, 5003, torch.float16)
    labels = torch.randint(5003, (1500,), generator=g, device="cuda")
    first = None
    for _ in range(3):
        losses, lse = training.cross_entropy_forward(x, w, labels)
        out = (losses, lse) + training.cross_entropy_backward(x, w, labels, lse, dloss)
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_no_rows(training):
    x = torch.empty((0, 64), dtype=torch.float16, device="cuda")
    w = torch.randn((100, 64), device="cuda").half()
    labels = torch.empty(0, dtype=torch.int64, device="cuda")
    losses, lse = training.cross_entropy_forward(x, w, labels)
    dx, dw = training.cross_entropy_backward(x, w, labels, lse, torch.empty(0, device="cuda"))
    assert losses.shape == (0,) and dx.shape == (0, 64) and dw.shape == w.shape and not dw.any()


def test_differences(training):
    """dx against central differences of the loss: states and steps on a grid of 2^-6, so
    x +- step is exact in fp16.  The loss's third derivative along the step is bounded by the
    cube of the logits' spread along it."""
    g, _, w, dloss = operands(6, 64, 300, torch.float16)
    x = (torch.randint(-64, 65, (6, 64), generator=g, device="cuda") / 64.0).half()
    step = (torch.randint(-1, 2, (6, 64), generator=g, device="cuda") / 64.0).half()
    labels = torch.randint(300, (6,), generator=g, device="cuda")
    tokens = torch.randint(300, (6, 5), generator=g, device="cuda", dtype=torch.int32)
    logits = torch.randn((6, 5), generator=g, device="cuda")
    spread = (step.double() @ w.double().t())
    third = (spread.amax(1) - spread.amin(1)) ** 3 / 6
    for forward, backward, factor in (
            (lambda t: training.cross_entropy_forward(t, w, labels),
             lambda lse: training.cross_entropy_backward(x, w, labels, lse, dloss), 1.0),
            (lambda t: training.distillation_forward(t, w, tokens, logits, temperature=2.0),
             lambda lse: training.distillation_backward(x, w, tokens, logits, lse, dloss, temperature=2.0), 0.5)):
        _, lse = forward(x)
        dx, _ = backward(lse)
        slope = (forward(x + step)[0].double() - forward(x - step)[0].double()) / 2
        predicted = (dx.double() * step.double()).sum(1)
        # The two losses' errors (their bound without gradients), and dx's 16-bit roundings (its own
        # and G's, whose products with the table are summed).
        noise = 2.0 ** -15 * 4 + third * factor
        rough = torch.finfo(torch.float16).eps * (dx.double().abs() + 2 * w.double().abs().max()) @ step.double().abs().t()
        assert ((slope * dloss.double() - predicted).abs() <= noise * dloss.double().abs()
                + rough.diagonal() * (1 + dloss.double().abs())).all()


def test_autograd_tail(training):
    """The tail as it is trained: final norm with its residual, then both losses over one
    table, whose gradients add up on the shared leaves."""
    n, d, vocab = 200, 256, 1234
    g, x, w, dloss = operands(n, d, vocab, torch.bfloat16)
    r = torch.randn((n, d), generator=g, device="cuda").to(torch.bfloat16)
    gamma, beta = torch.rand(d, generator=g, device="cuda") + 0.5, torch.randn(d, generator=g, device="cuda")
    labels = torch.randint(vocab, (n,), generator=g, device="cuda")
    tokens = torch.randint(vocab, (n, 8), generator=g, device="cuda", dtype=torch.int32)
    logits = torch.randn((n, 8), generator=g, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, gamma, beta, r, w)]
    total, states = training.layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3])
    ce = training.cross_entropy(states, leaves[4], labels)
    kd = training.distillation(states, leaves[4], tokens, logits, temperature=2.0)
    (0.8 * ce.mean() + 0.2 * kd.mean() + 0.001 * total.float().square().mean()).backward()

    # The same by the explicit calls.
    total, states, stats = training.layer_norm_forward(x, gamma, beta, residual=r)
    _, lse = training.cross_entropy_forward(states, w, labels)
    _, lse_t = training.distillation_forward(states, w, tokens, logits, temperature=2.0)
    ones = torch.ones(n, device="cuda")
    dx1, dw1 = training.cross_entropy_backward(states, w, labels, lse, ones * (0.8 / n))
    dx2, dw2 = training.distillation_backward(states, w, tokens, logits, lse_t, ones * (0.2 / n), temperature=2.0)
    bf16 = lambda t: ref.rounding(t.double().abs(), torch.bfloat16)
    grad = leaves[4].grad.double()
    assert ((grad - dw1.double() - dw2.double()).abs() <= bf16(grad) + bf16(dw1) * 0.02 + bf16(dw2) * 0.02).all()
    states_grad = (dx1.double() + dx2.double()).to(torch.bfloat16)
    dsum = (total.float() * (0.002 / total.numel())).to(torch.bfloat16)
    dx, dgamma, dbeta = training.layer_norm_backward(states_grad, total, gamma, stats, dsum=dsum)
    for leaf, expected in zip(leaves, (dx, dgamma, dbeta, dx)):
        # One 16-bit step of the states' gradient (fp32 and fp64 sums may round apart) carries to
        # a share eps of the row's gradient.
        scale = expected.double().abs().amax() * torch.finfo(torch.bfloat16).eps * 2
        assert ((leaf.grad.double() - expected.double()).abs() <= scale).all()


def test_streams_graphs_and_other_leaves(training):
    """A captured training step is replayed on new inputs while eager graphs of the same
    leaves live and another stream runs the same operators."""
    n, d, vocab = 300, 256, 2000
    g, x, w, dloss = operands(n, d, vocab, torch.float16)
    labels = torch.randint(vocab, (n,), generator=g, device="cuda")

    def step(x, stream=None):
        losses, lse = training.cross_entropy_forward(x, w, labels, stream=stream)
        return (losses, lse) + training.cross_entropy_backward(x, w, labels, lse, dloss, stream=stream)

    leaf_x, leaf_w = x.clone().requires_grad_(), w.clone().requires_grad_()
    alive = training.cross_entropy(leaf_x, leaf_w, labels).sum()  # an eager graph of the leaves
    leaf_gamma = torch.ones(d, device="cuda", requires_grad=True)
    alive_norm = training.layer_norm(x, leaf_gamma, leaf_gamma)
    step(x)
    torch.cuda.synchronize()
    static_x = leaf_x.detach()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static_x)
    # The autograd forms refuse a capture that the engine could not carry through.
    for call in (lambda: training.cross_entropy(leaf_x, leaf_w, labels),
                 lambda: training.layer_norm(static_x, torch.ones(d, device="cuda"), leaf_gamma)):
        with pytest.raises(RuntimeError, match="eager autograd graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del alive, alive_norm
    with torch.cuda.graph(second, pool=graph.pool()):
        captured_leaf = torch.autograd.grad(training.cross_entropy(leaf_x, leaf_w, labels).sum(), (leaf_x, leaf_w))
    new_x = torch.randn((n, d), generator=g, device="cuda").half()
    expected = step(new_x)
    ones = torch.ones(n, device="cuda")
    expected_leaf = training.cross_entropy_backward(new_x, w, labels, expected[1], ones)
    static_x.copy_(new_x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph.replay()
    beside = step(new_x, stream=side)
    torch.cuda.synchronize()
    for a, b, c in zip(captured, beside, expected):
        assert torch.equal(a, c) and torch.equal(b, c)
    second.replay()
    torch.cuda.synchronize()
    for a, c in zip(captured_leaf, expected_leaf):
        assert torch.equal(a, c)


def test_python_refusals(training):
    g, x, w, dloss = operands(4, 64, 100, torch.float16)
    labels = torch.zeros(4, dtype=torch.int64, device="cuda")
    tokens, logits = torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.zeros((4, 2), device="cuda")
    ce, kd = training.cross_entropy_forward, training.distillation_forward
    for call in (lambda: ce(x.float(), w, labels), lambda: ce(x, w.bfloat16(), labels), lambda: ce(x, w[:, :56], labels),
                 lambda: ce(x[:, :56], w, labels), lambda: ce(x, w, labels[:3]), lambda: ce(x, w, labels.short()),
                 lambda: ce(x, w, labels.cpu()), lambda: ce(x.cpu(), w, labels), lambda: ce(x, w[:0], labels),
                 lambda: kd(x, w, tokens.long(), logits), lambda: kd(x, w, tokens, logits.double()),
                 lambda: kd(x, w, tokens, logits[:, :1]), lambda: kd(x, w, tokens, logits, temperature=0.0),
                 lambda: kd(x, w, tokens, logits, temperature=float("nan")),
                 lambda: kd(x, w, tokens.repeat(1, 129), logits.repeat(1, 129)),
                 lambda: training.cross_entropy_backward(x, w, labels, dloss, dloss, want_dx=False, want_dweight=False),
                 lambda: training.cross_entropy_backward(x, w, labels, dloss[:3], dloss),
                 lambda: training.cross_entropy_backward(x, w, labels, dloss, dloss.double()),
                 lambda: training.layer_norm_forward(x, dloss, dloss),
                 lambda: training.layer_norm_forward(x, w[0].float(), w[0].float(), residual=x.bfloat16())):
        with pytest.raises(ValueError):
            call()
    misaligned = torch.empty(4 * 64 + 1, dtype=torch.float16, device="cuda")[1:].view(4, 64)
    with pytest.raises(training.native.NativeError):
        ce(misaligned, w, labels)
    with pytest.raises(training.native.NativeError):
        ce(x[:, :60].contiguous(), w[:, :60].contiguous(), labels)
