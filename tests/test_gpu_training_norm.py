"""LayerNorm forward with statistics and its gradients against 64 bits (bounds in
training_reference), over odd row counts, every width rule, both types, with and without the
residual stream."""

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
    return importlib.import_module(PACKAGE + ".training")


def make(rows, cols, dtype, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 131 + cols)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    x = (normal(rows, cols) * 2 + 0.5).to(dtype)
    r = normal(rows, cols).to(dtype) if residual else None
    return {"x": x, "residual": r, "gamma": 1 + 0.2 * normal(cols), "beta": 0.3 * normal(cols),
            "dy": normal(rows, cols).to(dtype), "dsum": normal(rows, cols).to(dtype) if residual else None}


def check(training, s, eps=1e-5):
    total, y, stats = training.layer_norm_forward(s["x"], s["gamma"], s["beta"], eps, residual=s["residual"])
    dx, dgamma, dbeta = training.layer_norm_backward(s["dy"], total, s["gamma"], stats, dsum=s["dsum"])
    e_total, e_y, mean, rstd = ref.layer_norm(s["x"], s["gamma"], s["beta"], eps, s["residual"])
    assert torch.equal(total, e_total)
    assert ref.worst(y, e_y, ref.layer_norm_bound(total, s["gamma"], s["beta"], e_y, mean, rstd)) <= 1
    e_dx, e_dg, e_db = ref.layer_norm_grads(s["dy"], total, s["gamma"], mean, rstd, s["dsum"])
    b_dx, b_dg, b_db = ref.layer_norm_grad_bounds(s["dy"], total, s["gamma"], mean, rstd, e_dx, s["dsum"])
    assert ref.worst(dx, e_dx, b_dx) <= 1
    assert ref.worst(dgamma, e_dg, b_dg) <= 1
    assert ref.worst(dbeta, e_db, b_db) <= 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 8), (2, 264), (3, 256), (20, 1280), (447, 384), (1001, 512), (333, 1000),
                                       (7, 4096), (2500, 768), (6001, 1280), (700, 2560), (149, 4088), (1001, 4096),
                                       (5003, 8), (9001, 256), (4444, 520)])
def test_against_64_bits(training, rows, cols, dtype, residual):
    check(training, make(rows, cols, dtype, residual))


@pytest.mark.parametrize("rows", [1, 2, 3, 591, 592, 593, 1183, 1184, 1185, 2367, 2368, 2369])
def test_row_counts_around_a_full_step(training, rows):
    """Around 148 SMs x 4 groups x 1, 2 and 4 rows, where the rows per step and the tail change."""
    check(training, make(rows, 1280, torch.float16, True, seed=3))


def test_offsets_past_32_bits(training):
    """2^31 elements and more: the last rows against 64 bits, the column sums against the sum of
    two halves of the rows."""
    rows, cols = (1 << 31) // 1280 + 1000, 1280
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((rows, cols), generator=g, device="cuda", dtype=torch.bfloat16)
    dy = torch.randn((rows, cols), generator=g, device="cuda", dtype=torch.bfloat16)
    gamma, beta = torch.rand(cols, generator=g, device="cuda") + 0.5, torch.randn(cols, generator=g, device="cuda")
    total, y, stats = training.layer_norm_forward(x, gamma, beta)
    dx, dgamma, dbeta = training.layer_norm_backward(dy, total, gamma, stats)
    last = slice(rows - 700, rows)
    _, e_y, mean, rstd = ref.layer_norm(x[last], gamma, beta, 1e-5)
    assert ref.worst(y[last], e_y, ref.layer_norm_bound(x[last], gamma, beta, e_y, mean, rstd)) <= 1
    e_dx, _, _ = ref.layer_norm_grads(dy[last], x[last], gamma, mean, rstd)
    b_dx, _, _ = ref.layer_norm_grad_bounds(dy[last], x[last], gamma, mean, rstd, e_dx)
    assert ref.worst(dx[last], e_dx, b_dx) <= 1
    halves = [training.layer_norm_backward(dy[part], x[part], gamma, stats[:, part].contiguous(), want_dx=False)
              for part in (slice(0, rows // 2), slice(rows // 2, rows))]
    # Sums of up to `rows` terms of size about 1 (each at most 32), in two orders.
    for whole, first, second in ((dgamma, halves[0][1], halves[1][1]), (dbeta, halves[0][2], halves[1][2])):
        assert ((whole - first - second).abs() <= 2 * rows * ref.U32 * 3 * rows ** 0.5).all()


def test_rows_behind_the_last_are_left(training):
    s = make(5, 1280, torch.bfloat16, True)
    keep = torch.full((9, 1280), 7.0, dtype=torch.bfloat16, device="cuda")
    native, fp8 = training.native, importlib.import_module(PACKAGE + ".fp8")
    import ctypes

    total, y = keep.clone(), keep.clone()
    stats = torch.full((2, 5), -1.0, device="cuda")
    a = native.LayerNormTrainArgs(ctypes.sizeof(native.LayerNormTrainArgs), 5, 1280, native.DT_BF16,
                                  s["x"].data_ptr(), s["residual"].data_ptr(), total.data_ptr(), s["gamma"].data_ptr(),
                                  s["beta"].data_ptr(), 1e-5, y.data_ptr(), stats.data_ptr())
    native.check(native.library().lffw_layer_norm_train(ctypes.byref(a), fp8._stream(None)), "lffw_layer_norm_train")
    assert torch.equal(total[5:], keep[5:]) and torch.equal(y[5:], keep[5:])
    expected = training.layer_norm_forward(s["x"], s["gamma"], s["beta"], residual=s["residual"])
    assert torch.equal(total[:5], expected[0]) and torch.equal(y[:5], expected[1]) and torch.equal(stats, expected[2])


def test_in_place_sum_and_gradient(training):
    """sum_out may be the residual, dx may be dsum: the residual stream updated in place."""
    import ctypes

    s = make(777, 1280, torch.float16, True)
    total, y, stats = training.layer_norm_forward(s["x"], s["gamma"], s["beta"], residual=s["residual"])
    dx, _, _ = training.layer_norm_backward(s["dy"], total, s["gamma"], stats, dsum=s["dsum"])
    native, fp8 = training.native, importlib.import_module(PACKAGE + ".fp8")
    stream_rows, y2, stats2 = s["residual"].clone(), torch.empty_like(y), torch.empty_like(stats)
    a = native.LayerNormTrainArgs(ctypes.sizeof(native.LayerNormTrainArgs), 777, 1280, native.DT_HALF,
                                  s["x"].data_ptr(), stream_rows.data_ptr(), stream_rows.data_ptr(),
                                  s["gamma"].data_ptr(), s["beta"].data_ptr(), 1e-5, y2.data_ptr(), stats2.data_ptr())
    native.check(native.library().lffw_layer_norm_train(ctypes.byref(a), fp8._stream(None)), "lffw_layer_norm_train")
    assert torch.equal(stream_rows, total) and torch.equal(y2, y)
    grad = s["dsum"].clone()
    b = native.LayerNormGradArgs(ctypes.sizeof(native.LayerNormGradArgs), 777, 1280, native.DT_HALF,
                                 s["dy"].data_ptr(), total.data_ptr(), s["gamma"].data_ptr(), stats.data_ptr(),
                                 grad.data_ptr(), grad.data_ptr(), None, None, None, 0)
    native.check(native.library().lffw_layer_norm_grad(ctypes.byref(b), fp8._stream(None)), "lffw_layer_norm_grad")
    assert torch.equal(grad, dx)


def test_subsets_of_the_gradients_are_the_same_bits(training):
    s = make(1500, 1280, torch.bfloat16, True)
    total, _, stats = training.layer_norm_forward(s["x"], s["gamma"], s["beta"], residual=s["residual"])
    dx, dgamma, dbeta = training.layer_norm_backward(s["dy"], total, s["gamma"], stats, dsum=s["dsum"])
    only_x = training.layer_norm_backward(s["dy"], total, s["gamma"], stats, dsum=s["dsum"], want_params=False)
    only_p = training.layer_norm_backward(s["dy"], total, s["gamma"], stats, want_dx=False)
    assert torch.equal(only_x[0], dx) and only_x[1] is None and only_x[2] is None
    assert only_p[0] is None and torch.equal(only_p[1], dgamma) and torch.equal(only_p[2], dbeta)


def test_non_finite_rows_stay_their_own(training):
    s = make(100, 1280, torch.float16, False)
    clean = training.layer_norm_forward(s["x"], s["gamma"], s["beta"])[1]
    bad = s["x"].clone()
    bad[17, 5] = float("nan")
    bad[41, 9] = float("inf")
    y = training.layer_norm_forward(bad, s["gamma"], s["beta"])[1]
    rows = torch.ones(100, dtype=torch.bool)
    rows[[17, 41]] = False
    assert torch.equal(y[rows], clean[rows])
    assert torch.isnan(y[17]).all() and torch.isnan(y[41]).all()


def test_constant_rows(training):
    """Zero variance: rstd is eps^-1/2 and y is beta."""
    x = torch.full((33, 384), 3.0, dtype=torch.bfloat16, device="cuda")
    gamma, beta = torch.randn(384, device="cuda"), torch.randn(384, device="cuda")
    total, y, stats = training.layer_norm_forward(x, gamma, beta, 1e-5)
    assert torch.equal(y, beta.to(torch.bfloat16).expand(33, 384))
    torch.testing.assert_close(stats[1], torch.full((33,), 1e-5 ** -0.5, device="cuda"), rtol=4 * ref.U32, atol=0)


def test_no_rows(training):
    x = torch.empty((0, 64), dtype=torch.float16, device="cuda")
    gamma, beta = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    total, y, stats = training.layer_norm_forward(x, gamma, beta)
    assert y.shape == (0, 64) and stats.shape == (2, 0)
    dx, dgamma, dbeta = training.layer_norm_backward(x, total, gamma, stats)
    assert dx.shape == (0, 64) and not dgamma.any() and not dbeta.any()


def test_differences(training):
    """The gradient against central differences of the forward in its own type: rows and
    steps lie on a grid of 2^-6, so x +- step is exact; what is left is the third-order term,
    which falls with the square of the step: halving it must quarter the gap or reach the
    rounding of y, (cols terms of) half a step of fp16 each."""
    cols = 64
    g = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.randint(-128, 128, (4, cols), generator=g, device="cuda") / 64.0).half()
    gamma, beta = torch.rand(cols, generator=g, device="cuda") + 0.5, torch.randn(cols, generator=g, device="cuda")
    dy = torch.randint(-8, 9, (4, cols), generator=g, device="cuda").half() / 8
    step = torch.randint(-1, 2, (4, cols), generator=g, device="cuda").half() / 64
    total, y, stats = training.layer_norm_forward(x, gamma, beta)
    dx, _, _ = training.layer_norm_backward(dy, total, gamma, stats)
    value = lambda t: (training.layer_norm_forward(t, gamma, beta)[1].double() * dy.double()).sum(1)
    slope = (value(x + step) - value(x - step)) / 2
    predicted = (dx.double() * step.double()).sum(1)
    # Rounding of the two y's and of dx; the third-order term from the 64-bit function.
    exact = lambda t: (ref.layer_norm(t, gamma, beta, 1e-5)[1] * dy.double()).sum(1)
    third = (exact(x + step) - exact(x - step)) / 2
    _, e_y, mean, rstd = ref.layer_norm(x, gamma, beta, 1e-5)
    e_dx = ref.layer_norm_grads(dy, total, gamma, mean, rstd)[0]
    third = (third - (e_dx * step.double()).sum(1)).abs()
    noise = (ref.rounding(e_y.abs() + 0.25, torch.float16) * dy.double().abs()).sum(1) \
        + (ref.rounding(e_dx.abs(), torch.float16) * step.double().abs()).sum(1) * 2 + 1e-5
    assert ((slope - predicted).abs() <= third + noise).all()


def test_autograd(training):
    s = make(130, 1280, torch.float16, True)
    leaves = [s[k].clone().requires_grad_() for k in ("x", "gamma", "beta", "residual")]
    total, y = training.layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3])
    torch.autograd.backward([y, total], [s["dy"], s["dsum"]])
    t, _, stats = training.layer_norm_forward(s["x"], s["gamma"], s["beta"], residual=s["residual"])
    dx, dgamma, dbeta = training.layer_norm_backward(s["dy"], t, s["gamma"], stats, dsum=s["dsum"])
    for leaf, expected in zip(leaves, (dx, dgamma, dbeta, dx)):
        assert torch.equal(leaf.grad, expected)
    # Only one of the outputs used, and an expanded (stride 0) gradient.
    x = s["x"].clone().requires_grad_()
    same, y = training.layer_norm(x, s["gamma"], s["beta"])
    assert same is x
    y.sum().backward()
    t, _, stats = training.layer_norm_forward(s["x"], s["gamma"], s["beta"])
    ones = torch.ones_like(s["x"])
    assert torch.equal(x.grad, training.layer_norm_backward(ones, t, s["gamma"], stats, want_params=False)[0])
    r = s["residual"].clone().requires_grad_()
    total, _ = training.layer_norm(s["x"], s["gamma"], s["beta"], residual=r)
    total.sum().backward()
    assert torch.equal(r.grad, ones)


def test_graph_and_streams(training):
    """A captured step replayed on new inputs, beside an eager call on a second stream."""
    s, other = make(512, 768, torch.bfloat16, True), make(512, 768, torch.bfloat16, True, seed=9)

    def step(s, stream=None):
        total, y, stats = training.layer_norm_forward(s["x"], s["gamma"], s["beta"], residual=s["residual"],
                                                      stream=stream)
        return (total, y) + training.layer_norm_backward(s["dy"], total, s["gamma"], stats, dsum=s["dsum"],
                                                         stream=stream)

    expected = step(other)
    step(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(s)
    for k, v in s.items():
        v.copy_(other[k])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph.replay()
    beside = step(other, stream=side)
    torch.cuda.synchronize()
    for a, b, c in zip(captured, beside, expected):
        assert torch.equal(a, c) and torch.equal(b, c)
