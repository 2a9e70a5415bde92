"""Captures of the autograd forms over leaves that reach them through a cast: refused while an
eager graph of the same leaves lives, carried through once it is gone."""

from __future__ import annotations

import gc
import importlib

import pytest
import torch

from conftest import PACKAGE

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def training(cuda):
    return importlib.import_module(PACKAGE + ".training")


def test_cast_leaves(training):
    n, d, vocab = 200, 128, 1000
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((n, d), generator=g, device="cuda").half()
    labels = torch.randint(vocab, (n,), generator=g, device="cuda")
    masters = [(torch.randn((vocab, d), generator=g, device="cuda") * 0.1).requires_grad_(),
               torch.randn(d, generator=g, device="cuda").half().requires_grad_(),
               torch.randn(2 * d, generator=g, device="cuda").requires_grad_()]

    def loss():
        table, gamma, beta = masters
        _, y = training.layer_norm(x, gamma.float(), beta[:d].contiguous())
        return training.cross_entropy(y, table.half(), labels).sum()

    expected = torch.autograd.grad(loss(), masters)
    torch.cuda.synchronize()
    calls = (lambda: training.cross_entropy(x, masters[0].half(), labels),
             lambda: training.distillation(x, masters[0].half().view(vocab, d), labels.int().unsqueeze(1),
                                           x[:, :1].contiguous()),
             lambda: training.layer_norm(x, masters[1].float(), torch.zeros(d, device="cuda")),
             lambda: training.layer_norm(x, torch.ones(d, device="cuda"), masters[2][:d].contiguous()))
    alive = loss()
    for call in calls:
        with pytest.raises(RuntimeError, match="eager autograd graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del alive
    gc.collect()  # what the refusals' tracebacks held
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = torch.autograd.grad(loss(), masters)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, expected):
        assert torch.equal(a, b)


def test_inputs_without_one_leaf_are_left_alone(training):
    """A sum of two leaves, a constant and a long chain are nobody's cast."""
    a, b = (torch.randn((4, 8), device="cuda", requires_grad=True) for _ in range(2))
    assert training._guard_capture(a + b, a.detach(), None) == []
    chain = a
    for _ in range(training._GUARDED_STEPS + 1):
        chain = chain.view(4, 8) * 1.0
    assert training._guard_capture(chain) == []
    assert len(training._guard_capture(a.half(), b)) == 2
    with torch.no_grad():
        assert training._guard_capture(a, b) == []
