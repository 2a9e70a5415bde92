"""Inputs of the scoring and training calls that are let go of while another stream still has to
read them: their memory is not handed out before it has."""

from __future__ import annotations

import importlib

import pytest
import torch

from conftest import PACKAGE

pytestmark = pytest.mark.gpu

N, D, VOCAB, K = 2000, 256, 3000, 4


@pytest.fixture(scope="module")
def training(cuda):
    return importlib.import_module(PACKAGE + ".training")


@pytest.fixture(scope="module")
def inputs(cuda):
    g = torch.Generator(device=cuda).manual_seed(12)
    normal = lambda *shape: torch.randn(shape, generator=g, device=cuda)
    return {"x": normal(N, D).half(), "r": normal(N, D).half(), "gamma": normal(D), "beta": normal(D),
            "dy": normal(N, D).half(), "dsum": normal(N, D).half(), "w": (normal(VOCAB, D) * 0.1).half(),
            "labels": torch.randint(VOCAB, (N,), generator=g, device=cuda), "dloss": normal(N),
            "tokens": torch.randint(VOCAB, (N, K), generator=g, device=cuda, dtype=torch.int32), "logits": normal(N, K)}


def calls(training, fixed):
    """name -> (what the call reads, the call)."""
    total, _, stats = training.layer_norm_forward(fixed["x"], fixed["gamma"], fixed["beta"], residual=fixed["r"])
    lse = training.cross_entropy_forward(fixed["x"], fixed["w"], fixed["labels"])[1]
    t_lse = training.distillation_forward(fixed["x"], fixed["w"], fixed["tokens"], fixed["logits"])[1]
    torch.cuda.synchronize()
    t = training
    return {
        "norm": (("x", "gamma", "beta", "r"), {},
                 lambda s, a: t.layer_norm_forward(a["x"], a["gamma"], a["beta"], residual=a["r"], stream=s)),
        "norm gradients": (("dy", "gamma", "dsum"), {"total": total, "stats": stats},
                           lambda s, a: t.layer_norm_backward(a["dy"], a["total"], a["gamma"], a["stats"],
                                                              dsum=a["dsum"], stream=s)),
        "loss": (("x", "w", "labels"), {}, lambda s, a: t.cross_entropy_forward(a["x"], a["w"], a["labels"], stream=s)),
        "loss gradients": (("x", "w", "labels", "dloss"), {"lse": lse},
                           lambda s, a: t.cross_entropy_backward(a["x"], a["w"], a["labels"], a["lse"], a["dloss"],
                                                                 stream=s)),
        "distillation": (("x", "w", "tokens", "logits"), {},
                         lambda s, a: t.distillation_forward(a["x"], a["w"], a["tokens"], a["logits"], stream=s)),
        "distillation gradients": (("x", "w", "tokens", "logits", "dloss"), {"lse": t_lse},
                                   lambda s, a: t.distillation_backward(a["x"], a["w"], a["tokens"], a["logits"],
                                                                        a["lse"], a["dloss"], stream=s)),
    }


@pytest.mark.parametrize("name", ["norm", "norm gradients", "loss", "loss gradients", "distillation",
                                  "distillation gradients"])
def test_inputs_that_are_let_go_of(training, inputs, name):
    reads, made, call = calls(training, inputs)[name]
    fixed = {**{k: inputs[k] for k in reads}, **made}
    expected = [t for t in call(None, fixed) if t is not None]
    block = torch.empty((8192, 8192), device="cuda", dtype=torch.bfloat16).normal_()
    out = torch.empty_like(block)
    side = torch.cuda.Stream()
    # The call's memory is there beforehand: an allocation that has to give cached memory back waits
    # for every stream.
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    call(side, fixed)
    args = {k: v.clone() for k, v in fixed.items()}
    taken = {k: (v.data_ptr(), v.numel() * v.element_size()) for k, v in args.items()}
    torch.cuda.synchronize()
    with torch.cuda.stream(side):  # some 70 ms of work before the call
        for _ in range(100):
            torch.mm(block, block, out=out)
    got = [t for t in call(side, args) if t is not None]
    shapes = [v.shape for v in args.values()], [v.dtype for v in args.values()]
    args.clear()
    # What the caller's stream is now given must be other memory: the side stream has not read the inputs.
    fresh = [torch.empty(shape, dtype=dtype, device="cuda") for shape, dtype in zip(*shapes)]
    assert not side.query(), "the side stream was to be busy"
    for t in fresh:
        begin, end = t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()
        assert all(end <= at or begin >= at + size for at, size in taken.values())
    torch.cuda.synchronize()
    for a, b in zip(got, expected):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["handle", "object", "current"])
def test_handles_record_nothing(training, inputs, kind):
    """A cudaStream_t is its owner's, who may destroy it once its work has run: a tensor that
    outlives it must not know it.  (A recorded tensor's memory stays active when it is let go of.)"""
    owner = torch.cuda.Stream()
    handle = owner.cuda_stream
    stream = handle if kind == "handle" else torch.cuda.ExternalStream(handle)
    if kind == "current":
        with torch.cuda.stream(stream):
            stream = torch.cuda.current_stream()
    active = lambda: torch.cuda.memory_stats()["active_bytes.all.current"]
    x = inputs["x"].clone()
    torch.cuda.synchronize()
    y = training.layer_norm_forward(x, inputs["gamma"], inputs["beta"], stream=stream)[1]
    torch.cuda.synchronize()
    before = active()
    size = x.numel() * x.element_size()
    del x
    assert before - active() >= size
    x = inputs["x"].clone()
    torch.cuda.synchronize()
    training.layer_norm_forward(x, inputs["gamma"], inputs["beta"], stream=owner)
    torch.cuda.synchronize()
    before = active()
    del x
    assert before == active()
    assert torch.equal(y, training.layer_norm_forward(inputs["x"], inputs["gamma"], inputs["beta"])[1])
