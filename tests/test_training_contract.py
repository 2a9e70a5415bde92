"""The scoring and training operators' C ABI and Python checks that need no GPU: bad calls are
refused before a device is touched."""

from __future__ import annotations

import ctypes
import importlib

import pytest
import torch

from conftest import PACKAGE


@pytest.fixture(scope="module")
def lib(native):
    return native.library()


@pytest.fixture(scope="module")
def training(lffw):
    return importlib.import_module(PACKAGE + ".training")


def fill(a, fields, change):
    a.struct_size = ctypes.sizeof(type(a))
    for key, value in {**fields, **change}.items():
        setattr(a, key, value)
    return ctypes.byref(a)


NORM = dict(rows=16, cols=1280, dtype=1, x=0x10000, residual=0x20000, sum_out=0x30000, gamma=0x40000, beta=0x50000,
            epsilon=1e-5, y=0x60000, stats=0x70000)


@pytest.mark.parametrize("change", [
    {"rows": 0}, {"rows": -1}, {"rows": 2**31}, {"cols": 0}, {"cols": 4}, {"cols": 1284}, {"cols": 4104},
    {"dtype": 0}, {"dtype": 2}, {"dtype": 6}, {"x": None}, {"gamma": None}, {"beta": None}, {"y": None},
    {"stats": None}, {"residual": None}, {"sum_out": None}, {"x": 0x10008}, {"residual": 0x20002},
    {"sum_out": 0x30004}, {"gamma": 0x40004}, {"y": 0x60008}, {"stats": 0x70002}, {"epsilon": -1.0},
    {"epsilon": float("nan")}, {"epsilon": float("inf")},
])
def test_layer_norm_train_refusals(native, lib, change):
    assert lib.lffw_layer_norm_train(fill(native.LayerNormTrainArgs(), NORM, change), None) == native.INVALID_ARGUMENT


NORM_GRAD = dict(rows=2000, cols=1280, dtype=7, dy=0x10000, s=0x20000, gamma=0x30000, stats=0x40000, dsum=0x50000,
                 dx=0x60000, dgamma=0x70000, dbeta=0x80000, workspace=0x90000, workspace_bytes=1 << 30)


@pytest.mark.parametrize("change", [
    {"rows": 0}, {"cols": 12}, {"dtype": 3}, {"dy": None}, {"s": None}, {"gamma": None}, {"stats": None},
    {"dgamma": None}, {"dbeta": None}, {"dx": None, "dgamma": None, "dbeta": None}, {"dy": 0x10008}, {"s": 0x20002},
    {"dsum": 0x50004}, {"dx": 0x60008}, {"dgamma": 0x70001}, {"workspace": 0x90008},
])
def test_layer_norm_grad_refusals(native, lib, change):
    assert lib.lffw_layer_norm_grad(fill(native.LayerNormGradArgs(), NORM_GRAD, change), None) == \
        native.INVALID_ARGUMENT


LOSS = dict(rows=100, width=1280, vocab=51866, dtype=1, x=0x10000, weight=0x20000, labels=0x30000, label_bytes=8,
            ignore_index=-100, temperature=1.0, losses=0x40000, lse=0x50000, dloss=0x60000, dx=0x70000,
            dweight=0x80000, workspace=0x100000, workspace_bytes=1 << 40)
TEACHER = dict(LOSS, labels=None, teacher_entries=5, teacher_dtype=0, teacher_tokens=0x30000, teacher_logits=0x38000)
SHARED = [
    (LOSS, {"rows": 0}), (LOSS, {"rows": 2**22 + 1}), (LOSS, {"width": 4}), (LOSS, {"width": 1284}),
    (LOSS, {"width": 2**16 + 8}), (LOSS, {"vocab": 0}), (LOSS, {"vocab": 2**22 + 1}), (LOSS, {"dtype": 0}),
    (LOSS, {"x": None}), (LOSS, {"weight": None}), (LOSS, {"x": 0x10002}), (LOSS, {"weight": 0x20008}),
    (LOSS, {"labels": None}), (LOSS, {"labels": 0x30004}), (LOSS, {"label_bytes": 2}), (LOSS, {"temperature": 2.0}),
    (LOSS, {"lse": None}), (LOSS, {"lse": 0x50002}), (LOSS, {"teacher_entries": -1}),
    (TEACHER, {"teacher_entries": 257}), (TEACHER, {"teacher_tokens": None}), (TEACHER, {"teacher_tokens": 0x30002}),
    (TEACHER, {"teacher_logits": None}), (TEACHER, {"teacher_logits": 0x38002}), (TEACHER, {"teacher_dtype": 2}),
    (TEACHER, {"temperature": 0.0}), (TEACHER, {"temperature": -1.0}), (TEACHER, {"temperature": float("nan")}),
    (TEACHER, {"temperature": float("inf")}), (TEACHER, {"temperature": 2.0**6.5}), (TEACHER, {"temperature": 2.0**-6.5}),
]


@pytest.mark.parametrize("base,change", SHARED)
def test_vocab_loss_refusals(native, lib, base, change):
    for call in (lib.lffw_vocab_loss, lib.lffw_vocab_loss_grad):
        assert call(fill(native.VocabLossArgs(), base, change), None) == native.INVALID_ARGUMENT
    if "lse" not in change:
        for grad in (0, 1):
            assert lib.lffw_vocab_loss_workspace(fill(native.VocabLossArgs(), base, change), grad) == -1


@pytest.mark.parametrize("change", [{"losses": None}, {"losses": 0x40002}])
def test_forward_refusals(native, lib, change):
    assert lib.lffw_vocab_loss(fill(native.VocabLossArgs(), LOSS, change), None) == native.INVALID_ARGUMENT


@pytest.mark.parametrize("change", [{"dloss": None}, {"dloss": 0x60002}, {"dx": 0x70008}, {"dweight": 0x80004},
                                    {"dx": None, "dweight": None}])
def test_backward_refusals(native, lib, change):
    assert lib.lffw_vocab_loss_grad(fill(native.VocabLossArgs(), LOSS, change), None) == native.INVALID_ARGUMENT


def test_abi_mismatch_and_null(native, lib):
    for kind, calls in ((native.LayerNormTrainArgs, (lib.lffw_layer_norm_train,)),
                        (native.LayerNormGradArgs, (lib.lffw_layer_norm_grad,)),
                        (native.VocabLossArgs, (lib.lffw_vocab_loss, lib.lffw_vocab_loss_grad))):
        a = kind()
        a.struct_size = 8
        for call in calls:
            assert call(ctypes.byref(a), None) == native.ABI_MISMATCH
            assert call(None, None) == native.INVALID_ARGUMENT
    assert lib.lffw_vocab_loss_workspace(None, 0) == -1
    assert lib.lffw_vocab_loss_error(None) == native.INVALID_ARGUMENT


def test_workspace_sizes(native, lib):
    """The workspace follows the shape: a piece of dz (512 MB at most, whatever the rows), never
    the logits; few LayerNorm rows need none."""
    size = lambda grad, base=LOSS, **change: lib.lffw_vocab_loss_workspace(
        fill(native.VocabLossArgs(), base, change), grad)
    assert 0 < size(0) < 1 << 20
    for rows in (1, 100, 5000, 14336, 200000):
        states = rows * 1280
        assert size(1, rows=rows) <= (512 << 20) + 6 * states + 20 * rows + (16 * 1280 * 148 * 128) + 4096
    assert size(1, dx=None) < size(1)
    assert size(0, base=TEACHER) > size(0)
    assert lib.lffw_layer_norm_grad_workspace(20, 1280) == 0
    assert 0 < lib.lffw_layer_norm_grad_workspace(100000, 1280) <= 4 << 20
    assert lib.lffw_layer_norm_grad_workspace(0, 1280) == -1 and lib.lffw_layer_norm_grad_workspace(4, 12) == -1


def test_python_refusals_on_the_host(training):
    x, w = torch.zeros((4, 64), dtype=torch.float16), torch.zeros((100, 64), dtype=torch.float16)
    gamma = torch.ones(64)
    labels = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: training.layer_norm_forward(x, gamma, gamma),
                 lambda: training.layer_norm_backward(x, x, gamma, torch.zeros((2, 4))),
                 lambda: training.cross_entropy_forward(x, w, labels),
                 lambda: training.distillation_forward(x, w, labels.int().view(4, 1), gamma[:4].view(4, 1)),
                 lambda: training.cross_entropy(x, w, labels),
                 lambda: training.layer_norm(x.float(), gamma, gamma)):
        with pytest.raises(ValueError):
            call()
