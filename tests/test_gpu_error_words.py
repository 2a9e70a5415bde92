"""The token and decoder error words are complete when they are read: work on streams that do
not follow the default stream is waited for."""

from __future__ import annotations

import importlib

import pytest
import torch

from conftest import PACKAGE

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def training(cuda):
    return importlib.import_module(PACKAGE + ".training")


@pytest.fixture
def busy(cuda):
    """A side stream with some 30 ms of work queued (forty 8192-wide products), and nothing else."""
    a = torch.randn((8192, 8192), device=cuda, dtype=torch.bfloat16)
    out = torch.empty_like(a)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(40):
            torch.mm(a, a, out=out)
    yield side
    torch.cuda.synchronize()


@pytest.mark.parametrize("device", [None, 0, "cuda:0"])
@pytest.mark.parametrize("teacher", [False, True])
def test_token_error_waits_for_side_streams(training, request, teacher, device):
    x = torch.randn((10, 64), device="cuda").half()
    w = torch.randn((200, 64), device="cuda").half()
    bad = torch.full((10, 1), 200, dtype=torch.int32, device="cuda")
    logits = torch.zeros((10, 1), device="cuda")
    labels = bad.view(-1)
    training.cross_entropy_forward(x, w, labels), training.distillation_forward(x, w, bad, logits)  # loads the kernels
    torch.cuda.synchronize()
    assert training.token_error(device) == 1 and training.token_error(device) == 0
    side = request.getfixturevalue("busy")
    if teacher:
        training.distillation_forward(x, w, bad, logits, stream=side)
    else:
        training.cross_entropy_forward(x, w, labels, stream=side)
    assert training.token_error(device) == 1
    assert training.token_error(device) == 0


def test_decoder_error_waits_for_side_streams(cuda, fp8, request):
    table, positions = torch.zeros((100, 64), device=cuda).half(), torch.zeros((10, 64), device=cuda).half()
    bad, lengths = torch.tensor([100], dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    fp8.decoder_embed(bad, lengths, table, positions)
    torch.cuda.synchronize()
    assert fp8.decoder_error() == 1 and fp8.decoder_error() == 0
    side = request.getfixturevalue("busy")
    fp8.decoder_embed(bad, lengths, table, positions, stream=side)
    assert fp8.decoder_error() == 1
    assert fp8.decoder_error() == 0
