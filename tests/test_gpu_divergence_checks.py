"""Decoder.divergence: a teacher's tokens of 64 bits, and refusals that come before the decode."""

from __future__ import annotations

import importlib

import pytest
import torch

from conftest import PACKAGE

pytestmark = pytest.mark.gpu

STREAMS, LENGTH = 2, 3


@pytest.fixture(scope="module")
def plan(cuda):
    dec = importlib.import_module(PACKAGE + ".decoder")
    config = dec.DecoderConfig(layers=1)
    weights = dec.DecoderWeights.from_checkpoint(dec.add_synthetic_decoder({}, config, seed=3, device=cuda), config)
    g = torch.Generator(device=cuda).manual_seed(4)
    cross_kv = torch.randn((2, STREAMS, config.heads, config.audio_positions, 64), generator=g, device=cuda).half()
    return dec.Decoder(weights, dec.calibrate(weights, cross_kv, STREAMS, steps=2), cross_kv, STREAMS)


@pytest.fixture
def transcripts(plan):
    return torch.tensor([[7, 8, 9], [10, 11, -100]], dtype=torch.int32, device="cuda")


def test_tokens_of_64_bits(plan, transcripts):
    """topk's indices are taken as they are; one past 32 bits is outside the vocabulary, whatever
    its low 32 bits say."""
    training = importlib.import_module(PACKAGE + ".training")
    training.token_error()
    g = torch.Generator(device="cuda").manual_seed(5)
    tokens = torch.randint(plan.config.vocab, (STREAMS, LENGTH, 4), generator=g, device="cuda")
    logits = torch.randn((STREAMS, LENGTH, 4), generator=g, device="cuda")
    narrow = plan.divergence(transcripts, tokens.int(), logits)
    assert torch.equal(plan.divergence(transcripts, tokens, logits), narrow) and training.token_error() == 0
    left_out = tokens.int()
    left_out[0, 1, 2] = -1
    for bad in (2 ** 32 + 5, 2 ** 31, -2 ** 40):
        tokens[0, 1, 2] = bad
        assert torch.equal(plan.divergence(transcripts, tokens, logits), plan.divergence(transcripts, left_out, logits))
        assert training.token_error() == (1 if bad > 0 else 0)


def test_refusals_leave_the_plan(plan, transcripts):
    """A call that is refused has decoded nothing: the caches stay as they were."""
    tokens = torch.zeros((STREAMS, LENGTH, 4), dtype=torch.int32, device="cuda")
    logits = torch.zeros((STREAMS, LENGTH, 4), device="cuda")
    plan.reset()
    for call in (lambda: plan.divergence(transcripts, tokens, logits.double()),
                 lambda: plan.divergence(transcripts, tokens, logits.cpu()),
                 lambda: plan.divergence(transcripts, tokens.cpu(), logits),
                 lambda: plan.divergence(transcripts.long(), tokens, logits),
                 lambda: plan.divergence(transcripts.cpu(), tokens, logits),
                 lambda: plan.divergence(transcripts, tokens[..., :0], logits[..., :0]),
                 lambda: plan.divergence(transcripts, tokens.repeat(1, 1, 65), logits.repeat(1, 1, 65)),
                 lambda: plan.divergence(transcripts, tokens, logits, temperature=0.0),
                 lambda: plan.divergence(transcripts, tokens, logits, temperature=float("nan"))):
        with pytest.raises(ValueError):
            call()
        assert not plan.lengths.any()
