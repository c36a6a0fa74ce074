"""Calls of the token scores whose arguments do not fit each other, refused
before a kernel reads them."""

import contextlib

import pytest
import torch

from bdm_amd import ops


def tokens(*shape):
    return torch.zeros(shape, dtype=torch.int64)


@pytest.fixture
def no_device(monkeypatch):
    """The checks behind the device's, on the CPU; what would have been launched is noted."""
    launched = []
    monkeypatch.setattr(ops, '_require_gpu', lambda *t: torch.device('cpu'))
    monkeypatch.setattr(ops, '_on', lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, 'token_gradients', lambda *a: launched.append(a))
    return launched


def gradient(**options):
    ops.token_gradient(torch.zeros(3, 8), tokens(3), torch.zeros(3, 2), **options)


@pytest.mark.parametrize('top_tokens,top', [
    (tokens(1, 2), torch.zeros(1, 2)),          # one row's alternatives for three rows
    (tokens(2), torch.zeros(2)),
    (tokens(3, 2, 1), torch.zeros(3, 2, 1)),
    (tokens(3, 2).int(), torch.zeros(3, 2)),    # half the bytes of a row of int64
    (torch.zeros(3, 2), torch.zeros(3, 2)),
    (tokens(3, 2), torch.zeros(3, 1)),
])
def test_token_gradient_checks_the_alternatives(no_device, top_tokens, top):
    """The kernel reads the alternatives of every row of the logits."""
    with pytest.raises(ValueError):
        gradient(top_tokens=top_tokens, grad_top_log_probs=top)
    assert not no_device
    gradient(top_tokens=tokens(3, 2), grad_top_log_probs=torch.zeros(3, 2))
    assert no_device


def test_token_gradient_of_a_loss_and_log_probs(no_device):
    """The loss' gradient takes the place of the log-probabilities': both at once are refused, none is dropped."""
    scalar = torch.zeros(())
    with pytest.raises(ValueError, match='loss'):
        gradient(grad_loss=scalar, inverse_count=scalar, grad_log_probs=torch.zeros(3))
    assert not no_device
    gradient(grad_loss=scalar, inverse_count=scalar)
    gradient(grad_log_probs=torch.zeros(3))
    assert len(no_device) == 2


@pytest.mark.parametrize('vocab', [2 ** 24 + 1, 2 ** 31 + 5, 2 ** 32 + 192])
def test_vocabularies_beyond_the_limit(no_device, vocab):
    """Sizes that a field of 32 bits holds as other ones are refused like any beyond 2^24 (the logits here take four
    bytes)."""
    logits = torch.zeros(1).expand(vocab)
    with pytest.raises(NotImplementedError, match='16777216'):
        ops.token_statistics(logits, tokens())
    with pytest.raises(NotImplementedError, match='16777216'):
        ops.token_gradient(logits, tokens(), torch.zeros(1, 2), grad_log_probs=torch.zeros(()))
    assert not no_device
