"""Padded positions: a token that is ignored passes no gradient to its row,
whatever the row holds."""

import pytest
import torch

from _rows import close, expected_gradient, expected_scores

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def padded(vocab, dtype):
    """Six rows, the ignored ones with a NaN, +inf, infinities of both signs, and nothing finite."""
    gen = torch.Generator(device='cuda').manual_seed(vocab)
    logits = (torch.randn(6, vocab, generator=gen, device='cuda') * 2).to(dtype)
    logits[1, vocab // 2] = torch.nan
    logits[2, 0] = torch.inf
    logits[3] = torch.nan
    logits[4] = torch.where(torch.arange(vocab, device='cuda') % 2 == 0, torch.inf, -torch.inf)
    tokens = torch.tensor([3, -100, -100, -100, -100, vocab - 1], device='cuda')
    return logits.requires_grad_(), tokens


@pytest.mark.parametrize('create', [False, True])
@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('vocab', [7, 192, 5003, 50257])
def test_ignored_rows_pass_no_gradient(vocab, dtype, create):
    from bdm_amd import token_log_probs, token_loss
    logits, tokens = padded(vocab, dtype)
    counted = tokens != -100
    each = torch.where(counted, -0.5, 0.0)  # two tokens count
    loss = token_loss(logits, tokens)
    want = expected_scores(logits[counted], tokens[counted])['log_probs']
    close(loss, -want[0].mean(), want[1].max() + 2.0 ** -23 * want[0].abs().max())
    out = token_log_probs(logits, tokens)
    assert (out.log_probs[~counted] == 0).all() and torch.isnan(out.entropy[~counted]).all()
    for value, gradient in ((loss, None), (out.log_probs, each)):
        grad, = torch.autograd.grad(value, [logits], gradient, create_graph=create)
        assert (grad[~counted] == 0).all()
        close(grad[counted], *expected_gradient(logits[counted], tokens[counted], given=each[counted]))


def test_entropies_of_ignored_rows_do():
    """The entropy is the distribution's, which such a row has not."""
    from bdm_amd import token_log_probs
    logits, tokens = padded(192, FP32)
    out = token_log_probs(logits, tokens)
    grad, = torch.autograd.grad(out.entropy.sum(), [logits])
    assert torch.isnan(grad[1:5]).any(-1).all() and torch.isfinite(grad[[0, 5]]).all()
