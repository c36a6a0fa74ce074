"""Long rows: the sums' error stays that of a short chain whatever the
vocabulary, in rows whose roundings all go one way too."""

import pytest
import torch

from _rows import close, expected_gradient, expected_scores

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def row_of(pattern, vocab, dtype):
    at = torch.arange(vocab, device='cuda')
    if pattern == 'level':
        row = torch.full((vocab,), 0.75, device='cuda')
    elif pattern == 'peak':      # one best token, all others alike: every term of a chain is rounded the same way
        row = torch.where(at == vocab // 3, 10.0, 0.0)
    elif pattern == 'low peak':
        row = torch.where(at == vocab // 3, 5.0, 0.0)
    elif pattern == 'peaks':
        row = torch.where(at % 4099 == 7, 3.0, -1.0 / 3)
    elif pattern == 'creeping':  # a new maximum all the way, each hardly above the last
        row = torch.linspace(0, 1e-3, vocab, device='cuda', dtype=torch.float64).float()
    elif pattern == 'rising':
        row = torch.linspace(-30, 30, vocab, device='cuda')
    elif pattern == 'falling':
        row = torch.linspace(30, -30, vocab, device='cuda')
    elif pattern == 'masked':
        row = torch.where(at % 3 == 0, 0.5, -torch.inf)
    else:
        row = torch.randn(vocab, generator=torch.Generator(device='cuda').manual_seed(3), device='cuda') * 2.5
    return row.to(dtype)


PATTERNS = ['level', 'peak', 'low peak', 'peaks', 'creeping', 'rising', 'falling', 'masked', 'random']


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('vocab', [4099, 50257, 65537, 131072, 262144, 2 ** 20 + 3, 2 ** 24])
@pytest.mark.parametrize('pattern', PATTERNS)
def test_long_rows(pattern, vocab, dtype):
    """Few rows and many, which take different kernels, each within the tests' bound of the formula.  The rows are one
    and the same in memory."""
    from bdm_amd import token_log_probs
    row = row_of(pattern, vocab, dtype)
    one = torch.tensor([vocab // 3], device='cuda')
    want = expected_scores(row[None], one)
    for rows in (3, 256, 300):
        out = token_log_probs(row.expand(rows, -1), one.expand(rows))
        for name in ('log_probs', 'entropy'):
            got = getattr(out, name)
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(got[:1].expand(rows)))  # equal rows, equal results
            close(got[:1], *want[name], (name, rows))


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('pattern', PATTERNS)
def test_gradient_of_long_rows(pattern, dtype):
    """The gradient takes the forward's statistics."""
    from bdm_amd import token_log_probs, token_loss
    vocab, rows = 262144, 256
    logits = row_of(pattern, vocab, dtype).expand(rows, -1).requires_grad_()
    token = torch.tensor([vocab // 3], device='cuda')
    out = token_log_probs(logits, token.expand(rows))
    grad, = torch.autograd.grad(out.log_probs.sum(), [logits])
    close(grad[:1], *expected_gradient(logits.detach()[:1], token, given=torch.ones(1, device='cuda')))
    loss = token_loss(logits, token.expand(rows))
    value, tolerance = expected_scores(logits.detach()[:1], token)['log_probs']
    close(loss, -value[0], tolerance[0] + 2.0 ** -23 * value[0].abs())


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('vocab', [65537, 131075, 200001])
def test_long_rows_of_every_kind(vocab, dtype):
    """Rows whose sums are joined several times: what is not finite or lowest stands at the start, in the middle, at the
    end; rows at every alignment."""
    from bdm_amd import token_log_probs
    rows, lowest = 272, torch.finfo(dtype).min
    gen = torch.Generator(device='cuda').manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=gen, device='cuda') * 2.5).to(dtype)
    tokens = torch.randint(vocab - 1, (rows,), generator=gen, device='cuda')
    for kind, (value, place) in enumerate((v, p) for v in (torch.nan, torch.inf, torch.finfo(dtype).max)
                                          for p in (0, vocab // 2, vocab - 1)):
        logits[kind::17, place] = value
    logits[9::17] = -torch.inf
    logits[10::17] = lowest
    logits[11::17, :vocab // 2] = lowest
    logits[12::17, vocab // 2:] = -torch.inf
    logits[13::17, 5:] = lowest
    logits[14::17, :-5] = -torch.inf
    logits[15::17] *= 1000
    for view in (logits, logits[:, 1:]):
        out = token_log_probs(view, tokens)
        want = expected_scores(view, tokens)
        for name in ('log_probs', 'entropy'):
            close(getattr(out, name), *want[name], name)
