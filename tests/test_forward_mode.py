"""Forward-mode derivatives: a dual tensor's tangent goes through the token
scores, the loss and the layer norm, whose kernels would drop it."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from _rows import STEP, close
from bdm_amd import LayerNorm, ops, token_log_probs, token_loss

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def normal(*shape, seed=0, device='cpu'):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(device)


@pytest.fixture
def kernels(monkeypatch, request):
    """On the CPU the kernels' results restated, without tangents as a kernel's are."""
    if request.getfixturevalue('device') == 'cuda':
        return
    from bdm_amd.lm import _layer_norm_ops
    from bdm_amd.scoring import _log_probs_ops

    def bare(t):
        return None if t is None else torch.from_numpy(fwad.unpack_dual(t).primal.detach().clone().numpy())

    def statistics(logits, tokens, *, alternatives=0, ignore_index=-100, entropy=True, stats=False):
        x = bare(logits)
        best = x.sort(dim=-1, descending=True, stable=True).indices[..., :alternatives] if alternatives else None
        given, entropies, top = _log_probs_ops(x, tokens, best, ignore_index)
        return given, entropies, top, best, None

    def mean(log_probs, tokens, *, ignore_index=-100):
        counted = tokens != ignore_index
        return -bare(log_probs).sum() / counted.sum(), 1 / counted.sum()

    def layer(x, weight, bias, eps, residual=None):
        x, weight, bias, residual = map(bare, (x, weight, bias, residual))
        total = x if residual is None else residual + x
        out = _layer_norm_ops(total, weight, bias, eps)
        return out if residual is None else (total, out)

    monkeypatch.setattr(ops, 'token_statistics', statistics)
    monkeypatch.setattr(ops, 'token_loss_mean', mean)
    monkeypatch.setattr(ops, 'layer_norm', layer)
    monkeypatch.setattr(ops, 'layer_norm_supported', lambda x: True)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('recorded', [False, True])
def test_token_scores(kernels, device, recorded):
    """d log p_i = v_i - sum p v, dH = -sum p v (log p + H); each a sum of at most 40 FP32 terms, four roundings and the
    exponentials' relative errors."""
    x, v = normal(5, 40, device=device), normal(5, 40, seed=1, device=device)
    tokens = torch.tensor([0, 39, 7, -100, 12], device=device)
    with fwad.dual_level(), torch.set_grad_enabled(recorded):
        out = token_log_probs(fwad.make_dual(x.clone().requires_grad_(recorded), v), tokens, alternatives=3)
        tangents = [fwad.unpack_dual(t).tangent for t in out[:3]]
        values = [fwad.unpack_dual(t).primal for t in out[:3]]
        loss = fwad.unpack_dual(token_loss(fwad.make_dual(x, v), tokens)).tangent
    assert all(t is not None for t in (*tangents, loss))
    logs = torch.log_softmax(x.double(), -1)
    p, vd = logs.exp(), v.double()
    slope = vd - (p * vd).sum(-1, keepdim=True)
    entropy = -(p * logs).sum(-1)
    counted = tokens != -100
    spot = torch.where(counted, tokens, 0)[:, None]
    given = torch.where(counted, slope.gather(1, spot)[:, 0], 0.0)
    best = out.top_tokens
    assert torch.equal(best, x.sort(dim=-1, descending=True, stable=True).indices[:, :3])
    size = 64 * STEP * (1 + vd.abs().max())
    close(tangents[0], given, size)
    close(tangents[1], -(p * vd * (logs + entropy[:, None])).sum(-1), 8 * size)
    close(tangents[2], slope.gather(1, best), size)
    close(values[0], torch.where(counted, logs.gather(1, spot)[:, 0], 0.0), 64 * STEP * 8)
    close(loss, -given.sum() / counted.sum(), size)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('which', ['x', 'residual', 'weight', 'bias'])
def test_layer_norm(kernels, device, which):
    """Against torch's own forward derivative in 64 bits, parameters frozen, one tensor dual."""
    width = 24
    tensors = dict(x=normal(4, width, device=device), residual=normal(4, width, seed=1, device=device),
                   weight=1 + 0.2 * normal(width, seed=2, device=device), bias=normal(width, seed=3, device=device))
    v = normal(*tensors[which].shape, seed=4, device=device)
    norm = LayerNorm(width).to(device)
    norm.requires_grad_(False)

    def run(tensors, module, dual):
        tensors = dict(tensors, **{which: fwad.make_dual(tensors[which], dual)})
        if not module:
            total = tensors['residual'] + tensors['x']
            return total, torch.nn.functional.layer_norm(total, (width,), tensors['weight'], tensors['bias'], 1e-5)
        del norm.weight, norm.bias
        norm.weight, norm.bias = tensors['weight'], tensors['bias']
        total, y = norm.add_norm(tensors['x'], tensors['residual'])
        if which != 'residual':
            assert fwad.unpack_dual(norm(tensors['x'])).tangent is not None
        return total, y

    with fwad.dual_level():
        got = [fwad.unpack_dual(t).tangent for t in run(tensors, True, v)]
        want = [fwad.unpack_dual(t).tangent
                for t in run({n: t.double() for n, t in tensors.items()}, False, v.double())]
    assert got[1] is not None
    close(got[1], want[1], 64 * STEP * 8 * (1 + want[1].abs()))
    if which in ('x', 'residual'):
        close(got[0], want[0], 2 * STEP * want[0].abs())


@pytest.mark.parametrize('device', DEVICES)
def test_kernels_behind_a_level(kernels, device, monkeypatch):
    """Tensors without a tangent take the kernels, inside a dual level too."""
    calls = []
    for name in ('token_statistics', 'layer_norm'):
        inner = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, _inner=inner, **k: (calls.append(1), _inner(*a, **k))[1])
    norm = LayerNorm(8).to(device).requires_grad_(False)
    x, tokens = normal(3, 8, device=device), torch.zeros(3, dtype=torch.int64, device=device)
    with fwad.dual_level():
        norm(x)
        token_log_probs(x, tokens)
    norm(x)
    token_loss(x, tokens)
    assert len(calls) == 4
