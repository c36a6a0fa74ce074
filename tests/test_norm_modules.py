"""A norm module that does more than its class' forward is called wherever the
model normalizes: no kernel stands in for it."""

import pytest
import torch
from torch import nn

from bdm_amd import BSDMConfig, ops
from bdm_amd.lm import BDMLanguageModel, LanguageModelConfig, LayerNorm, RMSNorm, _layer_norm_ops


def model_of(normalization, layers=2):
    memory = BSDMConfig(dim=64, bank_count=16, bank_size=8, selected_banks=4, value_width=64, num_heads=2)
    return BDMLanguageModel(LanguageModelConfig(memory=memory, vocab_size=50, layers=layers, ffn_multiple_of=32,
                                                normalization=normalization))


class HalvedLayer(LayerNorm):
    def forward(self, x):
        return super().forward(x) * 0.5


class HalvedRMS(RMSNorm):
    def forward(self, x):
        return super().forward(x) * 0.5


def derive(norm):
    norm.__class__ = HalvedLayer if isinstance(norm, LayerNorm) else HalvedRMS


def replace(norm):
    whole = norm.forward
    norm.forward = lambda x: whole(x) * 0.5


def hook(norm):
    norm.register_forward_hook(lambda module, inputs, out: out * 0.5)


def pre_hook(norm):
    norm.register_forward_pre_hook(lambda module, inputs: (inputs[0].flip(-1),))


CHANGES = {f.__name__: f for f in (derive, replace, hook, pre_hook)}


@pytest.fixture
def kernels(monkeypatch):
    """The norms' kernels restated in torch ops, taken for every tensor; their calls are noted."""
    calls = []

    def rms(x, weight, eps, residual=None):
        calls.append('rms')
        total = x if residual is None else residual + x
        out = (total * torch.rsqrt(total.square().mean(-1, keepdim=True) + eps)) * weight
        return out if residual is None else (total, out)

    def layer(x, weight, bias, eps, residual=None):
        calls.append('layer')
        total = x if residual is None else residual + x
        out = _layer_norm_ops(total, weight, bias, eps)
        return out if residual is None else (total, out)

    monkeypatch.setattr(ops, 'rms_norm_supported', lambda x: True)
    monkeypatch.setattr(ops, 'layer_norm_supported', lambda x: True)
    monkeypatch.setattr(ops, 'rms_norm', rms)
    monkeypatch.setattr(ops, 'layer_norm', layer)
    return calls


@pytest.mark.parametrize('change', CHANGES)
@pytest.mark.parametrize('kind', [RMSNorm, LayerNorm])
def test_add_norm(kernels, kind, change):
    """(the sum, the module of the sum), whatever calling the module does."""
    norm = kind(64)
    x, residual = torch.randn(2, 3, 64), torch.randn(2, 3, 64)
    with torch.no_grad():
        norm.add_norm(x, residual)
        assert len(kernels) == 1  # one kernel where the module is plain
        CHANGES[change](norm)
        total, normed = norm.add_norm(x, residual)
        assert torch.equal(total, residual + x)
        assert torch.equal(normed, norm(total))


@pytest.mark.parametrize('change', CHANGES)
@pytest.mark.parametrize('place', ['attention_norm', 'ffn_norm', 'norm'])
@pytest.mark.parametrize('normalization', ['rms', 'layer'])
def test_serving(kernels, normalization, place, change):
    """The blocks without autograd (prompts and tokens, dense and paged) against the modules called one by one."""
    model = model_of(normalization)
    CHANGES[change](model.norm if place == 'norm' else getattr(model.layers[1], place))
    hidden = torch.randn(2, 3, 64)

    def memory(i, normed):
        return normed * (i + 2)

    with torch.no_grad():
        want = hidden
        for i, block in enumerate(model.layers):
            want = want + memory(i, block.attention_norm(want))
            want = want + block.feed_forward(block.ffn_norm(want))
        want = nn.functional.linear(model.norm(want)[:, -1:], model.output.weight)
        assert torch.allclose(model._run_blocks(hidden, memory), want, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize('change', CHANGES)
def test_training(kernels, monkeypatch, change):
    """A block under autograd calls such a norm too."""
    monkeypatch.setattr(LayerNorm, '_trained', lambda self, *t: False)  # the forward's kernel alone
    block = model_of('layer', 1).layers[0]
    block.attention_norm = block.attention = block.feed_forward = nn.Identity()
    CHANGES[change](block.ffn_norm)
    hidden = torch.randn(2, 3, 64)
    total = hidden + hidden
    assert torch.equal(block(hidden), total + block.ffn_norm(total))


@pytest.fixture
def fused_step(monkeypatch):
    """The memory layer's part of the decode step taken for granted."""
    from bdm_amd import BankedDeltaMemory
    monkeypatch.setattr(BankedDeltaMemory, 'step_fused_norm_supported', lambda self, hidden, weight: True)


@pytest.mark.parametrize('place', ['attention_norm', 'ffn_norm', 'norm'])
@pytest.mark.parametrize('change', [*CHANGES, 'layer'])
def test_fused_step_takes_plain_norms_alone(fused_step, place, change):
    """The decode step's kernels form RMSNorm before a product: any other norm, in any place, is not theirs."""
    model = model_of('rms')
    hidden = torch.zeros(1, 1, 64)
    assert model._fused_decode_supported(hidden)
    owner = model if place == 'norm' else model.layers[1]
    if change == 'layer':
        setattr(owner, place, LayerNorm(64))
    else:
        CHANGES[change](getattr(owner, place))
    assert not model._fused_decode_supported(hidden)


def test_fused_step_takes_a_derived_class_without_a_forward(fused_step):
    class Named(RMSNorm):
        pass

    model = model_of('rms')
    for owner, place in ((model, 'norm'), (model.layers[0], 'attention_norm'), (model.layers[1], 'ffn_norm')):
        getattr(owner, place).__class__ = Named
    assert model._fused_decode_supported(torch.zeros(1, 1, 64))


class Wrapped(nn.Module):
    """A block inside a module that hands its attributes on, as compiled and checkpointed ones are."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def __getattr__(self, name):
        try:
            return super().__getattr__(name)
        except AttributeError:
            return getattr(super().__getattr__('inner'), name)


@pytest.mark.parametrize('place', [None, 'attention_norm', 'ffn_norm', 'norm'])
def test_fused_step_of_wrapped_blocks(fused_step, place):
    model = model_of('rms')
    model.layers[0], model.layers[1] = Wrapped(model.layers[0]), Wrapped(model.layers[1])
    if place:
        derive(model.norm if place == 'norm' else getattr(model.layers[1], place))
    assert model._fused_decode_supported(torch.zeros(1, 1, 64)) is (place is None)
