"""Models whose norms do more than their class' forward: prompts and tokens, in
dense caches and pages, are those of the modules called one after the other."""

import pytest
import torch

from test_gpu_training_step import batch_of, model_of
from test_norm_modules import CHANGES

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def by_modules(model, tokens, memory):
    """The logits of the last position, every norm called by itself behind a sum of torch's."""
    from bdm_amd import ops
    hidden = model.tok_embeddings(tokens)
    for i, block in enumerate(model.layers):
        hidden = hidden + memory(i, block.attention_norm(hidden))
        hidden = hidden + block.feed_forward(block.ffn_norm(hidden))
    return ops.linear(model.norm(hidden)[:, -1:], model.output.weight)


def changed(normalization, place, change):
    """A model with one changed norm, and the prompt's logits before."""
    model = model_of(BF16, normalization).eval()
    tokens, _ = batch_of(time=9)
    before, _ = model.prefill(tokens[:, :8])
    CHANGES[change](model.norm if place == 'norm' else getattr(model.layers[1], place))
    return model, tokens, before


def prompts(model, tokens):
    """(logits, caches) of the modules by themselves."""
    caches = [None] * len(model.layers)

    def memory(i, normed):
        out, caches[i] = model.layers[i].attention.prefill(normed, None)
        return out

    return by_modules(model, tokens, memory), caches


@pytest.mark.parametrize('change', CHANGES)
@pytest.mark.parametrize('place', ['attention_norm', 'ffn_norm', 'norm'])
@pytest.mark.parametrize('normalization', ['rms', 'layer'])
@torch.no_grad()
def test_prompts(normalization, place, change):
    model, tokens, before = changed(normalization, place, change)
    want, _ = prompts(model, tokens[:, :8])
    got, _ = model.prefill(tokens[:, :8])
    assert torch.equal(got, want) and not torch.equal(got, before)
    pages = model.create_pages(4, 4 * 2 * 16)
    assert torch.equal(model.prefill_pages(tokens[:, :8], pages, [0, 1, 2]), want)


def check_tokens(model, tokens):
    _, caches = prompts(model, tokens[:, :8])
    copies = [c.clone() for c in caches]

    def memory(i, normed):
        out, caches[i] = model.layers[i].attention.step(normed, caches[i])
        return out

    want = by_modules(model, tokens[:, 8:], memory)
    got, _ = model.step(tokens[:, 8:], copies)
    assert torch.equal(got, want)
    pages, others = (model.create_pages(4, 4 * 2 * 16) for _ in range(2))
    for p in (pages, others):
        model.prefill_pages(tokens[:, :8], p, [0, 1, 2])
    want = by_modules(model, tokens[:, 8:], lambda i, normed: model.layers[i].attention.step_pages(normed, others, i))
    assert torch.equal(model.step_pages(tokens[:, 8:], pages), want)


@pytest.mark.parametrize('change', CHANGES)
@pytest.mark.parametrize('place', ['attention_norm', 'ffn_norm', 'norm'])
@torch.no_grad()
def test_layer_norm_tokens(place, change):
    model, tokens, _ = changed('layer', place, change)
    check_tokens(model, tokens)


@pytest.mark.parametrize('change', CHANGES)
@pytest.mark.parametrize('place', ['attention_norm', 'ffn_norm', 'norm'])
@torch.no_grad()
def test_rms_norm_tokens(place, change):
    """The fused decode step leaves such a model to the modules."""
    model, tokens, _ = changed('rms', place, change)
    check_tokens(model, tokens)


@pytest.mark.parametrize('place', ['attention_norm', 'ffn_norm', 'norm'])
@torch.no_grad()
def test_tokens_of_mixed_norms(place):
    """One layer norm among RMS norms."""
    from bdm_amd import LayerNorm
    model = model_of(BF16, 'rms').eval()
    norm = LayerNorm(64).to(device='cuda', dtype=BF16)
    norm.bias.add_(0.5)
    setattr(model if place == 'norm' else model.layers[1], place, norm)
    check_tokens(model, batch_of(time=9)[0])
