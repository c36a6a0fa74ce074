"""Training and scoring steps of the language model with its loss, layer norms,
clipping and optimizer together, and with what each replaces."""

import math

import pytest
import torch
import torch.nn.functional as F
from torch import nn

from _rows import CHAIN, STEP, close, expected_scores, half_step

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def model_of(dtype, normalization='layer', vocab=203, layers=2):
    from bdm_amd import BSDMConfig
    from bdm_amd.lm import BDMLanguageModel, LanguageModelConfig
    memory = BSDMConfig(dim=64, bank_count=16, bank_size=8, selected_banks=4, value_width=64, num_heads=2)
    config = LanguageModelConfig(memory=memory, vocab_size=vocab, layers=layers, ffn_multiple_of=32,
                                 normalization=normalization)
    model = BDMLanguageModel(config).to(device='cuda', dtype=dtype)
    with torch.no_grad():   # norms that are not the identity
        gen = torch.Generator(device='cuda').manual_seed(2)
        for name, p in model.named_parameters():
            if 'norm' in name and 'output_norm' not in name:
                p.add_(torch.randn(p.shape, generator=gen, device='cuda').to(dtype) * 0.2)
    return model


def batch_of(vocab=203, batch=3, time=37, seed=0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    tokens = torch.randint(vocab, (batch, time + 1), generator=gen, device='cuda')
    target = tokens[:, 1:].clone()
    target[1, 20:] = -100   # padding behind a shorter sequence
    return tokens[:, :-1], target


class PlainNorm(nn.LayerNorm):
    """torch's layer norm in the place of the framework's."""

    def add_norm(self, x, residual):
        total = residual + x
        return total, self(total)


def plain_norms(model):
    for owner in [*model.layers, model]:
        for name in ('attention_norm', 'ffn_norm', 'norm'):
            old = getattr(owner, name, None)
            if old is not None:
                new = PlainNorm(old.weight.shape[0], eps=old.eps, device='cuda', dtype=old.weight.dtype)
                new.load_state_dict(old.state_dict())
                setattr(owner, name, new)
    return model


def test_layer_norm_model():
    """A model with layer norms against the same model with torch's: the loss and every gradient (FP32; the routes are
    the same, as no score lies within rounding of another), and without gradients."""
    tokens, target = batch_of()
    losses, gradients, logits = [], [], []
    for change in (lambda m: m, plain_norms):
        model = change(model_of(FP32))
        loss = model(tokens, target)
        loss.backward()
        losses.append(float(loss.detach()))
        gradients.append({n: p.grad for n, p in model.named_parameters()})
        with torch.no_grad():
            logits.append(model(tokens))
    assert losses[0] == pytest.approx(losses[1], rel=1e-5)
    assert float((logits[0] - logits[1]).abs().max()) <= 1e-4 * float(logits[1].abs().max())
    for name, grad in gradients[0].items():
        want = gradients[1][name]
        assert float((grad - want).norm()) <= 1e-3 * float(want.norm()) + 1e-7, name


def test_layer_norm_model_serves():
    """Prompt and tokens one by one, dense, paged and from a graph: the logits of the whole sequence (BF16: within the
    rounding of a residual stream of two layers)."""
    from bdm_amd import LanguageModelGraphDecoder
    model = model_of(BF16).eval()
    tokens, _ = batch_of(time=12)
    with torch.no_grad():
        whole = model(tokens).float()
        logits, caches = model.prefill(tokens[:, :8])
        pages = model.create_pages(4, 4 * 2 * 16)
        paged = model.prefill_pages(tokens[:, :8], pages, [0, 1, 2])
        decoder = LanguageModelGraphDecoder(model, [c.clone() for c in caches])
        size = float(whole.abs().max())
        for t in range(8, 12):
            close(logits[:, 0], whole[:, t - 1].double(), 0.06 * size)
            close(paged[:, 0], whole[:, t - 1].double(), 0.06 * size)
            step = tokens[:, t:t + 1]
            replayed = decoder.step(step).clone()
            logits, caches = model.step(step, caches)
            paged = model.step_pages(step, pages)
            assert torch.equal(replayed, logits)


@pytest.mark.parametrize('normalization', ['rms', 'layer'])
@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_loss_of_the_model(dtype, normalization):
    """The model's loss is its logits' cross entropy, and the logits receive its gradient."""
    model = model_of(dtype, normalization)
    tokens, target = batch_of()
    seen = []
    model.output.register_forward_hook(lambda m, i, out: (out.retain_grad(), seen.append(out))[0])
    loss = model(tokens, target)
    loss.backward()
    logits = seen[0]
    reference = logits.detach().double().requires_grad_()
    want = F.cross_entropy(reference.flatten(0, 1), target.flatten())
    want.backward()
    close(loss, want.detach(), 2 * CHAIN * STEP + 4 * STEP * float(want.detach()))
    p = torch.softmax(reference.detach(), -1)
    share = (target != -100).double().unsqueeze(-1) / (target != -100).sum()
    # p's relative error, the given token's own term, and a rounding
    close(logits.grad, reference.grad, (half_step(dtype) * 1.01) * reference.grad.abs()
          + share * (2 * p * (CHAIN + 40) * STEP + 8 * STEP))


def test_score():
    model = model_of(BF16, 'rms')
    tokens, target = batch_of()
    with torch.no_grad():
        out = model.score(tokens, target, alternatives=5)
        logits = model(tokens)
    want = expected_scores(logits, target, 5)
    assert torch.equal(out.top_tokens, want['top_tokens'])
    for name in ('log_probs', 'entropy', 'top_log_probs'):
        close(getattr(out, name), *want[name], name)
    out = model.score(tokens, target)
    (out.log_probs.sum() + out.entropy.sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())


def test_steps_together():
    """Two updates of a layer-norm model: the loss, every gradient clipped in place, the optimizer with the FP32 norm.
    The second norm, of clipped gradients, is the largest allowed one, and the weights move."""
    from bdm_amd import clip_gradients, gradient_norm
    from bdm_amd.optim import MasterAdamW
    model = model_of(BF16)
    params = list(model.parameters())
    optimizer = MasterAdamW(params, lr=1e-3, max_norm=0.25, float32_norm=True)
    for seed in range(2):
        before = [p.detach().clone() for p in params]
        optimizer.zero_grad()
        loss = model(*batch_of(seed=seed))
        loss.backward()
        gradients = [p.grad for p in params]
        want = math.sqrt(math.fsum(float(g.double().square().sum()) for g in gradients))
        norm = clip_gradients(gradients, 0.25)
        assert abs(float(norm) - want) <= 2 * STEP * want
        largest = min(want, 0.25)
        # each clipped value is off by half a BF16 step at most
        assert abs(float(gradient_norm(gradients)) - largest) <= 1.01 * half_step(BF16) * largest
        assert abs(float(optimizer.step()) - largest) <= 1.01 * half_step(BF16) * largest
        assert any(not torch.equal(p, b) for p, b in zip(params, before))
        assert all(torch.isfinite(p).all() for p in params)


@pytest.mark.parametrize('normalization', ['rms', 'layer'])
def test_logits_behind_a_step(normalization):
    """Logits without gradients before and behind an update: the second ones are those of a new model with the updated
    weights, whatever the first call has prepared of the old ones."""
    from bdm_amd.optim import MasterAdamW
    model = model_of(BF16, normalization)
    tokens, target = batch_of()
    optimizer = MasterAdamW(list(model.parameters()), lr=0.05)
    with torch.no_grad():
        before = model(tokens)
    model(tokens, target).backward()
    optimizer.step()
    other = model_of(BF16, normalization)
    other.load_state_dict(model.state_dict())
    with torch.no_grad():
        after, want = model(tokens), other(tokens)
    assert not torch.equal(before, want)
    assert torch.equal(after, want)
