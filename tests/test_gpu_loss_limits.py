"""The model's loss at sizes that the token scores do not take: torch's cross
entropy, as for the types that they do not take."""

import pytest
import torch
import torch.nn.functional as F

BF16, FP32 = torch.bfloat16, torch.float32


def test_supported():
    """Fewer than 2^24 rows of at most 2^24 logits, whatever the leading shape (no memory behind these)."""
    from bdm_amd import ops

    def takes(*shape, dtype=BF16):
        return ops.token_scores_supported(torch.empty(shape, dtype=dtype, device='meta'))

    assert takes(2 ** 24 - 1, 2) and takes(4, 2 ** 20, 192, dtype=FP32) and takes(1, 2 ** 24) and takes(0, 5)
    assert not takes(2 ** 24, 2) and not takes(16, 2 ** 20, 192) and not takes(1, 2 ** 24 + 1)
    assert not takes(3, 5, dtype=torch.float16) and not takes(3, 0) and not takes()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('shape', [(16, 2 ** 20, 2), (1, 2, 2 ** 24 + 1)])
def test_model_beyond_the_limits(shape, dtype):
    from bdm_amd import BSDMConfig
    from bdm_amd.lm import BDMLanguageModel, LanguageModelConfig
    memory = BSDMConfig(dim=64, bank_count=16, bank_size=8, selected_banks=4, value_width=64, num_heads=2)
    model = BDMLanguageModel(LanguageModelConfig(memory=memory, vocab_size=2, layers=1, ffn_multiple_of=32))
    gen = torch.Generator(device='cuda').manual_seed(1)
    logits = torch.randn(shape, generator=gen, device='cuda').to(dtype).requires_grad_()
    target = torch.randint(shape[-1], shape[:-1], generator=gen, device='cuda')
    model._hidden = lambda tokens: tokens
    model.norm = torch.nn.Identity()
    model.output = torch.nn.Identity()
    loss = model(logits, target)
    grad, = torch.autograd.grad(loss, [logits])
    want = F.cross_entropy(logits.float().flatten(0, -2), target.flatten())
    assert torch.equal(loss, want)
    assert torch.equal(grad, torch.autograd.grad(want, [logits])[0])
