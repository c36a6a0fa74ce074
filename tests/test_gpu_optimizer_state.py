"""An optimizer's saved state holds the norm that it clips by."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def optimizer_of(**options):
    from bdm_amd.optim import MasterAdamW
    gen = torch.Generator(device='cuda').manual_seed(1)
    params = [torch.nn.Parameter(torch.randn(s, generator=gen, device='cuda').to(BF16)) for s in ((31, 40), (9,))]
    return MasterAdamW(params, lr=1e-2, **options)


def step(optimizer, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    for p in optimizer.params:
        p.grad = torch.randn(p.shape, generator=gen, device='cuda').to(BF16)
    return optimizer.step()


@pytest.mark.parametrize('saved,fresh', [(True, False), (False, True)])
def test_resumes_by_the_same_norm(saved, fresh):
    """A run of another norm than the new optimizer's goes on bit for bit."""
    first = optimizer_of(max_norm=0.5, float32_norm=saved)
    step(first, 5)
    other = optimizer_of(max_norm=1.0, float32_norm=fresh)
    other.load_state_dict(first.state_dict())
    other_norm, norm = step(other, 6), step(first, 6)
    assert other_norm.dtype == norm.dtype == (torch.float32 if saved else BF16)
    assert torch.equal(other_norm, norm)
    for i in range(2):
        assert torch.equal(other.master_of(i), first.master_of(i))
        assert all(torch.equal(a, b) for a, b in zip(other.moments_of(i), first.moments_of(i)))


def test_states_without_it_keep_the_option():
    state = optimizer_of().state_dict()
    state.pop('float32_norm', None)
    other = optimizer_of(float32_norm=True)
    other.load_state_dict(state)
    assert other.float32_norm
