"""The factor that clips: given by the norm's call, and applied by the optimizer.

Adam's update hardly changes when all gradients are scaled alike; its moments do."""

import math

import pytest
import torch

from _rows import STEP, close, half_step

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
SHAPES = [(33, 64), (64,), (128, 7)]


def gradients_of(seed, std=1.0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return [(torch.randn(s, generator=gen, device='cuda') * std).to(BF16) for s in SHAPES]


def norm_of(gradients):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in gradients))


@pytest.mark.parametrize('share', [0.0, 1e-3, 0.3, 0.999, 1.0, 1.001, 7.0, math.inf])
def test_factor(share):
    """min(1, max / (n + 1e-6)) in FP64, rounded once; the norm beside it is the one without a factor."""
    from bdm_amd import gradient_norm, ops
    gradients = gradients_of(1)
    norm = norm_of(gradients)
    got, factor = ops.gradient_norm(gradients, max_norm=norm * share)
    assert torch.equal(got, gradient_norm(gradients)) and factor.dtype == FP32 and factor.shape == ()
    want = min(1.0, norm * share / (norm + 1e-6))
    assert abs(float(factor) - want) <= 1.01 * STEP * want
    if share > 1:
        assert float(factor) == 1


def test_factor_of_other_norms():
    """No gradients but zeros, infinite and NaN ones, and none at all."""
    from bdm_amd import ops
    g = torch.zeros(50, device='cuda')
    assert [float(t) for t in ops.gradient_norm([g], max_norm=0.5)] == [0, 1]
    assert [float(t) for t in ops.gradient_norm([g], max_norm=0.0)] == [0, 0]
    g[3] = math.inf
    assert [float(t) for t in ops.gradient_norm([g], max_norm=0.5)] == [math.inf, 0]
    g[4] = math.nan
    assert all(math.isnan(float(t)) for t in ops.gradient_norm([g], max_norm=0.5))
    assert [float(t) for t in ops.gradient_norm([], max_norm=0.5)] == [0, 1]


@pytest.mark.parametrize('share', [0.02, 0.5, 3.0])
def test_optimizer_applies_it(share):
    """The moments behind the first step: (1 - beta1) c g and (1 - beta2) (c g)^2, with c the factor; behind a second
    one their running means.  The update takes c g rounded to BF16, as clipping in place would leave it: half a step of
    the value in the first moment, and (1 + h)^2 - 1 <= 2.01 h of its square in the second."""
    from bdm_amd.optim import MasterAdamW
    params = [torch.nn.Parameter(p) for p in gradients_of(2)]
    first = norm_of(gradients_of(3))
    optimizer = MasterAdamW(params, lr=1e-3, max_norm=first * share, float32_norm=True)
    beta1, beta2 = optimizer.betas
    means = [(torch.zeros(s, device='cuda', dtype=torch.float64),) * 2 for s in SHAPES]
    for seed in (3, 4):
        gradients = gradients_of(seed, 1.0 if seed == 3 else 2.5)
        for p, g in zip(params, gradients):
            p.grad = g
        norm = norm_of(gradients)
        assert abs(float(optimizer.step()) - norm) <= 2 * STEP * norm
        factor = min(1.0, first * share / (norm + 1e-6))
        for i, g in enumerate(gradients):
            # the rounding to BF16; the factor, the products and sums of FP32, each within a few steps
            clipped = g.double() * factor
            m, v = means[i]
            bound = [beta1 * m.abs() + (1 - beta1) * clipped.abs(), beta2 * v + (1 - beta2) * clipped.square()]
            means[i] = (beta1 * m + (1 - beta1) * clipped, beta2 * v + (1 - beta2) * clipped.square())
            # 1 - 0.95 of FP32 numbers is off by 2^-25 / 0.05, beta itself by half a step
            for got, want, size, rounding in zip(optimizer.moments_of(i), means[i], bound, (1, 2.01)):
                close(got, want, (rounding * half_step(BF16) + 40 * STEP) * size + 1e-37)
