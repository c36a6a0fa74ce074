"""The gradients' norm and clipping against sums in 64 bits."""

import math

import pytest
import torch

from _rows import STEP, close, half_step

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def gradients_of(shapes, dtypes, seed=0, std=1.0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return [(torch.randn(s, generator=gen, device='cuda') * std).to(d) for s, d in zip(shapes, dtypes)]


def norm_of(gradients):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in gradients))


def check_norm(gradients):
    from bdm_amd import gradient_norm
    got, want = gradient_norm(gradients), norm_of(gradients)
    assert got.dtype == FP32 and got.shape == ()
    # FP64 sums and one rounding
    assert abs(float(got) - want) <= 2 * STEP * want


def check_clip(gradients, max_norm, out=None):
    from bdm_amd import clip_gradients
    before = [g.clone() for g in gradients]
    want = norm_of(before)
    norm = clip_gradients(gradients, max_norm, out=out)
    assert abs(float(norm) - want) <= 2 * STEP * want
    factor = min(1.0, max_norm / (want + 1e-6))
    for g, b, o in zip(gradients, before, out or gradients):
        # the factor and the product in FP32, and one rounding; below the smallest normal number half of the smallest
        value = b.double() * factor
        close(o, value, (3 * STEP + half_step(o.dtype)) * value.abs() * 1.01 + 2.0 ** -134)
        if out is not None:
            assert torch.equal(g, b)
        elif factor == 1.0:
            assert torch.equal(o, b)


SHAPES = {
    'one': [(1,)],
    'scalar': [()],
    'odd': [(7,), (33, 65), (1, 1), (), (16385,), (3, 5, 7)],
    'empty': [(0,), (5,), (4, 0, 3), (8,)],
    'chunks': [(16384,), (16383,), (32768,), (65537,), (300001,)],
    'many': [(i % 37 + 1, i % 11 + 1) for i in range(700)],
    'model': [(128, 512), (512,), (192, 128)] * 40,
    'large': [(4096, 4099), (50257, 129)],
}


@pytest.mark.parametrize('kind', ['bf16', 'fp32', 'mixed'])
@pytest.mark.parametrize('shapes', SHAPES)
def test_tensors(shapes, kind):
    shapes = SHAPES[shapes]
    dtypes = [BF16 if kind == 'bf16' or (kind == 'mixed' and i % 2) else FP32 for i in range(len(shapes))]
    gradients = gradients_of(shapes, dtypes)
    check_norm(gradients)
    norm = norm_of(gradients)
    check_clip(gradients, 2 * norm + 1)   # nothing to clip
    check_clip(gradients, norm / 3)
    for out in (BF16, FP32):
        gradients = gradients_of(shapes, dtypes, 1)
        check_clip(gradients, norm / 3, [torch.full_like(g, 7, dtype=out) for g in gradients])
        check_clip(gradients, 2 * norm + 1, [torch.full_like(g, 7, dtype=out) for g in gradients])


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_unaligned(dtype):
    """Tensors that start and end anywhere, next to each other in one buffer."""
    flat = torch.randn(70000, device='cuda').to(dtype)
    cuts = [0, 1, 4, 9, 1000, 1003, 17390, 50001, 70000]
    views = [flat[a:b] for a, b in zip(cuts, cuts[1:])]
    check_norm(views)
    target = torch.full((70001,), 7.0, device='cuda', dtype=BF16)
    check_clip(views, 1.0, [target[1:][a:b] for a, b in zip(cuts, cuts[1:])])
    assert float(target[0]) == 7
    check_clip(views[1::2], 1.0)
    check_clip(views, 1.0)


def test_very_large():
    """A tensor of more than 2^30 elements, in several entries of a launch."""
    from bdm_amd import clip_gradients, gradient_norm
    n = (1 << 30) + 17
    g = torch.full((n,), 0.5, device='cuda', dtype=BF16)
    g[-1] = 2.0 ** 14
    want = math.sqrt(0.25 * (n - 1) + 2.0 ** 28)
    assert abs(float(gradient_norm([g])) - want) <= 2 * STEP * want
    clip_gradients([g], want / 4)
    ends = torch.cat([g[:3], g[(1 << 29) - 2:(1 << 29) + 2], g[-3:]]).double().cpu()
    close(ends, torch.tensor([0.125] * 9 + [2.0 ** 12], dtype=torch.float64), 2.0 ** -8 * torch.ones(10) * ends.abs())
    assert float((g[:-1].float() - 0.125).abs().max()) <= 2.0 ** -8 * 0.125


def test_layouts():
    """Transposed gradients are clipped in place; those with holes have a norm, and go to out."""
    from bdm_amd import clip_gradients
    base = torch.randn(64, 96, device='cuda')
    check_norm([base.t(), base[:, ::2]])
    check_clip([base.t()], 1.0)
    check_clip([base.t()], 0.5, [torch.empty(64, 96, device='cuda').t()])
    check_clip([base.t()], 0.5, [torch.empty(96, 64, device='cuda', dtype=BF16)])
    check_clip([base[:, ::2]], 0.25, [torch.empty(64, 48, device='cuda')])
    with pytest.raises(ValueError, match='fill'):
        clip_gradients([base[:, ::2]], 1.0)
    with pytest.raises(ValueError, match='contiguous'):
        clip_gradients([base], 1.0, out=[torch.empty(96, 64, device='cuda').t()])


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_range(dtype):
    """Values whose squares FP32 does not hold, and far smaller ones."""
    for scale in (1e30, 1e-30, 1e-38):
        check_norm([(torch.randn(5000, device='cuda') * scale).to(dtype)])
    check_clip([(torch.randn(5000, device='cuda') * 1e30).to(dtype)], 1.0)
    check_clip([(torch.randn(5000, device='cuda') * 1e30).to(dtype), torch.randn(100, device='cuda').to(dtype)], 1e20)
    check_clip([(torch.randn(50, device='cuda') * 1e-30).to(dtype)], 1.0)
    check_norm([torch.zeros(100, device='cuda', dtype=dtype)])
    check_clip([torch.zeros(100, device='cuda', dtype=dtype)], 0.0)
    check_clip([torch.randn(100, device='cuda').to(dtype)], 0.0)
    check_clip([torch.randn(100, device='cuda').to(dtype)], math.inf)
    # the largest values: the norm is beyond FP32
    from bdm_amd import clip_gradients, gradient_norm
    big = torch.full((1000,), torch.finfo(dtype).max, device='cuda', dtype=dtype)
    assert float(gradient_norm([big])) == math.inf
    want = big.double() * (1.0 / (float(big[0]) * math.sqrt(1000)))
    clip_gradients([big], 1.0)
    # the factor is below the smallest normal FP32 number: half of 2^-149 of 9e-41 more
    close(big, want, (half_step(dtype) * 1.01 + 1e-4) * want)


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_not_finite(dtype):
    """As torch's clipping: an infinite norm gives the factor 0, a NaN NaN."""
    from bdm_amd import clip_gradients
    a, b = torch.ones(100, device='cuda', dtype=dtype), torch.ones(7, device='cuda', dtype=dtype)
    a[3] = math.inf
    assert float(clip_gradients([a, b], 1.0)) == math.inf
    assert torch.isnan(a[3]) and (a[:3] == 0).all() and (b == 0).all()
    b[2] = math.nan
    assert math.isnan(float(clip_gradients([a, b], 1.0)))
    assert torch.isnan(a).all() and torch.isnan(b).all()


def test_lists():
    """None is passed over, a repeated tensor counts twice in the norm, generators are taken, no tensors have norm 0."""
    from bdm_amd import clip_gradients, gradient_norm
    g = torch.randn(100, device='cuda')
    want = norm_of([g])
    assert abs(float(gradient_norm([None, g, None])) - want) <= 2 * STEP * want
    assert abs(float(gradient_norm([g, g])) - want * 2 ** 0.5) <= 2 * STEP * want * 2
    assert float(gradient_norm(t for t in [g])) == float(gradient_norm([g]))
    assert float(gradient_norm([])) == 0 and float(gradient_norm([None])) == 0 and float(clip_gradients([], 1.0)) == 0
    assert float(gradient_norm([torch.empty(0, device='cuda')])) == 0
    out = torch.full((100,), 7.0, device='cuda')
    clip_gradients([None, g], 1.0, out=[out, g.clone()])
    assert (out == 7).all()
    clip_gradients(iter([None, g]), want / 2)
    assert abs(norm_of([g]) - want / 2) <= 1e-5 * want


def test_shared_memory_is_refused():
    from bdm_amd import clip_gradients
    g = torch.randn(100, device='cuda')
    before = g.clone()
    for gradients, out in (([g, g], None), ([g[:60], g[50:]], None), ([g], [g.view(BF16)[:100]]),
                           ([g[:50], torch.randn(50, device='cuda')], [torch.empty(50, device='cuda'), g[:50]]),
                           ([g[:50], g[50:]], [g[50:], g[:50]]), ([g[1:]], [g[:-1]])):
        with pytest.raises(ValueError, match='share memory'):
            clip_gradients(gradients, 1.0, out=out)
    assert torch.equal(g, before)
    clip_gradients([g[:60], g[50:]], 1.0, out=[torch.empty(60, device='cuda'), torch.empty(50, device='cuda')])


def test_repeats_streams_and_graphs():
    """The same bits on every call and stream; captured calls replayed beside each other with new gradients."""
    from bdm_amd import clip_gradients, gradient_norm
    gradients = gradients_of(SHAPES['many'] + SHAPES['chunks'], [BF16, FP32] * 400)
    first = gradient_norm(gradients)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            again = gradient_norm(gradients)
        assert torch.equal(gradient_norm(gradients), first)
        torch.cuda.synchronize()
        assert torch.equal(again, first)
    graphs = []
    for seed in range(2):
        mine = gradients_of(SHAPES['odd'] + SHAPES['many'], [BF16, FP32] * 400, seed)
        out = [torch.empty_like(g, dtype=FP32) for g in mine]
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            clip_gradients(mine, 1.0, out=out)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                norm = clip_gradients(mine, 1.0, out=out)
        torch.cuda.current_stream().wait_stream(side)
        graphs.append((graph, mine, out, norm))
    for turn in range(4):
        for graph, mine, out, norm in graphs:
            for g, n in zip(mine, gradients_of([g.shape for g in mine], [g.dtype for g in mine], 10 + turn, 0.01 + turn)):
                g.copy_(n)
        for graph, *_ in graphs:
            graph.replay()
        for _, mine, out, norm in graphs:
            eager = [torch.empty_like(o) for o in out]
            assert torch.equal(clip_gradients(mine, 1.0, out=eager), norm)
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
        torch.cuda.synchronize()


def test_optimizer():
    """MasterAdamW with float32_norm: the norm of all gradients, and an update by the gradients clipped with it."""
    from bdm_amd.optim import MasterAdamW
    shapes = [(33, 64), (64,), (128, 7)]
    norms, weights = [], []
    for exact in (False, True):
        params = [torch.nn.Parameter(p) for p in gradients_of(shapes, [BF16] * 3, 3)]
        optimizer = MasterAdamW(params, lr=1e-2, max_norm=0.5, float32_norm=exact)
        for step in range(2):
            for p, g in zip(params, gradients_of(shapes, [BF16] * 3, 5 + step)):
                p.grad = g
            norms.append((optimizer.step(), norm_of([p.grad for p in params])))
        weights.append([optimizer.master_of(i).clone() for i in range(3)])
    for norm, want in norms[:2]:
        assert abs(float(norm) - want) <= 4 * half_step(BF16) * want  # torch's: tensors' norms and the total rounded to BF16
    for norm, want in norms[2:]:
        assert norm.dtype == FP32 and abs(float(norm) - want) <= 2 * STEP * want
    # Adam's first steps are lr * sign-like: clipped gradients that differ by 2^-7 move a weight by far less than lr
    for a, b in zip(*weights):
        assert float((a - b).abs().max()) <= 1e-2
    params = [torch.nn.Parameter(p) for p in gradients_of(shapes, [BF16] * 3, 3)]
    torch_norm = MasterAdamW(params, max_norm=-1.0, float32_norm=True)
    for p in params:
        p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match='negative'):
        torch_norm.step()


@pytest.mark.parametrize('inplace', [True, False])
def test_autograd_sees_the_write(inplace):
    """A tensor that a backward pass has saved and that is clipped, or written as an output, is refused by it."""
    from bdm_amd import clip_gradients
    gen = torch.Generator(device='cuda').manual_seed(4)
    g, other = (torch.randn(50, generator=gen, device='cuda') for _ in range(2))
    leaf = torch.ones(50, device='cuda', requires_grad=True)
    y = leaf * g
    read = other._version
    clip_gradients([None, g if inplace else other], 0.5, out=None if inplace else [None, g])
    assert other._version == read
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
