"""Layer normalization forward and backward, also behind a residual add, against
the formulas in 64 bits."""

import pytest
import torch

from _rows import CHAIN, STEP, close, expected_norm

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def rows_of(shape, dtype, seed=0, offset=0.0):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(shape, generator=gen, device='cuda') + offset).to(dtype)


def module_of(width, dtype, bias=True, eps=1e-5, seed=3):
    from bdm_amd import LayerNorm
    norm = LayerNorm(width, eps=eps, bias=bias).to(device='cuda', dtype=dtype)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.3 * rows_of((width,), FP32, seed))
        if bias:
            norm.bias.copy_(0.3 * rows_of((width,), FP32, seed + 1))
    return norm


def check(x, norm, residual=None):
    """Without gradients, then with them."""
    want = expected_norm(x, norm.weight, norm.bias, norm.eps, residual, grad=rows_of(x.shape, x.dtype, 7),
                         grad_sum=None if residual is None else rows_of(x.shape, x.dtype, 8))
    with torch.no_grad():
        if residual is None:
            y = norm(x)
        else:
            total, y = norm.add_norm(x, residual)
            close(total, *want['total'], 'total')
    assert y.dtype == x.dtype and y.shape == x.shape
    close(y, *want['y'], 'y')
    x = x.detach().requires_grad_()
    leaves = [x, norm.weight] + ([] if norm.bias is None else [norm.bias])
    if residual is None:
        again = norm(x)
        grads = torch.autograd.grad(again, leaves, rows_of(x.shape, x.dtype, 7))
    else:
        residual = residual.detach().requires_grad_()
        again_total, again = norm.add_norm(x, residual)
        assert torch.equal(again_total, total)
        *grads, second = torch.autograd.grad([again_total, again], [*leaves, residual],
                                             [rows_of(x.shape, x.dtype, 8), rows_of(x.shape, x.dtype, 7)])
        assert torch.equal(second, grads[0])
    assert torch.equal(again, y)
    for name, grad in zip(('dx', 'dw', 'db'), grads):
        close(grad, *want[name], name)


WIDTHS = [1, 2, 3, 7, 8, 9, 31, 63, 64, 65, 127, 128, 255, 511, 512, 513, 1000, 1001, 1024, 1025, 1536, 2047, 2048, 2049,
          4096, 4099, 8191, 8192, 8200, 12288, 16383, 16384]


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('width', WIDTHS)
def test_widths(width, dtype):
    check(rows_of((37, width), dtype), module_of(width, dtype))
    check(rows_of((5, width), dtype), module_of(width, dtype), rows_of((5, width), dtype, 1))


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('rows', [1, 2, 3, 31, 32, 33, 255, 1023, 4097, 20011])
def test_rows(rows, dtype):
    check(rows_of((rows, 96), dtype), module_of(96, dtype))
    check(rows_of((rows, 1001), dtype), module_of(1001, dtype), rows_of((rows, 1001), dtype, 1))


@pytest.mark.parametrize('params', [BF16, FP32])
@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_parameters(dtype, params):
    """Parameters of another type than the rows', and none of a bias."""
    for bias in (True, False):
        check(rows_of((19, 520), dtype), module_of(520, params, bias))
        check(rows_of((19, 77), dtype), module_of(77, params, bias), rows_of((19, 77), dtype, 2))


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_without_parameters(dtype):
    from bdm_amd import ops
    x, dy = rows_of((11, 200), dtype), rows_of((11, 200), dtype, 1)
    want = expected_norm(x, None, None, 1e-5, grad=dy)
    close(ops.layer_norm(x, None, None, 1e-5), *want['y'])
    grad, *none = ops.layer_norm_backward(x, dy, None, None, 1e-5)
    close(grad, *want['dx'])
    assert none == [None, None]
    bias = rows_of((200,), dtype, 4)
    grad, none, db = ops.layer_norm_backward(x, dy, None, bias, 1e-5)
    assert none is None
    close(db, *expected_norm(x, None, bias, 1e-5, grad=dy)['db'])


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_values(dtype):
    """Rows far from zero, level ones (variance 0), large and small ones, columns that stand out."""
    norm = module_of(1024, dtype)
    for offset in (100.0, -1000.0):
        check(rows_of((16, 1024), dtype, 0, offset), norm)
    x = rows_of((8, 1024), dtype)
    x[0] = 3.0
    x[1] = 0.0
    x[2] *= 1e4
    x[3] *= 1e-4
    x[:, 100] = 200.0
    check(x, norm)
    level = torch.full((4, 1024), 5.0, device='cuda', dtype=dtype)
    with torch.no_grad():
        close(norm(level), norm.bias.detach().double().expand(4, -1), 1e-6)


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_not_finite(dtype):
    """A NaN or infinity stays in its row (and in the parameters' gradients, as they sum over rows)."""
    norm = module_of(512, dtype)
    x = rows_of((6, 512), dtype)
    clean = norm(x)
    x[1, 3] = torch.nan
    x[4, 500] = torch.inf
    y = norm(x)
    keep = [0, 2, 3, 5]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[1]).all() and torch.isnan(y[4]).any()


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_layouts(dtype):
    """Leading dimensions, slices, transposed and unaligned rows, and gradients of those layouts."""
    norm = module_of(40, dtype)
    base = rows_of((6, 9, 41), dtype)
    for x in (base[..., 1:], base[..., :40], base[::2, 1:, 1:], rows_of((40, 9), dtype).t(), rows_of((40,), dtype),
              rows_of((1, 40), dtype).expand(12, 40), rows_of((2, 3, 4, 40), dtype)):
        check(x, norm)
        check(x, norm, rows_of(x.shape, dtype, 1))
    x = rows_of((12, 40), dtype).requires_grad_()
    turned = rows_of((40, 12), dtype, 2).t()
    grad, = torch.autograd.grad(norm(x), [x], turned)
    close(grad, *expected_norm(x, norm.weight, norm.bias, norm.eps, grad=turned)['dx'])
    grad, = torch.autograd.grad(norm(x).sum(), [x])   # an expanded gradient
    close(grad, *expected_norm(x, norm.weight, norm.bias, norm.eps, grad=torch.ones_like(x))['dx'])


def test_no_rows():
    norm = module_of(64, BF16)
    x = torch.empty(0, 64, device='cuda', dtype=BF16, requires_grad=True)
    y = norm(x)
    grads = torch.autograd.grad(y, [x, norm.weight, norm.bias], torch.empty_like(y))
    assert y.shape == (0, 64) and (grads[1] == 0).all() and (grads[2] == 0).all()


def test_parts_of_the_gradients():
    """The sum's gradient alone, the norm's alone, parameters without gradients."""
    x, r = (rows_of((10, 96), FP32, s).requires_grad_() for s in (0, 1))
    norm = module_of(96, FP32)
    total, y = norm.add_norm(x, r)
    dy = rows_of((10, 96), FP32, 7)
    grad, = torch.autograd.grad(total, [x], dy, retain_graph=True)
    assert torch.equal(grad, dy)
    grad, = torch.autograd.grad(y, [r], dy, retain_graph=True)
    close(grad, *expected_norm(x, norm.weight, norm.bias, norm.eps, residual=r, grad=dy)['dx'])
    norm.weight.requires_grad_(False)
    norm.bias.requires_grad_(False)
    y = norm(x)
    y.backward(dy)
    close(x.grad, *expected_norm(x, norm.weight, norm.bias, norm.eps, grad=dy)['dx'])
    assert norm.weight.grad is None


def test_gradient_against_differences():
    """Central differences along directions: the third derivatives are below 20 for directions of length 1 of rows of
    width 24, the function's FP32 error that of 3 values of about 3 in every sum of 24."""
    norm = module_of(24, FP32)
    x, dy = rows_of((3, 24), FP32).requires_grad_(), rows_of((3, 24), FP32, 7)
    grads = torch.autograd.grad((norm(x) * dy).sum(), [x, norm.weight, norm.bias])
    h = 2.0 ** -6
    for i, leaf in enumerate((x, norm.weight, norm.bias)):
        direction = rows_of(leaf.shape, FP32, 30 + i)
        direction = direction / direction.norm()
        with torch.no_grad():
            ends = []
            for sign in (1, -1):
                leaf += sign * h * direction
                ends.append((norm(x).double() * dy).sum())
                leaf -= sign * h * direction
        slope = (ends[0] - ends[1]) / (2 * h)
        noise = 72 * 3 * 8 * STEP * 3 / h + 20 * h * h / 6 * 9
        assert abs(float(slope - (grads[i].double() * direction).sum())) <= noise


def test_second_gradient():
    norm = module_of(16, FP32)
    x, r = (rows_of((3, 16), FP32, s).requires_grad_() for s in (0, 1))
    dy, v = rows_of((3, 16), FP32, 7), rows_of((3, 16), FP32, 9)

    def second(form):
        total, y = form(x, r)
        grad, = torch.autograd.grad((y * dy).sum() + total.square().sum(), [x], create_graph=True)
        return torch.autograd.grad((grad * v).sum(), [r, norm.weight])

    def plain(x, r):
        total = x + r
        return total, torch.nn.functional.layer_norm(total, (16,), norm.weight, norm.bias, norm.eps)

    for got, want in zip(second(norm.add_norm), second(plain)):
        close(got, want.double(), 64 * CHAIN * STEP * (want.abs() + 1).double())


def test_rows_beyond_32_bits():
    from bdm_amd import ops
    rows, width = 140000, 16000
    x = torch.zeros(rows, width, device='cuda', dtype=BF16)
    x[-2:] = rows_of((2, width), BF16)
    norm = module_of(width, BF16)
    want = expected_norm(x[-2:], norm.weight, norm.bias, norm.eps, grad=x[-2:])
    with torch.no_grad():
        y = norm(x)
        close(y[-2:], *want['y'])
        del y
        dx, dw, db = ops.layer_norm_backward(x, x, norm.weight, norm.bias, norm.eps)
    close(dx[-2:], *want['dx'])
    close(dw, *want['dw'])
    close(db, *want['db'])


def test_repeats_streams_and_graphs():
    from bdm_amd import ops
    side = torch.cuda.Stream()
    graphs = []
    for seed in range(2):
        x, dy = rows_of((3000, 1001), BF16, seed), rows_of((3000, 1001), BF16, 7 + seed)
        norm = module_of(1001, BF16)

        def work(x=x, dy=dy, norm=norm):
            with torch.no_grad():
                total, y = norm.add_norm(x, dy)
                return total, y, *ops.layer_norm_backward(x, dy, norm.weight, norm.bias, 1e-5, grad_sum=y)

        first = work()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            again = work()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = work()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        graphs.append((graph, x, dy, out, work))
    for turn in range(4):
        for _, x, dy, _, _ in graphs:
            x.copy_(rows_of(x.shape, BF16, 20 + turn))
            dy.copy_(rows_of(x.shape, BF16, 30 + turn))
        for graph, *_ in graphs:
            graph.replay()
        for *_, out, work in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, work()))
        torch.cuda.synchronize()
