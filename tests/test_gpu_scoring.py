"""Token log-probabilities, entropies, alternatives, the mean loss and their
gradients against the formulas in 64 bits."""

import pytest
import torch

from _rows import CHAIN, STEP, close, distribution, expected_gradient, expected_scores, order

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


def logits_of(rows, vocab, dtype, seed=0, std=2.5):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(rows, vocab, generator=gen, device='cuda') * std).to(dtype)


def tokens_of(rows, vocab, seed=1):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randint(vocab, (rows,), generator=gen, device='cuda')


def check(logits, tokens, alternatives=0, ignore_index=-100, out=None):
    from bdm_amd import token_log_probs
    if out is None:
        out = token_log_probs(logits, tokens, alternatives=alternatives, ignore_index=ignore_index)
    want = expected_scores(logits, tokens, alternatives, ignore_index)
    close(out.log_probs, *want['log_probs'], 'log_probs')
    close(out.entropy, *want['entropy'], 'entropy')
    if alternatives:
        assert torch.equal(out.top_tokens, want['top_tokens'])
        close(out.top_log_probs, *want['top_log_probs'], 'top_log_probs')
    else:
        assert out.top_log_probs is None and out.top_tokens is None
    return out


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('vocab', [1, 2, 3, 7, 8, 63, 64, 65, 191, 192, 511, 512, 513, 1000, 2047, 2049, 4096, 4099, 8191,
                                   16384, 16391, 32001, 32768, 50257, 65535, 65536, 65537, 131072, 262144])
def test_vocabularies(vocab, dtype):
    rows = 5 if vocab > 20000 else 67
    logits, tokens = logits_of(rows, vocab, dtype, vocab), tokens_of(rows, vocab)
    check(logits, tokens)
    for k in (1, 4, 32):
        if k <= vocab:
            check(logits, tokens, k)


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('rows', [1, 2, 63, 64, 255, 256, 257, 1023, 2049])
def test_rows(rows, dtype):
    for vocab in (192, 5003, 9001):
        check(logits_of(rows, vocab, dtype, rows), tokens_of(rows, vocab))
        check(logits_of(rows, vocab, dtype, rows), tokens_of(rows, vocab), 5)


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('vocab', [9001, 50257])
def test_many_rows(vocab, dtype):
    """Rows of every alignment, masked, empty, level, not finite ones among many."""
    rows = 600
    logits, tokens = logits_of(rows, vocab, dtype), tokens_of(rows, vocab)
    lowest = torch.finfo(dtype).min
    for first, change in ((0, -torch.inf), (1, lowest), (2, torch.finfo(dtype).max), (3, 7.0)):
        logits[first::16] = change
    logits[4::16, 5:] = -torch.inf
    logits[5::16, :-5] = lowest
    logits[6::16, vocab // 3] = torch.nan
    logits[7::16, vocab // 2] = torch.inf
    logits[8::16, ::2] = -torch.inf
    logits[9::16] *= 1000
    logits[10::16] = torch.linspace(-90, 90, vocab, device='cuda').to(dtype)
    logits[11::16] = torch.linspace(90, -90, vocab, device='cuda').to(dtype)
    check(logits, tokens)
    check(logits, tokens, 3)
    check(logits[:, 1:], tokens_of(rows, vocab - 1))


@pytest.mark.parametrize('vocab', [5, 192, 3001, 20000, 50257])
@pytest.mark.parametrize('k', [1, 2, 5, 8, 20, 31, 32])
def test_alternatives(k, vocab):
    if k > vocab:
        k = vocab
    for dtype in (BF16, FP32):
        check(logits_of(9, vocab, dtype, k), tokens_of(9, vocab), k)


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('vocab', [192, 700, 1500, 3000, 4099, 10000, 20000, 40000, 50257, 60000, 70000])
def test_masks(vocab, dtype):
    """Rows that keep a few tokens, one, or none; masks of -inf and of the type's lowest value."""
    for mask in (-torch.inf, torch.finfo(dtype).min):
        logits, tokens = logits_of(8, vocab, dtype), tokens_of(8, vocab)
        logits[0] = mask
        logits[1, 1:] = mask
        logits[2, :-1] = mask
        logits[3, vocab // 2:] = mask
        logits[4, torch.arange(vocab, device='cuda') % 97 != 5] = mask
        logits[5, :vocab - 3] = mask
        tokens[:3] = torch.tensor([0, 0, vocab - 1], device='cuda')
        for k in (0, 1, 8, 32):
            out = check(logits, tokens, k)
        if mask == -torch.inf:
            assert float(out.entropy[0]) == 0 and float(out.log_probs[0]) == -torch.inf
            assert float(out.log_probs[1]) == 0 and float(out.entropy[1]) == 0


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('vocab', [192, 700, 1500, 3000, 4099, 10000, 20000, 40000, 50257, 60000, 70001])
def test_ties_and_orders(vocab, dtype):
    """Level rows, ascending and descending ones, two values, both zeros, most of the best in one place."""
    ramp = torch.linspace(-20, 20, vocab, device='cuda')
    rows = [torch.zeros(vocab, device='cuda'), torch.full((vocab,), -7.5, device='cuda'), ramp, ramp.flip(0),
            (torch.arange(vocab, device='cuda') % 2).float(), (torch.arange(vocab, device='cuda') % 31 == 30).float(),
            torch.where(torch.arange(vocab, device='cuda') % 3 == 0, -0.0, 0.0),
            torch.where(torch.arange(vocab, device='cuda') < 8, 5.0 + ramp, -1.0),
            torch.where(torch.arange(vocab, device='cuda') % 1024 < 8, 5.0 + ramp, ramp.sin())]
    logits = torch.stack(rows).to(dtype)
    for k in (1, 3, 17, 32):
        check(logits, tokens_of(len(rows), vocab), k)


@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('vocab', [192, 700, 1500, 3000, 4099, 10000, 20000, 40000, 50257, 60000, 70001])
def test_not_finite(vocab, dtype):
    """A NaN or +inf makes its row NaN, and only that row; the alternatives keep their order, a NaN first."""
    logits, tokens = logits_of(6, vocab, dtype), tokens_of(6, vocab)
    logits[0, vocab // 3] = torch.nan
    logits[1, vocab // 2] = torch.inf
    logits[2, 3::7] = torch.nan
    logits[3] = torch.nan
    logits[4] = -torch.inf
    logits[4, 5] = torch.nan
    out = check(logits, tokens, 8)
    assert torch.isnan(out.log_probs[:5]).all() and torch.isnan(out.entropy[:5]).all()
    assert torch.isfinite(out.log_probs[5])


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_large_values(dtype):
    """Logits far apart and near the type's largest: no overflow of what is finite."""
    logits = logits_of(4, 5000, dtype, 3, 1e4)
    logits[1] = logits[1] * 1e30
    logits[2] = 1e38
    logits[3, 17] = torch.finfo(dtype).max
    tokens = logits.argmax(-1)
    check(logits, tokens, 6)


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_strides(dtype):
    """Slices of padded vocabularies, rows that start anywhere, transposed and repeated rows, leading dimensions."""
    from bdm_amd import token_log_probs
    wide = logits_of(24, 4123, dtype)
    for first in (0, 1, 2, 3, 5, 8):
        view = wide[:, first:first + 4099]
        check(view, tokens_of(24, 4099), 4)
    check(wide.t()[:100], tokens_of(100, 24), 4)
    check(wide[::3], tokens_of(8, 4123), 4)
    check(wide[:1].expand(7, -1), tokens_of(7, 4123), 4)
    cube = wide.view(2, 3, 4, 4123)
    for view in (cube, cube[:, :, 1:3, 7:], cube.transpose(0, 2), cube[:, 1]):
        tokens = torch.randint(view.shape[-1], view.shape[:-1], device='cuda')
        check(view, tokens, 3)
        check(view, torch.randint(view.shape[-1], (*view.shape[:-1], 2), device='cuda')[..., 0], 3)
    one = wide[0]
    out = token_log_probs(one, torch.tensor(9, device='cuda'), alternatives=2)
    assert out.log_probs.shape == () and out.top_tokens.shape == (2,)
    check(one, torch.tensor(9, device='cuda'), 2)


def test_no_rows():
    from bdm_amd import token_log_probs, token_loss
    out = token_log_probs(torch.empty(0, 192, device='cuda'), torch.empty(0, device='cuda', dtype=torch.int64), alternatives=3)
    assert out.log_probs.shape == out.entropy.shape == (0,) and out.top_tokens.shape == (0, 3)
    logits = torch.empty(2, 0, 192, device='cuda', requires_grad=True)
    loss = token_loss(logits, torch.empty(2, 0, device='cuda', dtype=torch.int64))
    assert torch.isnan(loss)
    loss.backward()
    assert logits.grad.shape == logits.shape


def test_ignored_and_outside_tokens():
    from bdm_amd import token_log_probs
    logits = logits_of(6, 300, FP32).requires_grad_()
    tokens = torch.tensor([-100, 0, 299, 300, -1, 2 ** 40], device='cuda')
    out = token_log_probs(logits, tokens, alternatives=2)
    check(logits, tokens, 2, out=out)
    assert float(out.log_probs[0].detach()) == 0 and torch.isnan(out.log_probs[3:]).all()
    out.entropy.sum().backward()
    assert torch.isfinite(logits.grad).all()  # the outside tokens' NaN is the log-probabilities' alone
    logits.grad = None
    token_log_probs(logits, tokens).log_probs.sum().backward()
    assert (logits.grad[0] == 0).all() and torch.isfinite(logits.grad[1:3]).all() and torch.isnan(logits.grad[3:]).all()
    check(logits.detach(), torch.where(tokens == -100, 7, tokens), ignore_index=7)


# ------------------------------------------------------------------ gradients

@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('vocab', [1, 7, 192, 1001, 4096, 16391, 50257, 131075])
@pytest.mark.parametrize('wanted', ['given', 'entropy', 'top', 'given+entropy', 'given+entropy+top'])
def test_gradients(vocab, dtype, wanted):
    from bdm_amd import token_log_probs
    rows, k = 7, min(5, vocab)
    logits = logits_of(rows, vocab, dtype, 5)
    tokens = tokens_of(rows, vocab)
    tokens[0] = logits[0].argmax()   # also an alternative
    tokens[1] = -100
    if vocab > 100:
        logits[2, ::2] = -torch.inf
        logits[3] = -torch.inf
        logits[4, 1:] = torch.finfo(dtype).min
    logits.requires_grad_()
    gen = torch.Generator(device='cuda').manual_seed(9)
    out = token_log_probs(logits, tokens, alternatives=k)
    given, entropy = (torch.randn(rows, generator=gen, device='cuda') for _ in range(2))
    top = torch.randn(rows, k, generator=gen, device='cuda')
    pick = [(n, o, g) for n, o, g in (('given', out.log_probs, given), ('entropy', out.entropy, entropy),
                                      ('top', out.top_log_probs, top)) if n in wanted.split('+')]
    grad, = torch.autograd.grad([o for _, o, _ in pick], [logits], [g for _, _, g in pick])
    want = expected_gradient(logits, tokens, out.top_tokens, **{n: g for n, _, g in pick})
    assert grad.dtype == dtype and grad.is_contiguous()
    close(grad, *want, wanted)


@pytest.mark.parametrize('dtype', [BF16, FP32])
def test_gradients_of_views(dtype):
    """A padded vocabulary's slice and transposed logits: the gradient goes back to where they came from."""
    from bdm_amd import token_log_probs
    base = logits_of(12, 1031, dtype).requires_grad_()
    tokens = tokens_of(12, 1001)
    weight = torch.randn(12, device='cuda')
    (token_log_probs(base[:, 3:1004], tokens).log_probs * weight).sum().backward()
    want, tolerance = expected_gradient(base[:, 3:1004], tokens, given=weight)
    close(base.grad[:, 3:1004], want, tolerance)
    assert (base.grad[:, :3] == 0).all() and (base.grad[:, 1004:] == 0).all()
    base.grad = None
    turned = base.t()[:500]
    tokens = tokens_of(500, 12)
    token_log_probs(turned, tokens).entropy.sum().backward()
    want, tolerance = expected_gradient(turned, tokens, entropy=torch.ones(500, device='cuda'))
    close(base.grad.t()[:500], want, tolerance)
    # rows repeated by expand: their gradients add up
    base.grad = None
    row = base[:1].expand(9, -1)
    tokens = tokens_of(9, 1031)
    token_log_probs(row, tokens).log_probs.sum().backward()
    want, tolerance = expected_gradient(row, tokens, given=torch.ones(9, device='cuda'))
    # torch adds the nine rows, rounding each partial sum to the type at most
    close(base.grad[0], want.sum(0), tolerance.sum(0) + 9 * torch.finfo(dtype).eps * want.abs().sum(0))


def test_gradient_against_differences():
    """Central differences along a direction: f is smooth, the step's error is h^2 / 6 of the third derivative (below 10
    for directions of length 1) and 2 f's FP32 error / 2h."""
    from bdm_amd import token_log_probs
    logits, tokens = logits_of(4, 777, FP32).requires_grad_(), tokens_of(4, 777)
    weights = [torch.randn(4, device='cuda') for _ in range(2)]

    def f(x):
        out = token_log_probs(x, tokens)
        return (out.log_probs.double() * weights[0]).sum() + (out.entropy.double() * weights[1]).sum()

    grad, = torch.autograd.grad(f(logits), [logits])
    h = 2.0 ** -5
    for seed in range(4):
        direction = logits_of(4, 777, FP32, 20 + seed)
        direction = direction / direction.norm()
        with torch.no_grad():
            slope = (f(logits + h * direction) - f(logits - h * direction)) / (2 * h)
        size = sum(float(w.abs().sum()) for w in weights)
        noise = size * (2 * CHAIN * STEP * 10) / (2 * h) + 10 * h * h / 6
        assert abs(float(slope - (grad.double() * direction).sum())) <= noise


def test_second_gradient():
    """create_graph runs the backward in torch ops: the same first gradient, and the second one's formula."""
    from bdm_amd import token_log_probs
    logits, tokens = logits_of(3, 40, FP32).requires_grad_(), tokens_of(3, 40)
    plain, = torch.autograd.grad(token_log_probs(logits, tokens).log_probs.sum(), [logits])
    grad, = torch.autograd.grad(token_log_probs(logits, tokens).log_probs.sum(), [logits], create_graph=True)
    close(grad, plain.double(), 4 * CHAIN * STEP * (plain.abs() + 1e-3).double())
    v = torch.randn(3, 40, device='cuda')
    second, = torch.autograd.grad((grad * v).sum(), [logits])
    _, p, *_ = distribution(logits)
    want = -p * (v.double() - (p * v).sum(-1, keepdim=True))
    close(second, want, 8 * CHAIN * STEP * (p * (v.abs() + (p * v.abs()).sum(-1, keepdim=True))) + 1e-9)


# ------------------------------------------------------------------ the loss

@pytest.mark.parametrize('dtype', [BF16, FP32])
@pytest.mark.parametrize('rows,vocab', [(1, 192), (2, 1), (33, 192), (1000, 4099), (257, 50257), (4100, 192)])
def test_loss(rows, vocab, dtype):
    from bdm_amd import token_loss
    logits, tokens = logits_of(rows, vocab, dtype).requires_grad_(), tokens_of(rows, vocab)
    tokens[1::5] = -100
    loss = token_loss(logits, tokens)
    loss.backward(torch.tensor(1.7, device='cuda'))
    counted = tokens != -100
    want = expected_scores(logits, tokens)['log_probs']
    mean = -want[0].sum() / counted.sum()
    close(loss, mean, want[1].max() + 2 * STEP * mean.abs())
    each = torch.full((rows,), -1.7, device='cuda', dtype=torch.float64) / counted.sum()
    close(logits.grad, *expected_gradient(logits, tokens, given=each))
    with torch.no_grad():
        assert torch.equal(token_loss(logits, tokens), loss.detach())
    reference = torch.nn.functional.cross_entropy(logits.detach().double(), tokens)
    close(loss, reference, want[1].max() + 2 * STEP * mean.abs())


def test_loss_without_tokens():
    from bdm_amd import token_loss
    logits = logits_of(5, 192, FP32).requires_grad_()
    loss = token_loss(logits, torch.full((5,), -100, device='cuda'))
    assert torch.isnan(loss)
    loss.backward()
    assert (logits.grad == 0).all()


def test_loss_of_shaped_tokens():
    from bdm_amd import token_loss
    logits, tokens = logits_of(24, 300, BF16), tokens_of(24, 300)
    whole = token_loss(logits, tokens)
    assert torch.equal(token_loss(logits.view(2, 3, 4, 300), tokens.view(2, 3, 4)), whole)


# ------------------------------------------------------------------ use

def test_rows_beyond_32_bits():
    """Offsets past 2^31 elements, in both directions."""
    from bdm_amd import token_log_probs
    rows, vocab = 65600, 32771
    logits = torch.zeros(rows, vocab, device='cuda', dtype=BF16)
    logits[-3:] = logits_of(3, vocab, BF16)
    logits.requires_grad_()
    tokens = tokens_of(rows, vocab)
    out = token_log_probs(logits, tokens, alternatives=3)
    check(logits.detach()[-3:], tokens[-3:], 3, out=type(out)(*(t[-3:] for t in out)))
    grad, = torch.autograd.grad(out.log_probs.sum(), [logits])
    close(grad[-3:], *expected_gradient(logits.detach()[-3:], tokens[-3:], given=torch.ones(3, device='cuda')))


def test_widest_vocabularies():
    """Joins of many parts: level lists in every part, whose bounds admit more candidates than fit, and the largest size."""
    from bdm_amd import ops
    vocab = 64 * 16384
    logits = logits_of(2, 16384, FP32).repeat(1, 64)
    for k in (1, 31, 32):
        check(logits, tokens_of(2, vocab), k)
    logits = logits_of(1, 1 << 24, BF16)
    check(logits, tokens_of(1, 1 << 24))
    check(logits, tokens_of(1, 1 << 24), 32)
    check(torch.zeros_like(logits), tokens_of(1, 1 << 24), 32)
    with pytest.raises(NotImplementedError):
        ops.token_statistics(torch.zeros(1, (1 << 24) + 1, device='cuda', dtype=BF16), tokens_of(1, 5))


def test_repeats_and_streams():
    """The same call gives the same bits, on any stream and beside another call."""
    from bdm_amd import token_log_probs
    logits, tokens = logits_of(300, 50257, BF16), tokens_of(300, 50257)
    wide = logits_of(3, 262144, FP32)
    first = token_log_probs(logits, tokens, alternatives=8)
    other = token_log_probs(wide, tokens[:3], alternatives=8)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(a):
            one = token_log_probs(logits, tokens, alternatives=8)
            three = token_log_probs(wide, tokens[:3], alternatives=8)
        with torch.cuda.stream(b):
            two = token_log_probs(logits, tokens, alternatives=8)
            four = token_log_probs(wide, tokens[:3], alternatives=8)
        torch.cuda.synchronize()
        for got, want in ((one, first), (two, first), (three, other), (four, other)):
            assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize('vocab', [192, 50257, 131075])
def test_captured(vocab):
    """Scores, the loss and its gradient in two graphs, replayed in turn with new inputs and eager calls between."""
    from bdm_amd import ops, token_log_probs
    rows = 33
    graphs = []
    for g in range(2):
        logits, tokens = logits_of(rows, vocab, BF16, g), tokens_of(rows, vocab, g)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())

        def work(logits=logits, tokens=tokens):
            scores = ops.token_statistics(logits, tokens, alternatives=6, stats=True)
            loss, inverse = ops.token_loss_mean(scores[0], tokens)
            grad = ops.token_gradient(logits, tokens, scores[4], grad_loss=torch.ones_like(loss), inverse_count=inverse)
            return (*scores, loss, grad)

        with torch.cuda.stream(side):
            work()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = work()
        torch.cuda.current_stream().wait_stream(side)
        graphs.append((graph, logits, tokens, out, work))
    for turn in range(4):
        for graph, logits, tokens, out, work in graphs:
            logits.copy_(logits_of(rows, vocab, BF16, 50 + turn))
            tokens.copy_(tokens_of(rows, vocab, 60 + turn))
        for graph, *_ in graphs:
            graph.replay()
        for _, logits, tokens, out, work in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, work()))
        torch.cuda.synchronize()


def test_order_oracle():
    """The oracle's own order: NaN, descending, lower index."""
    x = torch.tensor([[0.0, torch.nan, 2.0, -0.0, torch.inf, 2.0, torch.nan]], device='cuda')
    assert order(x, 7).tolist() == [[1, 6, 4, 2, 5, 0, 3]]
