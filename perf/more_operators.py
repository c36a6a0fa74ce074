"""What a training or scoring step of the language model runs besides its
products and memory layers: log-probabilities of given tokens and their loss,
the global norm of the gradients and their clipping, and layer normalization.

``score``   log-probabilities of given tokens, the entropy of their
            distributions and the best alternatives (``token_log_probs``);
``policy``  log-probabilities and entropy, and the gradient of the logits from
            gradients of both (``token_log_probs`` under autograd);
``loss``    the mean negative log-probability of the next tokens, padding left
            out, and the gradient of the logits (``token_loss``);
``norm``    the global norm of a model's gradients (``gradient_norm``);
``clip``    the gradients scaled to a largest norm, into the buffers that the
            optimizer reads (``clip_gradients``);
``layer``   layer normalization without gradients, also behind a residual add
            (``LayerNorm``);
``train``   layer normalization and the gradients of its input, weight and
            bias, also behind a residual add (``LayerNorm``).

``listed`` are sizes of this repository's configurations, benchmark and tests.
``run`` computes each in elementary torch operations, or through the package
where ``own`` is set; ``exact`` restates them in float64.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}
IGNORED = -100  # the token of a padded position
EPS = 1e-5


def listed():
    return [
        # the package's default vocabulary, one decoded token of eight sequences with its best alternatives
        dict(name='score_step', kind='score', rows=8, vocab=192, dtype='bf16', alternatives=4, masked=False),
        # a service of 64 sequences over a large vocabulary: the sampled tokens' log-probabilities with alternatives
        dict(name='score_serving', kind='score', rows=64, vocab=50257, dtype='bf16', alternatives=8, masked=True),
        # the widest vocabulary of the tests, a few FP32 rows: less than a row for each part of the chip
        dict(name='score_wide', kind='score', rows=3, vocab=262144, dtype='fp32', alternatives=20, masked=False),
        # evaluation: eight prompts of 1,024 tokens
        dict(name='score_prompts', kind='score', rows=8192, vocab=50257, dtype='bf16', alternatives=0, masked=False),
        # updates from sampled continuations with an entropy term, FP32 logits, an odd vocabulary
        dict(name='policy_fp32', kind='policy', rows=1023, vocab=32001, dtype='fp32', masked=True),
        # the whole model's training step at 8,192 tokens
        dict(name='loss_model', kind='loss', rows=8192, vocab=50257, dtype='bf16'),
        # the gradients of the package's default model: some hundred small tensors
        dict(name='clip_default', kind='clip', layers=8, dim=128, ffn=512, vocab=192, rows=4, banks=1024, dtype='bf16',
             out='bf16', align=4, norm=3.0),
        # the gradients of the whole model of the benchmark, 16 layers: the norm alone
        dict(name='norm_model', kind='norm', layers=16, dim=2048, ffn=5632, vocab=50257, rows=8, banks=1024,
             dtype='bf16', norm=3.0),
        # a model of 4 such layers: BF16 gradients clipped into the FP32 gradients of the masters
        dict(name='clip_model', kind='clip', layers=4, dim=2048, ffn=5632, vocab=50257, rows=8, banks=1024,
             dtype='bf16', out='fp32', align=4, norm=3.0),
        # one decoded token of 64 sequences: a block's residual add and its normalization
        dict(name='layer_step', kind='layer', rows=64, width=1024, dtype='bf16', residual=True),
        # training on 8 prompts of 4,096 tokens
        dict(name='train_prompts', kind='train', rows=32768, width=1024, dtype='bf16', residual=True),
        # a small FP32 layer of odd width
        dict(name='train_odd_fp32', kind='train', rows=777, width=1001, dtype='fp32', residual=False),
    ]


def _spread(rng, low, high):
    """A size spread over the logarithm of its range, odd or even."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(['score', 'score', 'policy', 'loss', 'norm', 'clip', 'layer', 'train', 'train'])
    dtype = rng.choice(['bf16', 'bf16', 'fp32'])
    if kind in ('score', 'policy', 'loss'):
        vocab = _spread(rng, 64, 262144)
        case = dict(kind=kind, rows=_spread(rng, 1, max(2, min(8192, 200_000_000 // vocab))), vocab=vocab, dtype=dtype)
        if kind == 'score':
            case.update(alternatives=rng.choice([0, rng.randint(1, 8), rng.randint(1, min(32, vocab // 4))]))
        if kind != 'loss':
            case.update(masked=rng.random() < 0.4)
        return case
    if kind in ('norm', 'clip'):
        dim = _spread(rng, 32, 2048)
        case = dict(kind=kind, layers=rng.randint(1, 8), dim=dim, ffn=_spread(rng, 2 * dim, 3 * dim),
                    vocab=_spread(rng, 64, 50257), rows=rng.choice([1, 4, 5, 8]), banks=rng.choice([64, 256, 1024]),
                    dtype=rng.choice(['bf16', 'bf16', 'fp32', 'mixed']), norm=round(rng.uniform(0.2, 5.0), 2))
        while sum(math.prod(s) for s in _shapes(case)) > 200_000_000 and case['layers'] > 1:
            case['layers'] -= 1
        if kind == 'clip':
            case.update(out=rng.choice(['bf16', 'fp32']), align=rng.choice([1, 4, 64]))
        return case
    width = _spread(rng, 16, 16384)
    return dict(kind=kind, rows=_spread(rng, 1, max(2, min(65536, 60_000_000 // width))), width=width, dtype=dtype,
                residual=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------- inputs

def _shapes(c):
    """The parameters' shapes of a model of one head: embedding, head and, for
    each layer, the memory layer's projections, router, gates and factors, the
    feed-forward's three weights and the norms."""
    d, s, ffn, vocab, banks = c['dim'], c['rows'], c['ffn'], c['vocab'], c['banks']
    first = max(f for f in range(1, math.isqrt(banks) + 1) if banks % f == 0)
    route = first + banks // first
    layer = [(1,), (s,), (64, d), (banks * s // 64, d), (d,), (d,), (s, d), (s, d), (d, d), (route, d), (route,),
             (route, d), (route,), (route, d), (route,), (d, d), (s, d), (s, d), (d, d), (d, d), (d,), (d, d), (d,),
             (ffn, d), (ffn, d), (d, ffn), (d,), (d,)]
    return layer * c['layers'] + [(vocab, d), (d,), (vocab, d)]


def _places(c):
    """Where the tensors start in a flat buffer, at multiples of ``align``, and
    its length."""
    starts, length = [], 0
    for shape in _shapes(c):
        starts.append(length)
        length += -(-math.prod(shape) // c['align']) * c['align']
    return starts, length


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device='cuda')
    gen.manual_seed(int(seed) * 1013 + 7)
    kind = c['kind']
    state = dict(case=c)

    def normal(*shape, std=1.0):
        return torch.empty(shape, device='cuda').normal_(0, std, generator=gen)

    def uniform(*shape):
        return torch.empty(shape, device='cuda').uniform_(generator=gen)

    if kind in ('score', 'policy', 'loss'):
        n, v = c['rows'], c['vocab']
        tokens = torch.randint(v, (n,), generator=gen, device='cuda')
        x = normal(n, v, std=2.5)
        # most given tokens are likely ones
        boost = torch.where(uniform(n) < 0.7, 6.0 + normal(n), 0.0)
        x.scatter_add_(1, tokens[:, None], boost[:, None])
        if c.get('masked'):
            # tokens that a grammar or a filter of the sampling rules out; never the given ones
            out = uniform(n, v) < 0.4
            out.scatter_(1, tokens[:, None], False)
            x.masked_fill_(out, -math.inf)
        state['logits'] = x.to(DTYPES[c['dtype']]).requires_grad_(own and kind != 'score')
        if kind == 'loss':
            tokens = torch.where(uniform(n) < 0.1, IGNORED, tokens)
            tokens[0] = 0  # one position at least counts
        state['tokens'] = tokens
        if kind == 'policy':
            state['grad_log_probs'], state['grad_entropy'] = normal(n), torch.full((n,), -0.01, device='cuda')
    elif kind in ('norm', 'clip'):
        shapes = _shapes(c)
        total = sum(math.prod(s) for s in shapes)
        types = [torch.float32 if c['dtype'] == 'fp32' or (c['dtype'] == 'mixed' and len(s) == 1) else torch.bfloat16
                 for s in shapes]
        # every tensor's gradients of a size of their own, about `norm` all together
        state['gradients'] = [(normal(*s, std=1.0) * (c['norm'] * total ** -0.5 * math.exp(0.3 * (i % 7 - 3)))).to(t)
                              for i, (s, t) in enumerate(zip(shapes, types))]
        if kind == 'clip':
            # one flat buffer, as an optimizer keeps it
            starts, length = _places(c)
            state['flat'] = torch.zeros(length, device='cuda', dtype=DTYPES[c['out']])
            state['out'] = [state['flat'][i:i + math.prod(s)].view(s) for i, s in zip(starts, shapes)]
    else:
        n, width, dtype = c['rows'], c['width'], DTYPES[c['dtype']]
        # a residual stream: some columns lie far from zero, most rows near it
        x = normal(n, width) + 8 * normal(width) * (uniform(width) < 0.02)
        state['x'] = x.to(dtype)
        state['residual'] = normal(n, width).to(dtype) if c['residual'] else None
        state['weight'] = (1 + 0.2 * normal(width)).to(dtype)
        state['bias'] = (0.2 * normal(width)).to(dtype)
        if kind == 'train':
            state['grad'] = normal(n, width, std=0.1).to(dtype)
            state['grad_total'] = normal(n, width, std=0.1).to(dtype) if c['residual'] else None
        if own:
            from bdm_amd import LayerNorm
            norm = LayerNorm(width, eps=EPS).to(device='cuda', dtype=dtype)
            with torch.no_grad():
                norm.weight.copy_(state['weight'])
                norm.bias.copy_(state['bias'])
            state['module'] = norm
            state['x'].requires_grad_(kind == 'train')
    return state


# ---------------------------------------------------------------------------------------------- plain forms

def _distribution(x):
    """Log-probabilities and probabilities of rows of logits in 32 bits."""
    x = x.float()
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    return x - total.log(), e / total


def _score(s):
    logs, p = _distribution(s['logits'])
    entropy = -torch.where(p > 0, p * logs, 0.0).sum(-1)
    given = logs.gather(1, s['tokens'][:, None])[:, 0]
    if not s['case']['alternatives']:
        return dict(log_probs=given, entropy=entropy)
    best = s['logits'].sort(dim=-1, descending=True, stable=True).indices[:, :s['case']['alternatives']]
    return dict(log_probs=given, entropy=entropy, top_log_probs=logs.gather(1, best), top_tokens=best)


def _policy(s):
    logs, p = _distribution(s['logits'])
    entropy = -torch.where(p > 0, p * logs, 0.0).sum(-1)
    tokens = s['tokens'][:, None]
    by_token, by_entropy = s['grad_log_probs'][:, None], s['grad_entropy'][:, None]
    grad = -p * by_token - torch.where(p > 0, p * (logs + entropy[:, None]), 0.0) * by_entropy
    grad.scatter_add_(1, tokens, by_token)
    return dict(log_probs=logs.gather(1, tokens)[:, 0], entropy=entropy, grad=grad.to(s['logits'].dtype))


def _loss(s):
    logs, p = _distribution(s['logits'])
    counted = s['tokens'] != IGNORED
    tokens = torch.where(counted, s['tokens'], 0)[:, None]
    each = counted.float() / counted.sum()
    loss = -(logs.gather(1, tokens)[:, 0] * each).sum()
    grad = p * each[:, None]
    grad.scatter_add_(1, tokens, -each[:, None])
    return dict(loss=loss, grad=grad.to(s['logits'].dtype))


def _norm(s):
    return torch.stack([g.float().square().sum() for g in s['gradients']]).sum().sqrt()


def _clip(s):
    norm = _norm(s)
    scale = (1.0 / (norm + 1e-6)).clamp(max=1.0)
    for g, out in zip(s['gradients'], s['out']):
        out.copy_(g.float() * scale)
    return [norm, s['flat']]


def _layer(s):
    x, dtype = s['x'], s['x'].dtype
    if s['residual'] is not None:
        x = (x.float() + s['residual'].float()).to(dtype)
    xf = x.float()
    centred = xf - xf.mean(-1, keepdim=True)
    scale = (centred.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xh = centred * scale
    y = (xh * s['weight'].float() + s['bias'].float()).to(dtype)
    if s['case']['kind'] == 'layer':
        return [y] if s['residual'] is None else [x, y]
    dy = s['grad'].float()
    dxh = dy * s['weight'].float()
    dx = (dxh - dxh.mean(-1, keepdim=True) - xh * (dxh * xh).mean(-1, keepdim=True)) * scale
    if s['residual'] is not None:
        dx = dx + s['grad_total'].float()
    grads = [dx.to(dtype), (dy * xh).sum(0).to(dtype), dy.sum(0).to(dtype)]
    return [y, *grads] if s['residual'] is None else [x, y, *grads]


# ---------------------------------------------------------------------------------------------- one pass

def _run_own(s):
    import bdm_amd
    c = s['case']
    kind = c['kind']
    if kind == 'score':
        out = bdm_amd.token_log_probs(s['logits'], s['tokens'], alternatives=c['alternatives'])
        if not c['alternatives']:
            return dict(log_probs=out.log_probs, entropy=out.entropy)
        return dict(log_probs=out.log_probs, entropy=out.entropy, top_log_probs=out.top_log_probs,
                    top_tokens=out.top_tokens)
    if kind == 'policy':
        out = bdm_amd.token_log_probs(s['logits'], s['tokens'])
        grad, = torch.autograd.grad([out.log_probs, out.entropy], [s['logits']],
                                    [s['grad_log_probs'], s['grad_entropy']])
        return dict(log_probs=out.log_probs.detach(), entropy=out.entropy.detach(), grad=grad)
    if kind == 'loss':
        loss = bdm_amd.token_loss(s['logits'], s['tokens'], ignore_index=IGNORED)
        grad, = torch.autograd.grad(loss, [s['logits']])
        return dict(loss=loss.detach(), grad=grad)
    if kind == 'norm':
        return bdm_amd.gradient_norm(s['gradients'])
    if kind == 'clip':
        norm = bdm_amd.clip_gradients(s['gradients'], 1.0, out=s['out'])
        return [norm, s['flat']]
    norm = s['module']
    if kind == 'layer':
        with torch.no_grad():
            return [norm(s['x'])] if s['residual'] is None else list(norm.add_norm(s['x'], s['residual']))
    leaves = [s['x'], norm.weight, norm.bias]
    if s['residual'] is None:
        y = norm(s['x'])
        return [y.detach(), *torch.autograd.grad(y, leaves, s['grad'])]
    total, y = norm.add_norm(s['x'], s['residual'])
    return [total.detach(), y.detach(), *torch.autograd.grad([total, y], leaves, [s['grad_total'], s['grad']])]


_PLAIN = dict(score=_score, policy=_policy, loss=_loss, norm=_norm, clip=_clip, layer=_layer, train=_layer)


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state['case']['kind']](state)


# ---------------------------------------------------------------------------------------------- work and 64 bits

def work(case):
    c = case
    kind = c['kind']
    if kind in ('score', 'policy', 'loss'):
        logits, es = c['rows'] * c['vocab'], DTYPES[c['dtype']].itemsize
        if kind == 'score':
            return dict(bytes=logits * es + c['rows'] * (16 + 12 * c['alternatives']), flops=6 * logits)
        rows = c['rows'] * (24 if kind == 'policy' else 8)
        return dict(bytes=2 * logits * es + rows, flops=(14 if kind == 'policy' else 10) * logits)
    if kind in ('norm', 'clip'):
        shapes = _shapes(c)
        wide = sum(math.prod(s) for s in shapes)
        read = sum(math.prod(s) * (4 if c['dtype'] == 'fp32' or (c['dtype'] == 'mixed' and len(s) == 1) else 2)
                   for s in shapes)
        if kind == 'norm':
            return dict(bytes=read + 4, flops=2 * wide)
        return dict(bytes=read + wide * DTYPES[c['out']].itemsize + 4, flops=3 * wide)
    elements, es = c['rows'] * c['width'], DTYPES[c['dtype']].itemsize
    if kind == 'layer':
        return dict(bytes=(elements * (4 if c['residual'] else 2) + 2 * c['width']) * es, flops=8 * elements)
    return dict(bytes=(elements * (7 if c['residual'] else 4) + 4 * c['width']) * es, flops=20 * elements)


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    kind = c['kind']
    if kind in ('score', 'policy', 'loss'):
        x, tokens = s['logits'].detach().double(), s['tokens']
        logs = torch.log_softmax(x, -1)
        del x
        row = torch.arange(c['rows'], device='cuda')
        if kind == 'loss':
            counted = (tokens != IGNORED).nonzero()[:, 0]
            loss = -logs[counted, tokens[counted]].mean()
            weight = torch.zeros(c['rows'], device='cuda', dtype=torch.float64)
            weight[counted] = 1 / counted.numel()
            grad = logs.exp_().mul_(weight[:, None])
            grad[counted, tokens[counted]] -= weight[counted]
            return dict(loss=loss, grad=grad)
        given = logs[row, tokens]
        p = logs.exp()
        entropy = torch.special.entr(p).sum(-1)
        if kind == 'policy':
            lifted = torch.nan_to_num(logs, neginf=0.0) + entropy[:, None]
            grad = -p * (s['grad_log_probs'].double()[:, None] + s['grad_entropy'].double()[:, None] * lifted)
            grad[row, tokens] += s['grad_log_probs'].double()
            return dict(log_probs=given, entropy=entropy, grad=grad)
        if not c['alternatives']:
            return dict(log_probs=given, entropy=entropy)
        return dict(log_probs=given, entropy=entropy, top_log_probs=logs.topk(c['alternatives'], -1).values,
                    top_tokens=None)
    if kind in ('norm', 'clip'):
        norm = math.sqrt(math.fsum(float(g.double().pow(2).sum()) for g in s['gradients']))
        value = torch.tensor(norm, device='cuda', dtype=torch.float64)
        if kind == 'norm':
            return value
        scale = min(1.0, 1.0 / (norm + 1e-6))
        flat = torch.zeros(s['flat'].numel(), device='cuda', dtype=torch.float64)
        for start, g in zip(_places(c)[0], s['gradients']):
            flat[start:start + g.numel()] = g.double().flatten() * scale
        return [value, flat]
    x = s['x'].detach()
    weight, bias = (s[k].double().requires_grad_(kind == 'train') for k in ('weight', 'bias'))
    total = None
    if s['residual'] is not None:
        total = x.double() + s['residual'].double()
        x = total.to(x.dtype)  # the sum is held in the rows' type
    x = x.double().requires_grad_(kind == 'train')
    y = F.layer_norm(x, (c['width'],), weight, bias, EPS)
    head = [y.detach()] if total is None else [total, y.detach()]
    if kind == 'layer':
        return head
    dx, dw, db = torch.autograd.grad(y, [x, weight, bias], s['grad'].double())
    return [*head, dx if total is None else dx + s['grad_total'].double(), dw, db]
