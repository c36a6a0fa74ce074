"""Formulas in 64 bits, and how far FP32 kernels may be from them.

A sum of FP32 numbers in chains of at most k additions is off by at most
k * 2^-24 of the sum of their magnitudes; rounding to a type by at most half a
step, finfo.eps / 2 of the value.  The chains here: a lane's own values and the
tree over lanes and waves (CHAIN), rows of one part and the parts' sums (ROWS).
"""

import torch

STEP = 2.0 ** -24
CHAIN = 128    # at most 96 values a lane, 6 steps over the lanes, 16 waves, a few joined parts, and the exponentials' error
ROWS = 512


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tolerance, what=''):
    """Every value within its tolerance; infinities and NaN in the same places."""
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, what
    tolerance = torch.as_tensor(tolerance, device=want.device, dtype=torch.float64).expand_as(want)
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)]), what
    error = (got - want).abs()[finite] - tolerance[finite]
    assert error.numel() == 0 or float(error.max()) <= 0, (what, float(error.max()),
                                                         float((got - want).abs()[finite].max()))


# ------------------------------------------------------------------ tokens

def distribution(logits):
    """(log p, p, m, log s, entropy) of rows in 64 bits; an empty row has log p = -inf, p = 0, entropy 0."""
    x = logits.detach().double()
    high = x.amax(-1, keepdim=True)
    high = torch.where(high == -torch.inf, 0.0, high)
    e = (x - high).exp()
    total = e.sum(-1, keepdim=True)
    empty = total == 0
    logs = torch.where(empty, -torch.inf, x - high - total.log())
    p = torch.where(empty, 0.0, e / total)
    # 0 log 0 = 0, but a NaN row stays NaN
    entropy = -torch.where(p == 0, 0.0, p * logs).sum(-1)
    return logs, p, high, total.log(), entropy


def order(logits, k):
    """The k best of each row: a NaN first, then descending, equal ones by the lower index."""
    x = logits.detach().double() + 0.0
    x = torch.where(torch.isnan(x), torch.inf, x)
    first = torch.isnan(logits)
    # stable sorts, the less important key first
    by_value = x.sort(dim=-1, descending=True, stable=True).indices
    by_nan = first.gather(-1, by_value).int().sort(dim=-1, descending=True, stable=True).indices
    return by_value.gather(-1, by_nan)[..., :k]


def expected_scores(logits, tokens, alternatives=0, ignore_index=-100):
    """{name: (value, tolerance)} of token_log_probs in 64 bits."""
    logs, p, high, log_sum, entropy = distribution(logits)
    vocab = logits.shape[-1]
    outside = (tokens < 0) | (tokens >= vocab)
    given = logs.gather(-1, torch.where(outside, 0, tokens).unsqueeze(-1)).squeeze(-1)
    given = torch.where(tokens == ignore_index, 0.0, torch.where(outside, torch.nan, given))
    spread = torch.where(p == 0, 0.0, p * (logs + log_sum).abs()).sum(-1)  # sum p |x - m|
    out = dict(log_probs=(given, CHAIN * STEP + 4 * STEP * given.abs()),
               entropy=(entropy, 2 * CHAIN * STEP * (1 + spread) + 4 * STEP * log_sum.squeeze(-1).abs()))
    if alternatives:
        best = order(logits, alternatives)
        top = logs.gather(-1, best)
        out.update(top_log_probs=(top, CHAIN * STEP + 4 * STEP * top.abs()), top_tokens=best)
    return out


def expected_gradient(logits, tokens, top_tokens=None, *, given=None, entropy=None, top=None, ignore_index=-100):
    """(gradient, tolerance) of the logits in 64 bits."""
    logs, p, _, _, h = distribution(logits)
    vocab = logits.shape[-1]
    zero = torch.zeros(tokens.shape, device=logits.device, dtype=torch.float64)
    a = zero if given is None else given.double()
    outside = (tokens < 0) | (tokens >= vocab)
    a = torch.where(tokens == ignore_index, 0.0, torch.where(outside & (given is not None), torch.nan, a))
    b = zero if entropy is None else entropy.double()
    total = a + (0.0 if top is None else top.double().sum(-1))
    magnitude = a.abs() + (0.0 if top is None else top.double().abs().sum(-1))
    lifted = torch.where(p == 0, 0.0, logs + h.unsqueeze(-1))
    grad = -p * (total.unsqueeze(-1) + b.unsqueeze(-1) * lifted)
    # p's relative error: that of its exponent, of log s and the exponential's own; and the entropy's
    relative = CHAIN * STEP + 4 * STEP * torch.where(p == 0, 0.0, logs.abs())
    size = magnitude.unsqueeze(-1) + b.abs().unsqueeze(-1) * (lifted.abs() + 2 * h.unsqueeze(-1) + 2)
    tolerance = 2 * relative * p * size
    empty = (p == 0).all(-1, keepdim=True)
    spot = torch.zeros_like(grad)
    spot.scatter_add_(-1, torch.where(outside, 0, tokens).unsqueeze(-1), torch.where(outside, 0.0, a).unsqueeze(-1))
    if top is not None:
        spot.scatter_add_(-1, top_tokens, top.double())
    weight = torch.zeros_like(grad).scatter_add_(-1, torch.where(outside, 0, tokens).unsqueeze(-1), a.abs().unsqueeze(-1))
    if top is not None:
        weight.scatter_add_(-1, top_tokens, top.double().abs())
    grad = torch.where(empty, 0.0, grad + spot)
    return grad, tolerance + 40 * STEP * weight.nan_to_num() + half_step(logits.dtype) * 1.01 * grad.abs() + 1e-37


# ------------------------------------------------------------------ layer norm

def expected_norm(x, weight, bias, eps, residual=None, grad=None, grad_sum=None):
    """{name: (value, tolerance)} of a layer norm and, with ``grad``, its gradients in 64 bits."""
    dtype, out = x.dtype, {}
    x = x.detach().double()
    if residual is not None:
        x = x + residual.detach().double()
        out['total'] = (x, half_step(dtype) * x.abs() * 1.01)
        x = x.to(dtype).double()
    width = x.shape[-1]
    w = torch.ones(width, device=x.device, dtype=torch.float64) if weight is None else weight.detach().double()
    b = torch.zeros_like(w) if bias is None else bias.detach().double()
    mean = x.mean(-1, keepdim=True)
    r = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * r
    y = xh * w + b
    # the centred value's error: the mean's and its own rounding, in units of the row's deviation
    off = r * x.abs().mean(-1, keepdim=True)
    slack = CHAIN * STEP
    dxh = slack * (xh.abs() + off)
    out['y'] = (y, dxh * w.abs() + 4 * STEP * (xh * w).abs() + 2 * STEP * b.abs() + half_step(dtype) * 1.01 * y.abs())
    if grad is None:
        return out
    dy = grad.detach().double()
    g = dy * w
    plain, dot = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = r * (g - plain - xh * dot)
    size = xh.abs() + off
    tolerance = r * 4 * slack * (g.abs() + g.abs().mean(-1, keepdim=True) + size * (g.abs() * size).mean(-1, keepdim=True))
    if grad_sum is not None:
        dx = dx + grad_sum.detach().double()
        tolerance = tolerance + 2 * STEP * grad_sum.detach().double().abs()
    out['dx'] = (dx, tolerance + half_step(dtype) * 1.01 * dx.abs())
    param = dtype if weight is None and bias is None else (bias if weight is None else weight).dtype

    def over_rows(t):
        return t.reshape(-1, width).sum(0)

    dw, db = over_rows(dy * xh), over_rows(dy)
    out['dw'] = (dw, (slack * 2 + ROWS * STEP) * over_rows(dy.abs() * size) + half_step(param) * 1.01 * dw.abs())
    out['db'] = (db, ROWS * STEP * over_rows(dy.abs()) + half_step(param) * 1.01 * db.abs())
    return out
