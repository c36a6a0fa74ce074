"""Beam search's selection and the reordering of dense caches against plain
restatements in 64 bits, at the sizes, layouts and masks where they can go
wrong.

Tolerance of a score: the kernel's sum of exponentials is FP32.  A thread adds
at most 33 exponentials, a wave's lanes join in 6 steps and four waves in 4
additions; an exponential is off by a few units of the last place (its exponent
relative to the maximum, whose error its own smallness outweighs).  That is at
most 60 roundings of 2^-24 relative to the sum, so 60 * 2^-24 in its logarithm;
the score itself is rounded once.  Tokens and parents have to be the exact ones,
except where candidates of two beams are nearer to each other than that.
Two of one beam differ by their logits' difference exactly, but s + (x - l) in 64
bits is rounded twice, each time by 2^-53 of |s + x - l| at most (s and x - l are
not positive here), and the division by a length once: where different logits are
nearer than four to six such roundings, 2^-50 of the total, the restatement
cannot tell them apart, and either is taken.  Equal logits go to the lower token.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

LOG_SUM = 60 * 2.0 ** -24


def reference(logits, scores, width, finished=None, eos=None, lengths=None, penalty=0.0):
    """Totals [B, K*V] and compared values [B, K*V] in 64 bits on the CPU."""
    x = logits.double().cpu()
    score = scores.double().cpu()
    live = torch.isfinite(score) & ~torch.isnan(x).any(-1) & ~(x == math.inf).any(-1) & (x > -math.inf).any(-1)
    lse = torch.logsumexp(torch.where(live[..., None], x, torch.zeros_like(x)), -1, keepdim=True)
    total = torch.where(live[..., None], score[..., None] + (x - lse), torch.full_like(x, -math.inf))
    grown = torch.ones_like(score)
    if finished is not None:
        finished = finished.cpu()
        grown = (~finished).double()
        own = torch.full_like(x, -math.inf)
        own[..., eos] = torch.where(torch.isfinite(score), score, torch.full_like(score, -math.inf))
        total = torch.where(finished[..., None], own, total)
    compared = total
    if penalty:
        compared = total / (lengths.cpu().double() + grown)[..., None].pow(penalty)
        compared = torch.where(torch.isfinite(compared), compared, torch.full_like(compared, -math.inf))
    return total.flatten(1), compared.flatten(1)


def check(logits, scores, width, **options):
    from bdm_amd import ops
    print('CASE beam', tuple(logits.shape), logits.dtype, logits.stride(), width,
          {k: v for k, v in options.items() if not torch.is_tensor(v)}, flush=True)
    out = ops.beam_select(logits, scores, width=width, **options)
    torch.cuda.synchronize()
    finished, eos, lengths = options.get('finished'), options.get('eos'), options.get('lengths')
    total, compared = reference(logits, scores, width, finished, eos, lengths, options.get('length_penalty', 0.0))
    batch, beams, vocab = logits.shape
    order = compared.sort(dim=-1, descending=True, stable=True).indices[:, :width]
    parents, tokens = out.parents.cpu(), out.tokens.cpu()
    base = torch.arange(batch)[:, None] * beams
    place = (parents - base) * vocab + tokens
    assert ((parents >= base) & (parents < base + beams) & (tokens >= 0) & (tokens < vocab)).all()
    for b in range(batch):
        assert len(set(place[b].tolist())) == width, 'a continuation twice'
        for i in range(width):
            mine, best = int(place[b, i]), int(order[b, i])
            if mine != best:
                a, c = float(compared[b, mine]), float(compared[b, best])
                if mine // vocab != best // vocab:
                    assert abs(a - c) <= 2 * LOG_SUM + abs(c) * 2.0 ** -50, (b, i, a, c)
                else:
                    x, y = (float(logits[b, at // vocab, at % vocab]) for at in (mine, best))
                    near = abs(float(total[b, best])) * 2.0 ** -50
                    assert x != y and abs(x - y) <= near and abs(a - c) <= abs(c) * 2.0 ** -50, (b, i, a, c, x, y)
    want = total.gather(1, place)
    want = torch.where(torch.isfinite(compared.gather(1, place)), want, torch.full_like(want, -math.inf))
    got = out.scores.cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and not torch.isnan(got).any()
    fine = torch.isfinite(want)
    assert ((got - want)[fine].abs() <= LOG_SUM + want[fine].abs() * 2.0 ** -24).all()
    flat = parents.flatten()
    if eos is not None:
        ended = finished.cpu().flatten()[flat] if finished is not None else torch.zeros_like(flat, dtype=torch.bool)
        assert torch.equal(out.finished.cpu().flatten(), ended | (tokens.flatten() == eos))
    else:
        assert out.finished is None
    if lengths is not None:
        grown = ~finished.cpu().flatten()[flat] if finished is not None else torch.ones_like(flat, dtype=torch.bool)
        assert torch.equal(out.lengths.cpu().flatten(), lengths.cpu().flatten()[flat] + grown.int())
    return out


def inputs(device, batch, beams, vocab, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(batch, beams, vocab, generator=gen) * 2.5).to(dtype).to(device)
    scores = (-20 - 4 * torch.rand(batch, beams, generator=gen)).to(device)
    return logits, scores, gen


SIZES = [
    # batch, beams, vocabulary, width
    (1, 1, 1, 1), (2, 3, 7, 5), (1, 1, 5, 5), (1, 4, 192, 4), (3, 5, 513, 7), (2, 16, 2048, 16), (2, 16, 2047, 64),
    (2, 17, 2048, 3), (1, 64, 100, 64), (2, 8, 2049, 8), (1, 2, 50257, 64), (3, 3, 16389, 1), (70, 4, 8192, 4),
    (0, 4, 192, 4),
]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('size', SIZES, ids=lambda s: 'x'.join(map(str, s)))
def test_select_sizes(device, size, dtype):
    batch, beams, vocab, width = size
    logits, scores, _ = inputs(device, batch, beams, vocab, dtype, sum(size))
    check(logits, scores, width)


@pytest.mark.parametrize('vocab', [192, 4099])
@pytest.mark.parametrize('penalty', [0.0, 0.7, -0.5])
def test_select_ended_beams_and_lengths(device, vocab, penalty):
    logits, scores, gen = inputs(device, 4, 6, vocab, torch.bfloat16, vocab)
    finished = (torch.rand(4, 6, generator=gen) < 0.4)
    finished[1] = True   # nothing but ended beams: fewer candidates than places
    finished[2] = False
    lengths = torch.randint(1, 30, (4, 6), generator=gen, dtype=torch.int32).to(device)
    check(logits, scores, 6, finished=finished.to(device), eos=vocab - 1, lengths=lengths, length_penalty=penalty)
    check(logits, scores, 6, eos=3)
    # an ended beam's score beside live ones that are near it
    check(logits, scores * 0.01 - 0.5, 6, finished=finished.to(device), eos=0, lengths=lengths, length_penalty=penalty)


@pytest.mark.parametrize('vocab', [192, 2048, 20000])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_select_masked_rows(device, vocab, dtype):
    logits, scores, gen = inputs(device, 8, 3, vocab, dtype, vocab + 1)
    logits[0] = -math.inf                       # nothing anywhere
    logits[1, :, 2:] = -math.inf                # two tokens a beam
    logits[2, 0] = -math.inf                    # one empty row among others
    logits[3, 1, vocab // 2] = math.nan         # a row that holds a NaN
    logits[4, 2, vocab - 1] = math.inf          # and one with +inf
    logits[5, :, ::2] = -math.inf
    logits[6, 0] = torch.finfo(dtype).min       # a mask of the lowest value: a uniform row
    scores[7, 0] = -math.inf                    # a beam that does not exist
    scores[7, 1] = math.nan
    check(logits, scores, 8)
    logits[:] = -math.inf
    logits[:, 1, vocab - 1] = 0.0
    check(logits, scores, 3)


@pytest.mark.parametrize('vocab', [1500, 12000, 50257])
def test_select_contiguous_masks(device, vocab):
    # the lowest value, zero and huge values in blocks, so that some lanes hold nothing else
    logits, scores, _ = inputs(device, 4, 6, vocab, torch.float32, vocab + 2)
    logits[0, :, : vocab // 2] = torch.finfo(torch.float32).min
    logits[1, :, vocab // 3:] = -math.inf
    logits[2, :, : vocab // 2] = -0.0
    logits[2, :, vocab // 2: vocab // 2 + 40] = 0.0
    logits[3, 2, 7] = 3e38
    logits[3, 3] = -torch.rand(vocab, device=device) * 1e-30
    check(logits, scores, 12)
    check(logits.bfloat16(), scores, 12)


JOINS = [
    # batch, beams, vocabulary, width: each with more listed values than a workgroup's threads keep
    (1, 16, 50257, 64), (1, 64, 50257, 12), (5, 64, 9000, 64), (9, 16, 50257, 50),
]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('size', JOINS, ids=lambda s: 'x'.join(map(str, s)))
def test_select_joins_many_lists(device, size, dtype):
    batch, beams, vocab, width = size
    logits, scores, gen = inputs(device, batch, beams, vocab, dtype, sum(size))
    check(logits, scores, width)
    finished = torch.rand(batch, beams, generator=gen) < 0.3
    lengths = torch.randint(1, 30, (batch, beams), generator=gen, dtype=torch.int32).to(device)
    check(logits, scores, width, finished=finished.to(device), eos=11, lengths=lengths, length_penalty=0.8)


@pytest.mark.parametrize('size', [(2, 8, 1000, 8), (2, 16, 50257, 16), (1, 16, 50257, 64), (2, 64, 9000, 48),
                                  (1, 64, 131072, 8)],
                         ids=lambda s: 'x'.join(map(str, s)))
def test_select_one_beam_has_all_the_best(device, size):
    # every other beam is far behind, or level with it in all its values: first few candidates near the bound, then
    # more of them than are ranked at once, then more than are kept
    batch, beams, vocab, width = size
    logits, scores, _ = inputs(device, batch, beams, vocab, torch.float32, sum(size) + 1)
    ahead = scores - 300
    ahead[:, beams // 2] += 290
    check(logits, ahead, width)
    check(logits[:, :1].expand(-1, beams, -1), scores[:, :1].expand(-1, beams).contiguous(), width)
    flat = torch.zeros_like(logits)
    check(flat, scores[:, :1].expand(-1, beams).contiguous(), width)
    near = flat.clone()
    near[..., : 3 * width] = 1.0
    finished = torch.zeros(batch, beams, dtype=torch.bool, device=device)
    finished[:, beams // 3] = True
    level = scores[:, :1].expand(-1, beams).contiguous()
    level[:, beams // 3] -= math.log(vocab)
    lengths = torch.full((batch, beams), 9, dtype=torch.int32, device=device)
    check(near, level, width, finished=finished, eos=5, lengths=lengths, length_penalty=0.7)


@pytest.mark.parametrize('vocab', [100, 2048, 2049, 30001])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_select_ties(device, vocab, dtype):
    """Equal logits by the thousand: more at the bound than LDS holds."""
    logits, scores, gen = inputs(device, 2, 3, vocab, dtype, vocab + 2)
    logits[0] = 1.25
    logits[1] = torch.randint(0, 3, (3, vocab), generator=gen).to(dtype).to(device)
    logits[1, 1, 5::7] = -0.0
    check(logits, scores, 64)
    scores[:] = -3.0          # and between the beams
    logits[:] = 0.5
    check(logits, scores, 64)
    logits[0, 2, vocab - 1] = 0.75
    check(logits, scores, 64)


def test_select_one_lane_holds_the_best(device):
    """The best logits side by side, so that few lanes hold them all."""
    logits, scores, _ = inputs(device, 1, 2, 40000, torch.float32, 9)
    logits[0, 0, 8000:8064] += 40
    logits[0, 1, 39990:] += 30
    check(logits, scores, 64)


def test_select_layouts(device):
    wide, scores, gen = inputs(device, 6, 4, 5000, torch.bfloat16, 11)
    flat = wide.flatten()
    check(wide[:, :, 3:4001], scores, 4)                       # rows that start anywhere
    check(wide[::2, 1:4], scores[::2, 1:4], 3)                 # strided batch and beams
    check(wide[:, :, :300][:, 1::2], scores[:, ::2], 2)
    check(flat[1:1 + 2 * 4 * 5000].view(2, 4, 5000), scores[:2], 4)
    check(wide.transpose(1, 2)[:, :4], scores.new_zeros(6, 4), 4)  # last dimension not contiguous
    check(wide[:, :1].expand(6, 4, 5000), scores, 4)
    check(wide, scores.t().contiguous().t(), 4)


def test_select_on_a_side_stream_and_in_a_graph(device):
    from bdm_amd import ops
    logits, scores, _ = inputs(device, 8, 8, 9001, torch.bfloat16, 13)
    want = ops.beam_select(logits, scores)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.beam_select(logits, scores)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want[:3], got[:3]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.beam_select(logits, scores)
    for seed in range(3):
        other, more, _ = inputs(device, 8, 8, 9001, torch.bfloat16, 20 + seed)
        logits.copy_(other)
        scores.copy_(more)
        graph.replay()
        want = ops.beam_select(other, more)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want[:3], out[:3]))


def test_two_selections_at_once_and_two_graphs(device):
    from bdm_amd import ops
    given = [inputs(device, 6, 5, 20011, torch.float32, 40 + i)[:2] for i in range(2)]
    want = [ops.beam_select(*g) for g in given]
    sides = [torch.cuda.Stream() for _ in given]
    got = []
    for _ in range(20):
        for side, g in zip(sides, given):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append(ops.beam_select(*g))
    graphs, outs = [], []
    torch.cuda.synchronize()
    for g in given:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.beam_select(*g))
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for n, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(want[n % 2][:3], out[:3]))
    for a, b in zip(want, outs):
        assert all(torch.equal(x, y) for x, y in zip(a[:3], b[:3]))


@pytest.mark.parametrize('vocab', [256, 700, 1024, 5000])
def test_select_around_zero(device, vocab):
    # many rows whose best values lie on both sides of zero, and rows with little else than zeros
    logits, scores, gen = inputs(device, 64, 8, vocab, torch.bfloat16, vocab + 3)
    check(logits - 2, scores, 8)
    logits[32:] = torch.where((torch.rand(32, 8, vocab, generator=gen) < 0.97).to(device), 0, logits[32:] * 1e-20)
    check(logits, scores, 8)


REORDER = [
    # prompts, beams, row shape, dtype
    (1, 1, (4, 8), torch.float32), (1, 4, (1024, 4, 128), torch.bfloat16), (3, 5, (7, 3, 5, 9), torch.bfloat16),
    (2, 8, (16, 8, 128), torch.bfloat16), (2, 16, (33,), torch.float32), (1, 32, (1000,), torch.bfloat16),
    (2, 33, (129, 2), torch.float32), (1, 64, (4096,), torch.bfloat16), (4, 3, (11,), torch.uint8), (2, 2, (), torch.int64),
    (2, 4, (0, 3), torch.float32),
]


@pytest.mark.parametrize('case', REORDER, ids=lambda c: f'{c[0]}x{c[1]}x{c[2]}')
def test_reorder(device, case):
    from bdm_amd import ops
    prompts, beams, shape, dtype = case
    print('CASE reorder', case, flush=True)
    gen = torch.Generator().manual_seed(prompts * 100 + beams)
    rows = prompts * beams
    states = [torch.randint(0, 100, (rows, *shape), generator=gen).to(dtype).to(device) for _ in range(3)]
    states.append(torch.randn(rows, 6, generator=gen).to(device))
    base = torch.arange(rows) // beams * beams
    choices = [torch.randint(0, beams, (rows,), generator=gen) + base, torch.arange(rows), base,
               base + beams - 1 - torch.arange(rows) % beams]
    for parents in choices:
        want = [t.cpu()[parents] for t in states]
        ops.reorder_states(states, parents.to(device).view(prompts, beams), beams=beams)
        torch.cuda.synchronize()
        for t, w in zip(states, want):
            assert torch.equal(t.cpu(), w)


def test_reorder_of_many_tensors_and_in_a_graph(device):
    from bdm_amd import ops
    states = [torch.randn(8, 10 + i, device=device) for i in range(70)]  # more than one launch
    parents = torch.tensor([1, 1, 3, 2, 7, 4, 4, 6], device=device)
    want = [t[parents] for t in states]
    ops.reorder_states(states, parents, beams=4)
    assert all(torch.equal(a, b) for a, b in zip(states, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.reorder_states(states, parents, beams=4)
    for i in range(3):
        parents.copy_(torch.tensor([i, 0, 1, 2, 4, 5 + i % 3, 5, 6]))
        want = [t[parents] for t in states]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_reorder_clamps_parents_into_their_group(device):
    from bdm_amd import ops
    state = torch.arange(8, device=device).view(8, 1).clone()
    ops.reorder_states([state], torch.tensor([-5, 9, 2, 1, 99, 0, 5, 6], device=device), beams=4)
    assert state.flatten().tolist() == [0, 3, 2, 1, 7, 4, 5, 6]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('first', [0, 1], ids=['first-beam', 'second-beam'])
def test_select_joins_lists_whose_best_has_a_late_place(device, first, dtype):
    # more candidates level with each other than LDS holds, in lists whose first entries are not their lowest tokens: a
    # logit of 1e-20 leads its part of the row but has the total of the zeros
    vocab, width = 9000, 64
    logits = torch.zeros(1, 64, vocab, device=device, dtype=dtype)
    logits[..., 2047::2048] = 1e-20
    logits[..., -1] = 1e-20
    logits[..., :2008] = -math.inf
    logits[:, :first] = -math.inf
    scores = torch.full((1, 64), -3.0, device=device)
    out = check(logits, scores, width)
    assert torch.isfinite(out.scores).all()
    # totals that are equal in 64 bits go to the lower token, of the lowest beam that has any
    assert (out.parents == first).all()
    assert torch.equal(out.tokens.cpu(), torch.arange(2008, 2008 + width)[None])
    for _ in range(3):
        again = check(logits, scores, width)
        assert all(torch.equal(a, b) for a, b in zip(out[:3], again[:3]))


def places(out, beams, vocab):
    base = torch.arange(out.parents.shape[0])[:, None] * beams
    return (out.parents.cpu() - base) * vocab + out.tokens.cpu()


EQUAL = [
    # batch, beams, vocabulary, width: one launch and two, rows that start at every offset from a vector's boundary, beams
    # times vocabulary around a power of two, more lists than threads keep
    (3, 4, 193, 4), (2, 16, 2047, 16), (2, 8, 2049, 8), (2, 5, 5001, 16), (1, 64, 1023, 64), (1, 64, 1024, 64),
    (1, 64, 1025, 64), (1, 64, 9003, 64), (1, 16, 50257, 64),
]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('size', EQUAL, ids=lambda s: 'x'.join(map(str, s)))
def test_select_beams_that_are_equal(device, size, dtype):
    # equal rows and scores have equal totals, wherever a row starts in memory: the lower beam, then the lower token
    from bdm_amd import ops
    batch, beams, vocab, width = size
    print('CASE equal beams', size, dtype, flush=True)
    gen = torch.Generator().manual_seed(sum(size))
    for kind in range(4):
        rows = torch.randn(batch, 1, vocab, generator=gen) * 2.5
        if kind == 1:
            rows = torch.randint(0, 3, rows.shape, generator=gen).float()
        elif kind > 1:
            rows = torch.zeros_like(rows)
        rows = rows.to(dtype).to(device)
        scores = torch.full((batch, beams), -20.0, device=device)
        if kind == 3:
            scores[:, :beams // 2] = -math.inf
        first = beams // 2 if kind == 3 else 0
        level = rows.expand(batch, beams - first, vocab).flatten(1).float().cpu()
        want = level.sort(dim=-1, descending=True, stable=True).indices[:, :width] + first * vocab
        spaced = torch.empty(batch, beams, vocab + 3, device=device, dtype=dtype)[..., 2:vocab + 2]
        for logits in (rows.expand(batch, beams, vocab), rows.expand(batch, beams, vocab).contiguous(),
                       spaced.copy_(rows.expand(batch, beams, vocab))):
            out = ops.beam_select(logits, scores, width=width)
            assert torch.equal(places(out, beams, vocab), want), (kind, logits.stride())
            fine = out.scores[:, :min(width, (beams - first) * vocab)]
            assert torch.isfinite(fine).all() and (fine.diff(dim=-1) <= 0).all()


def test_select_a_view_is_its_copy(device):
    from bdm_amd import ops
    wide, scores, _ = inputs(device, 6, 4, 5000, torch.bfloat16, 17)
    for first in range(9):
        view = wide[:, :, first:first + 4001]
        a, b = ops.beam_select(view, scores), ops.beam_select(view.contiguous(), scores)
        assert all(torch.equal(x, y) for x, y in zip(a[:3], b[:3])), first


def test_select_places_beyond_32_bits(device):
    # 64 beams over 2^26 + 3 tokens, one of them live: its best tokens, all level, lie on both sides of place 2^32
    from bdm_amd import ops
    vocab, width = 2 ** 26 + 3, 64
    row = torch.full((1, 1, vocab), -math.inf, dtype=torch.bfloat16, device=device)
    first = 2 ** 32 - 63 * vocab - 40
    row[..., first:] = 0.5
    scores = torch.full((1, 64), -math.inf, device=device)
    scores[:, 63] = -2.0
    print('CASE places beyond 32 bits', flush=True)
    out = ops.beam_select(row.expand(1, 64, vocab), scores, width=width)
    assert (out.parents == 63).all() and torch.isfinite(out.scores).all()
    assert torch.equal(out.tokens.cpu(), torch.arange(first, first + width)[None])


def test_reorder_refuses_shared_memory(device):
    from bdm_amd import ops
    parents = torch.tensor([1, 0, 3, 2], device=device)
    history = torch.arange(12, device=device).view(4, 3) % 4
    before = history.clone()
    for states, rows in (([parents], parents), ([history.view(-1)[:4], history.view(-1)[2:6]], parents),
                         ([history.view(-1)[4:8]], history.view(-1)[7:11])):
        with pytest.raises(ValueError):
            ops.reorder_states(states, rows, beams=2)
    torch.cuda.synchronize()
    assert parents.tolist() == [1, 0, 3, 2] and torch.equal(history, before)
    history[:, 1] = parents
    want = history[parents]
    ops.reorder_states([history], history[:, 1], beams=2)   # a column of a state is copied first
    assert torch.equal(history, want)
