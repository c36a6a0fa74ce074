"""Beam search and the paged bank cache: what is measured of them.

``select``   one selection of beam search over beams and vocabulary
             (``ops.beam_select``);
``reorder``  the dense caches of several layers put in the order of the chosen
             parents, in place (``ops.reorder_states``);
``step``     one decode token over a paged cache (``BankPages.decode``): of
             beams, behind the fork by their parents, so that the written
             banks are copied on write; or of sequences with banks of their own;
``fork``     the tables of all layers put in the order of the parents
             (``BankPages.fork``);
``load``     prefilled caches copied into pages, banks that equal the initial
             state shared with it, and back (``BankPages.load``, ``dense``);
``turn``     two changes of a service's requests: sequences released, the pool
             compacted, others loaded (``release``, ``compact``, ``load``).

``listed`` are the sizes of this repository's configurations, benchmark and
tests.  ``run`` computes each in elementary torch operations, or through the
package where ``own`` is set; ``exact`` restates them in float64.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


def listed():
    return [
        # the package's default vocabulary, four beams of one prompt: a latency-bound call
        dict(name='select_small', kind='select', batch=1, beams=4, width=4, vocab=192, dtype='bf16', finished=False,
             penalty=0.0),
        # a batch of prompts over a large vocabulary, some beams ended, lengths normalized
        dict(name='select_vocab', kind='select', batch=8, beams=8, width=8, vocab=50257, dtype='bf16', finished=True,
             penalty=0.6),
        # an offline batch with FP32 logits
        dict(name='select_large', kind='select', batch=64, beams=16, width=16, vocab=50257, dtype='fp32',
             finished=True, penalty=0.0),
        # four beams of the package's default geometry, all eight layers
        dict(name='reorder_default', kind='reorder', batch=1, beams=4, tensors=8, heads=1, rows=4, width=128,
             banks=1024, dtype='bf16'),
        # eight prompts of eight beams, four layers of the serving geometry
        dict(name='reorder_batch64', kind='reorder', batch=8, beams=8, tensors=4, heads=8, rows=8, width=128,
             banks=256, dtype='bf16'),
        # a beam search of one prompt at the default geometry, FP32
        dict(name='step_beams_small', kind='step', sequences=4, beams=4, banks=1024, heads=1, rows=4, width=128,
             selected=8, dtype='fp32', pages='fp32', decay=False),
        # eight prompts of eight beams at the serving geometry: every written bank is shared and copied
        dict(name='step_beams_batch64', kind='step', sequences=64, beams=8, banks=256, heads=8, rows=8, width=128,
             selected=8, dtype='bf16', pages='bf16', decay=True),
        # eight sequences of the whole model's layer (one wide head), each with banks of its own
        dict(name='step_wide', kind='step', sequences=8, beams=0, banks=1024, heads=1, rows=8, width=2048, selected=8,
             dtype='bf16', pages='bf16', decay=True),
        # the tables of sixteen layers and 64 beams
        dict(name='fork_layers16', kind='fork', layers=16, sequences=64, beams=8, banks=1024, heads=1, rows=4,
             width=128, pages='bf16'),
        # eight prefilled prompts into pages: 60 % of the banks written, the others those of the initial state
        dict(name='load_prompts', kind='load', sequences=9, take=8, banks=256, heads=8, rows=8, width=128, pages='bf16',
             written=0.6),
        # a small service at the default geometry: two sequences out of eight change at a time
        dict(name='turn_default', kind='turn', sequences=8, leaving=2, banks=1024, heads=1, rows=4, width=128,
             pages='bf16', written=0.5),
        # a service of 64 sequences of the serving geometry, eight of which change at a time
        dict(name='turn_batch64', kind='turn', sequences=64, leaving=8, banks=256, heads=8, rows=8, width=128,
             pages='bf16', written=0.6),
    ]


def _spread(rng, low, high):
    """A size spread over the logarithm of its range, odd or even."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(['select', 'select', 'reorder', 'step', 'step', 'fork', 'load', 'turn'])
    if kind == 'select':
        beams, batch = rng.randint(1, 16), _spread(rng, 1, 64)
        return dict(kind='select', batch=batch, beams=beams, width=rng.randint(1, 16), vocab=_spread(rng, 64, 50257),
                    dtype=rng.choice(['bf16', 'bf16', 'fp32']), finished=rng.random() < 0.6,
                    penalty=rng.choice([0.0, 0.0, 0.6, 1.0]))
    heads, rows, width, banks = rng.choice([(1, 4, 128, 1024), (8, 8, 128, 256), (4, 8, 64, 256), (2, 16, 64, 64),
                                            (1, 8, 512, 144), (3, 8, 24, 256), (1, 5, 36, 1024)])
    pages = 'fp32' if rng.random() < 0.25 else 'bf16'
    shape = dict(banks=banks, heads=heads, rows=rows, width=width)
    beams = rng.randint(2, 12)
    most = max(4, min(64, 200_000_000 // (banks * heads * rows * width * (4 if pages == 'fp32' else 2))))
    if kind == 'reorder':
        return dict(kind='reorder', batch=max(1, _spread(rng, 2, most) // beams), beams=beams, tensors=rng.randint(1, 4),
                    dtype=pages, **shape)
    if kind == 'step':
        own_banks = rng.random() < 0.4
        groups = max(1, _spread(rng, 2, most) // beams)
        return dict(kind='step', sequences=_spread(rng, 1, most) if own_banks else groups * beams,
                    beams=0 if own_banks else beams, selected=rng.choice([4, 8, 8]), pages=pages,
                    dtype='fp32' if rng.random() < 0.25 else 'bf16', decay=rng.random() < 0.7, **shape)
    if kind == 'fork':
        return dict(kind='fork', layers=rng.randint(1, 8), sequences=max(1, _spread(rng, 2, most) // beams) * beams,
                    beams=beams, pages=pages, **shape)
    if kind == 'load':
        take = _spread(rng, 1, max(2, most // 4))
        return dict(kind='load', sequences=take + rng.randint(1, 4), take=take, pages=pages,
                    written=round(rng.uniform(0.05, 1.0), 2), **shape)
    leaving = rng.randint(1, max(1, most // 8))
    return dict(kind='turn', sequences=2 * leaving + rng.randint(1, max(1, most // 2)), leaving=leaving, pages=pages,
                written=round(rng.uniform(0.2, 1.0), 2), **shape)


# ---------------------------------------------------------------------------------------------- inputs

def _parents(c, gen):
    """A parent row for each row, within its group of beams."""
    beams = c['beams']
    rows = c.get('sequences') or c['batch'] * beams
    base = torch.arange(rows, device='cuda') // beams * beams
    return base + torch.randint(beams, (rows,), generator=gen, device='cuda')


def _states(shape, dtype, gen):
    """Bank states of a running service."""
    out = torch.empty(shape, device='cuda', dtype=dtype)
    return out.normal_(std=0.05, generator=gen)


def _paged(c, gen, layers, spare, shared=0.0):
    """The tensors of a paged cache: pool, table and reference counts.  The
    first sequence has a page for each bank, the others share a part ``shared``
    of them with it and have pages for the rest; ``spare`` pages more are free."""
    n, j = c['sequences'], c['banks']
    order = torch.rand(layers, n, j, generator=gen, device='cuda').argsort(-1).argsort(-1)
    ask = order < round((1 - shared) * j)
    ask[:, 0] = True
    table = (torch.cumsum(ask.flatten(), 0) - 1).view_as(ask)
    table = torch.where(ask, table, table[:, :1])
    used = int(ask.sum())
    references = torch.zeros(used + spare, dtype=torch.int32, device='cuda')
    references[:used] = torch.bincount(table.flatten(), minlength=used).int()
    pool = _states((used + spare, c['heads'], c['rows'], c['width']), DTYPES[c['pages']], gen)
    return dict(pool=pool, table=table.int(), references=references)


def _prompts(c, gen, take, base):
    """Prefilled caches: the base's banks, a part of them written."""
    states = _states((take, c['banks'], c['heads'], c['rows'], c['width']), DTYPES[c['pages']], gen)
    kept = torch.rand(take, c['banks'], generator=gen, device='cuda') >= c['written']
    return torch.where(kept[:, :, None, None, None], base, states)


def _token(c, gen):
    """Controllers and routes of one token for each sequence."""
    n, h, s, v, j, sel = (c[x] for x in ('sequences', 'heads', 'rows', 'width', 'banks', 'selected'))
    dtype = DTYPES[c['dtype']]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device='cuda')

    q, k = (torch.nn.functional.normalize(normal(n, h, s), dim=-1).to(dtype) for _ in range(2))
    value, w = normal(n, h, v).to(dtype), torch.sigmoid(normal(n, h, v)).to(dtype)
    b, g = torch.sigmoid(normal(n, h, s)).to(dtype), -torch.nn.functional.softplus(normal(n, h, s) - 2)
    wi, ri = (torch.rand(n, j, generator=gen, device='cuda').argsort(-1)[:, :sel].contiguous() for _ in range(2))
    ww, rw = (torch.softmax(normal(n, sel), -1).to(dtype) for _ in range(2))
    return (q, k, value, g, b, w, wi, ww, ri, rw)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device='cuda')
    gen.manual_seed(int(seed) * 1013 + 7)
    kind = c['kind']
    state = dict(case=c)
    if kind == 'select':
        b, k, v = c['batch'], c['beams'], c['vocab']
        x = torch.randn(b, k, v, generator=gen, device='cuda') * 2.5
        state['logits'] = x.to(DTYPES[c['dtype']])
        # summed log-probabilities of some tens of tokens, the beams of a prompt near each other
        state['scores'] = (-20 - 40 * torch.rand(b, 1, generator=gen, device='cuda')
                           - 4 * torch.rand(b, k, generator=gen, device='cuda'))
        state['lengths'] = torch.randint(5, 40, (b, k), generator=gen, device='cuda', dtype=torch.int32)
        state['finished'] = (torch.rand(b, k, generator=gen, device='cuda') < 0.2) & bool(c['finished'])
    elif kind == 'reorder':
        shape = (c['batch'] * c['beams'], c['banks'], c['heads'], c['rows'], c['width'])
        state['states'] = [_states(shape, DTYPES[c['dtype']], gen) for _ in range(c['tensors'])]
        state['parents'] = _parents(c, gen)
    elif kind == 'step':
        spare = c['sequences'] * c['selected']
        state.update(_paged(c, gen, 1, spare))
        state['parents'] = _parents(c, gen) if c['beams'] else None
        state['token'] = _token(c, gen)
    elif kind == 'fork':
        state.update(_paged(c, gen, c['layers'], 0, shared=0.7))
        state['parents'] = _parents(c, gen)
    elif kind == 'load':
        state.update(_paged(c, gen, 1, 64))
        base = state['pool'][state['table'][0, 0].long()]
        state['prompts'] = _prompts(c, gen, c['take'], base)
    else:
        # room for both groups with every bank written
        state.update(_paged(c, gen, 1, 2 * c['leaving'] * c['banks'], shared=1 - c['written']))
        base = state['pool'][state['table'][0, 0].long()]
        state['prompts'] = [_prompts(c, gen, c['leaving'], base) for _ in range(2)]
    return state


# ---------------------------------------------------------------------------------------------- plain forms

def _select(s):
    """Every candidate's total in 64 bits (two beams' candidates can be near
    each other), sorted stably: ties go to the lowest index."""
    c, x, scores, finished, lengths = s['case'], s['logits'], s['scores'], s['finished'], s['lengths']
    eos, beams, vocab = 0, c['beams'], c['vocab']
    x = x.double()
    top = x.amax(-1, keepdim=True)
    x = x - (top + (x - top).exp().sum(-1, keepdim=True).log())
    total = scores.double().unsqueeze(-1) + x
    ended = torch.full_like(x[:1, :1], -math.inf).expand_as(x).clone()
    ended[..., eos] = scores.double()
    total = torch.where(finished.unsqueeze(-1), ended, total)
    length = lengths + (~finished).int()
    compared = total / length.double().pow(c['penalty']).unsqueeze(-1)
    compared = torch.where(torch.isfinite(compared), compared, -math.inf).flatten(1)
    index = compared.sort(dim=-1, descending=True, stable=True).indices[:, :c['width']]
    parent, token = index // vocab, index % vocab
    ends = finished.gather(1, parent) | (token == eos)
    base = torch.arange(c['batch'], device=x.device).unsqueeze(-1) * beams
    return dict(scores=total.flatten(1).gather(1, index).float(), tokens=token, parents=base + parent,
                finished=ends & bool(c['finished']), lengths=length.gather(1, parent))


def _fork(s):
    table, references = s['table'], s['references']
    table.copy_(table[:, s['parents']])
    references.copy_(torch.bincount(table.flatten(), minlength=references.numel()))


def _step(s):
    """One token over pages: pages for shared banks that are written, the write
    rule and the reads, in 32 bits."""
    pool, table, references, (q, k, v, g, b, w, wi, ww, ri, rw) = s['pool'], s['table'][0], s['references'], s['token']
    if s['parents'] is not None:
        _fork(s)
    source = table.gather(1, wi).long()
    shared = references[source] > 1
    rank = torch.cumsum(shared.flatten().int(), 0).view_as(shared) - 1
    free = (references == 0).nonzero().flatten()
    target = torch.where(shared, free[rank.clamp(0, free.numel() - 1)], source)
    references.index_add_(0, source[shared], torch.full_like(source[shared], -1, dtype=torch.int32))
    references[target[shared]] = 1
    table.scatter_(1, wi, target.int())
    p = ww.float()[:, :, None, None]
    q, k, v, g, b, w = (t.float().unsqueeze(1) for t in (q, k, v, g, b, w))
    held = pool[source].float() * torch.exp(g * p if s['case']['decay'] else g).unsqueeze(-1)
    erased = ((b * p * k).unsqueeze(-1) * held).sum(-2)
    held = held + k.unsqueeze(-1) * (w * p * v - erased).unsqueeze(-2)
    pool[target] = held.to(pool.dtype)
    read = pool[table.gather(1, ri).long()].float()
    y = ((q * rw.float()[:, :, None, None]).unsqueeze(-1) * read).sum((1, 3)) * s['case']['rows'] ** -0.5
    return y.flatten(1).to(s['token'][0].dtype)


def _release(s, first, count):
    table, references = s['table'][0, first:first + count], s['references']
    held = table[table >= 0].long()
    references.sub_(torch.bincount(held, minlength=references.numel()).int())
    table.fill_(-1)


def _load(s, first, prompts):
    """Sequences [first, first + n) take the prompts' banks: pages shared with
    sequence 0 where the bits agree, the lowest free pages otherwise."""
    pool, table, references = s['pool'], s['table'][0], s['references']
    _release(s, first, prompts.shape[0])
    base = table[0].long()
    word = torch.int32 if prompts.dtype == torch.float32 else torch.int16
    differs = (prompts.view(word) != pool[base].view(word)).flatten(2).any(-1)
    need = torch.cumsum(differs.flatten().int(), 0).view_as(differs) - 1
    free = (references == 0).nonzero().flatten()
    pages = torch.where(differs, free[need.clamp(min=0)], base)
    pool[pages[differs]] = prompts[differs]
    references.add_(torch.bincount(pages.flatten(), minlength=references.numel()).int())
    table[first:first + prompts.shape[0]] = pages.int()


def _compact(s):
    pool, table, references = s['pool'], s['table'], s['references']
    used = references > 0
    ids = torch.arange(used.numel(), device=used.device)
    low = ids < used.sum()
    source, target = ids[used & ~low], ids[~used & low]
    pool[target] = pool[source]
    references[target], references[source] = references[source], 0
    moved = ids.clone()
    moved[source] = target
    table.copy_(torch.where(table >= 0, moved[table.clamp(min=0).long()].int(), table))


def _turn(s):
    """Two groups of sequences leave, one behind the other, and others take
    their places; the first sequence (the initial state) stays."""
    _release(s, 1, s['case']['leaving'])
    _compact(s)
    _load(s, 1, s['prompts'][0])
    _release(s, 1 + s['case']['leaving'], s['case']['leaving'])
    _compact(s)
    _load(s, 1 + s['case']['leaving'], s['prompts'][1])


# ---------------------------------------------------------------------------------------------- one pass

def _pages(s):
    """The handle that a program keeps over its paged cache."""
    from bdm_amd import BankPages
    if 'handle' not in s:
        s['handle'] = BankPages.over(s['pool'], s['table'], s['references'])
    return s['handle']


def _run_own(s):
    from bdm_amd import ops
    c = s['case']
    kind = c['kind']
    if kind == 'select':
        extra = dict(finished=s['finished'], eos=0) if c['finished'] else {}
        out = ops.beam_select(s['logits'], s['scores'], width=c['width'], lengths=s['lengths'],
                              length_penalty=c['penalty'], **extra)
        ended = out.finished if c['finished'] else torch.zeros_like(out.tokens, dtype=torch.bool)
        return dict(scores=out.scores, tokens=out.tokens, parents=out.parents, finished=ended, lengths=out.lengths)
    if kind == 'reorder':
        ops.reorder_states(s['states'], s['parents'], beams=c['beams'])
        return s['states']
    pages = _pages(s)
    if kind == 'fork':
        pages.fork(s['parents'])
        return [s['table'], s['references']]
    if kind == 'step':
        if s['parents'] is not None:
            pages.fork(s['parents'])
        y = pages.decode(0, *s['token'], scale=c['rows'] ** -0.5, routed_decay=c['decay'])
        return [y, s['pool'], s['table'], s['references']]
    if kind == 'load':
        group = range(1, 1 + c['take'])
        pages.load(0, group, s['prompts'], base=0)
        return [pages.dense(0, group), s['pool'], s['table'], s['references']]
    n = c['leaving']
    groups = range(1, 1 + n), range(1 + n, 1 + 2 * n)
    pages.release(groups[0])
    pages.compact()
    pages.load(0, groups[0], s['prompts'][0], base=0)
    pages.release(groups[1])
    pages.compact()
    pages.load(0, groups[1], s['prompts'][1], base=0)
    return [s['pool'], s['table'], s['references']]


def run(state):
    s, kind = state, state['case']['kind']
    if own:
        return _run_own(s)
    if kind == 'select':
        return _select(s)
    if kind == 'reorder':
        return [t.copy_(t[s['parents']]) for t in s['states']]
    if kind == 'fork':
        _fork(s)
        return [s['table'], s['references']]
    if kind == 'step':
        return [_step(s), s['pool'], s['table'], s['references']]
    if kind == 'load':
        _load(s, 1, s['prompts'])
        return [s['pool'][s['table'][0, 1:1 + s['case']['take']].long()], s['pool'], s['table'], s['references']]
    _turn(s)
    return [s['pool'], s['table'], s['references']]


# ---------------------------------------------------------------------------------------------- work and 64 bits

def work(case):
    c = case
    kind = c['kind']
    if kind == 'select':
        logits = c['batch'] * c['beams'] * c['vocab']
        return dict(bytes=logits * (4 if c['dtype'] == 'fp32' else 2) + c['batch'] * (13 * c['beams'] + 25 * c['width']),
                    flops=4 * logits)
    page = c['heads'] * c['rows'] * c['width']
    es = 4 if c.get('pages', c.get('dtype')) == 'fp32' else 2
    if kind == 'reorder':
        # of K beams with parents at random K - 1 move on average; a row is read if another beam continues it
        k = c['beams']
        rows = c['batch'] * ((k - 1) + k * (1 - (1 - 1 / k) ** (k - 1)))
        return dict(bytes=c['tensors'] * rows * c['banks'] * page * es + 8 * c['batch'] * k, flops=0)
    n, j = c['sequences'], c['banks']
    entries = n * j * 4
    if kind == 'fork':
        return dict(bytes=2 * c['layers'] * entries + 8 * n, flops=0)
    if kind == 'step':
        sel, ce = c['selected'], 4 if c['dtype'] == 'fp32' else 2
        both = sel * sel / j  # banks of a token that are written and read: read once
        controllers = n * c['heads'] * (c['rows'] * (3 * ce + 4) + 3 * c['width'] * ce) + n * sel * 2 * (8 + ce)
        return dict(bytes=n * (3 * sel - both) * page * es + controllers + (2 * entries if c['beams'] else 0),
                    flops=n * page * sel * (6 + 2))
    if kind == 'load':
        banks = c['take'] * j
        # the prompts and the base read, written banks stored; then all of them read and written out
        return dict(bytes=(banks * (1 + c['written'] + 1 + 1) + j) * page * es, flops=0)
    banks = 2 * c['leaving'] * j
    # the prompts read, written banks stored; about as many pages moved into the places of those that left
    return dict(bytes=(banks * (1 + 3 * c['written']) + 2 * j) * page * es, flops=0)


class _Book:
    """A paged cache's bookkeeping on Python lists, and its pages in float64."""

    def __init__(self, s):
        self.table = s['table'].tolist()
        self.references = s['references'].tolist()
        self.pool = s['pool'].double()

    def take(self):
        page = self.references.index(0, self.low)
        self.low, self.references[page] = page, 1
        return page

    def drop(self, layer, row):
        for page in self.table[layer][row]:
            if page >= 0:
                self.references[page] -= 1
        self.table[layer][row] = [-1] * len(self.table[layer][row])

    def fork(self, parents):
        for layer, rows in enumerate(self.table):
            self.table[layer] = [list(rows[p]) for p in parents]
        count = [0] * len(self.references)
        for rows in self.table:
            for row in rows:
                for page in row:
                    count[page] += 1
        self.references = count

    def fill(self, row, states):
        same = (states == self.pool[self.table[0][0]]).flatten(1).all(-1).tolist()
        pages = []
        for bank, shared in enumerate(same):
            if shared:
                page = self.table[0][0][bank]
                self.references[page] += 1
            else:
                page = self.take()
            pages.append(page)
        self.table[0][row] = pages
        self.pool[pages] = states

    def squeeze(self):
        used = [p for p, r in enumerate(self.references) if r]
        high = [p for p in used if p >= len(used)]
        low = [p for p in range(len(used)) if not self.references[p]]
        to = dict(zip(high, low))
        if high:
            self.pool[low] = self.pool[high]
        for a, b in to.items():
            self.references[b], self.references[a] = self.references[a], 0
        self.table = [[[to.get(p, p) for p in row] for row in rows] for rows in self.table]


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    kind = c['kind']
    if kind == 'select':
        out = []
        for b in range(c['batch']):
            logs = torch.log_softmax(s['logits'][b].double(), -1)
            totals = s['scores'][b].double()[:, None] + logs
            ended = s['finished'][b].nonzero().flatten().tolist()
            for k in ended:
                totals[k] = -math.inf
                totals[k, 0] = s['scores'][b, k].double()
            norm = [float(n + (0 if k in ended else 1)) ** c['penalty'] for k, n in enumerate(s['lengths'][b].tolist())]
            best = (totals / torch.tensor(norm, device='cuda', dtype=torch.float64)[:, None]).flatten()
            out.append(totals.flatten()[best.topk(c['width']).indices])
        return dict(scores=torch.stack(out), tokens=None, parents=None, finished=None, lengths=None)
    if kind == 'reorder':
        rows = s['parents'].tolist()
        return [torch.stack([t[r].double() for r in rows]) for t in s['states']]
    if kind == 'fork':
        return None  # whole numbers alone
    book = _Book(s)
    book.low = 0
    if kind == 'load':
        for row in range(1, 1 + c['take']):
            book.drop(0, row)
        for row in range(1, 1 + c['take']):
            book.fill(row, s['prompts'][row - 1].double())
        return [s['prompts'].double(), book.pool, None, None]
    if kind == 'turn':
        n = c['leaving']
        for group, prompts in zip((range(1, 1 + n), range(1 + n, 1 + 2 * n)), s['prompts']):
            for row in group:
                book.drop(0, row)
            book.squeeze()
            book.low = 0
            for row, states in zip(group, prompts):
                book.fill(row, states.double())
        return [book.pool, None, None]
    if s['parents'] is not None:
        book.fork(s['parents'].tolist())
    q, k, v, g, b, w = (t.double() for t in s['token'][:6])
    wi, ri = s['token'][6].tolist(), s['token'][8].tolist()
    ww, rw = s['token'][7].double(), s['token'][9].double()
    written = [[(i, book.table[0][i][bank]) for bank in banks] for i, banks in enumerate(wi)]
    shared = [[book.references[page] > 1 for _, page in row] for row in written]
    moves = []
    for i, row in enumerate(written):
        for j, (_, page) in enumerate(row):
            target = book.take() if shared[i][j] else page
            moves.append((i, j, page, target))
    for i, j, page, target in moves:
        if page != target:
            book.references[page] -= 1
            book.table[0][i][wi[i][j]] = target
    before = book.pool.clone()
    for i in range(c['sequences']):
        mine = [m for m in moves if m[0] == i]
        p = ww[i][:, None, None]
        state = before[[m[2] for m in mine]]
        state = torch.exp(g[i] * p if c['decay'] else g[i].expand(len(mine), -1, -1))[..., None] * state
        u = w[i] * p * v[i] - torch.einsum('jhs,jhsv->jhv', b[i] * p * k[i], state)
        book.pool[[m[3] for m in mine]] = state + torch.einsum('hs,jhv->jhsv', k[i], u)
    y = torch.stack([torch.einsum('jhs,jhsv->hv', rw[i][:, None, None] * q[i],
                                  book.pool[[book.table[0][i][bank] for bank in ri[i]]]).flatten()
                     for i in range(c['sequences'])])
    return [y * c['rows'] ** -0.5, book.pool, None, None]
