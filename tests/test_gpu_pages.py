"""The paged bank cache against a restatement on Python lists, and its decode
step against 64 bits and the dense step.

Tolerances of the decode step, relative to sums of magnitudes: an FP32
exponential of x is off by (1 + |x|) * 2^-22 at most (its scaled argument is
rounded), a sum of S <= 32 products by 34 * 2^-24; together less than
(1 + |x|) * 4e-6.  A stored state is rounded to the cache's dtype once
(eps / 2), y from the stored states to the controllers' (eps / 2), behind FP32
sums of at most 32 + 16 terms (50 * 2^-24).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


class Book:
    """A paged cache on Python lists: pages by number, contents on the CPU."""

    def __init__(self, pages):
        self.layers, self.sequences, self.banks = pages.table.shape
        self.table = pages.table.tolist()
        self.references = pages.references.tolist()
        self.content = list(pages.pool.cpu())

    def take(self):
        page = self.references.index(0)
        self.references[page] = 1
        return page

    def drop(self, layer, row):
        for page in self.table[layer][row]:
            if page >= 0:
                self.references[page] -= 1
        self.table[layer][row] = [-1] * self.banks

    def fork(self, parents):
        for layer in range(self.layers):
            old = self.table[layer]
            self.table[layer] = [list(old[min(p, self.sequences - 1)]) if p >= 0 else [-1] * self.banks for p in parents]
        self.references = [0] * len(self.references)
        for rows in self.table:
            for row in rows:
                for page in row:
                    if page >= 0:
                        self.references[page] += 1

    def load(self, layer, rows, states, base=None):
        for row in rows:
            self.drop(layer, row)
        for row, state in zip(rows, states):
            for bank in range(self.banks):
                shared = -1 if base is None else self.table[layer][base][bank]
                if shared >= 0 and torch.equal(self.content[shared], state[bank]):
                    self.references[shared] += 1
                    page = shared
                else:
                    page = self.take()
                    self.content[page] = state[bank].clone()
                self.table[layer][row][bank] = page

    def compact(self):
        used = [p for p, r in enumerate(self.references) if r]
        high = [p for p in used if p >= len(used)]
        low = [p for p in range(len(used)) if not self.references[p]]
        to = dict(zip(high, low))
        for a, b in to.items():
            self.content[b] = self.content[a]
            self.references[b], self.references[a] = self.references[a], 0
        self.table = [[[to.get(p, p) for p in row] for row in rows] for rows in self.table]

    def write(self, layer, wi):
        """New pages for shared banks that are written: (source, target) of each."""
        moves = []
        for i, banks in enumerate(wi):
            for j, bank in enumerate(banks):
                page = self.table[layer][i][bank]
                if page >= 0 and bank not in banks[:j]:
                    moves.append((i, bank, page, self.references[page] > 1))
        out = []
        for i, bank, page, shared in moves:
            out.append((i, bank, page, self.take() if shared else page))
        for i, bank, page, target in out:
            if target != page:
                self.references[page] -= 1
                self.table[layer][i][bank] = target
        return out

    def dense(self, layer, row):
        zero = torch.zeros_like(self.content[0])
        return torch.stack([self.content[p] if p >= 0 else zero for p in self.table[layer][row]])


def agree(pages, book, contents=True):
    torch.cuda.synchronize()
    assert pages.table.tolist() == book.table
    assert pages.references.tolist() == book.references
    words = [0] * ((pages.pages + 63) // 64)
    for page, r in enumerate(book.references):
        if r == 0:
            words[page // 64] |= 1 << (page % 64)
    assert [w & (2 ** 64 - 1) for w in pages.free_bits.tolist()] == words
    assert int(pages.used()) == sum(r > 0 for r in book.references)
    pages.check()
    if contents:
        pool = pages.pool.cpu()
        for page, r in enumerate(book.references):
            if r:
                assert torch.equal(pool[page], book.content[page]), page


def token(n, heads, s, width, banks, kw, kr, dtype, gen, device):
    def normal(*shape):
        return torch.randn(*shape, generator=gen)

    unit = torch.nn.functional.normalize
    q, k = unit(normal(n, heads, s), dim=-1).to(dtype), unit(normal(n, heads, s), dim=-1).to(dtype)
    v, w = normal(n, heads, width).to(dtype), torch.sigmoid(normal(n, heads, width)).to(dtype)
    b, g = torch.sigmoid(normal(n, heads, s)).to(dtype), -torch.nn.functional.softplus(normal(n, heads, s))
    wi = torch.rand(n, banks, generator=gen).argsort(-1)[:, :kw].contiguous()
    ri = torch.rand(n, banks, generator=gen).argsort(-1)[:, :kr].contiguous()
    ww, rw = torch.softmax(normal(n, kw), -1).to(dtype), torch.softmax(normal(n, kr), -1).to(dtype)
    return [t.to(device) for t in (q, k, v, g, b, w, wi, ww, ri, rw)]


def check_step(pages, layer, step, scale, decay, y, before):
    """y and the stored states of one step against 64 bits; `before`: dense
    states [N, J, H, S, v] on the CPU ahead of it."""
    q, k, v, g, b, w, wi, ww, ri, rw = (t.cpu() for t in step)
    n = q.shape[0]
    after = pages.dense(layer, range(n)).cpu()
    rows = torch.arange(n)[:, None]
    p = ww.double()[:, :, None, None]
    eg = g.double()[:, None] * (p if decay else torch.ones_like(p))
    hd = torch.exp(eg)[..., None] * before[rows, wi].double()
    a = b.double()[:, None] * p * k.double()[:, None]
    ewv = w.double()[:, None] * p * v.double()[:, None]
    u = ewv - (a[..., None] * hd).sum(-2)
    want = hd + k.double()[:, None, ..., None] * u[..., None, :]
    size = hd.abs() + k.double().abs()[:, None, ..., None] * (ewv.abs() + (a[..., None] * hd).abs().sum(-2))[..., None, :]
    half = torch.finfo(pages.dtype).eps / 2
    empty = torch.tensor([pages.table[layer, i, 0].item() < 0 for i in range(n)])
    want[empty] = 0
    got = after[rows, wi].double()
    tolerance = half * want.abs() + 4e-6 * (1 + eg.abs().amax(-1))[..., None, None] * size + 1e-30
    assert ((got - want).abs() <= tolerance).all()
    untouched = torch.ones(n, pages.banks, dtype=torch.bool)
    untouched.scatter_(1, wi, False)
    assert torch.equal(after[untouched], before[untouched])
    reads = after[rows, ri].double()
    terms = (q.double()[:, None] * rw.double()[:, :, None, None])[..., None] * reads
    exact = (terms.sum((1, 3)) * scale).flatten(1)
    bound = terms.abs().sum((1, 3)).flatten(1) * abs(scale) * 50 * 2.0 ** -24
    assert ((y.cpu().double() - exact).abs() <= torch.finfo(y.dtype).eps / 2 * exact.abs() + bound + 1e-30).all()


GEOMETRIES = [
    # sequences, banks, heads, bank size, width, KW, KR, controllers, pages
    (1, 8, 1, 8, 16, 1, 1, 'fp32', 'fp32'), (6, 32, 2, 8, 128, 8, 8, 'bf16', 'bf16'), (5, 16, 1, 4, 128, 8, 8, 'fp32', 'bf16'),
    (4, 16, 3, 8, 24, 4, 7, 'bf16', 'fp32'), (3, 20, 1, 5, 36, 5, 3, 'bf16', 'bf16'), (2, 20, 1, 16, 64, 16, 16, 'fp32', 'fp32'),
    (3, 9, 2, 32, 6, 2, 3, 'bf16', 'bf16'), (2, 9, 1, 3, 7, 3, 2, 'fp32', 'bf16'), (2, 12, 1, 8, 2048, 8, 8, 'bf16', 'bf16'),
    (4, 16, 1, 8, 64, 3, 0, 'fp32', 'fp32'), (4, 16, 1, 8, 64, 0, 3, 'bf16', 'bf16'), (67, 24, 1, 8, 16, 16, 2, 'bf16', 'bf16'),
]


@pytest.mark.parametrize('geometry', GEOMETRIES, ids=lambda c: 'x'.join(map(str, c)))
@pytest.mark.parametrize('decay', [True, False], ids=['decay', 'plain'])
def test_decode(device, geometry, decay):
    from bdm_amd import BankPages, ops
    n, banks, heads, s, width, kw, kr, ctrl, kept = geometry
    print('CASE pages decode', geometry, decay, flush=True)
    gen = torch.Generator().manual_seed(n * 31 + banks + width)
    dtype, kind = DTYPES[ctrl], DTYPES[kept]
    # the pages that a step abandons are free behind it only: one for every two banks that it writes at most
    pages = BankPages(n, n * banks + n * kw // 2 + 1, banks=banks, heads=heads, bank_size=s, head_width=width, dtype=kind,
                      device=device)
    states = (torch.randn(n, banks, heads, s, width, generator=gen) * 0.1).to(kind)
    pages.load(0, range(n), states.to(device))
    book = Book(pages)
    for turn in range(3):
        if turn:
            parents = torch.randint(0, n, (n,), generator=gen)
            pages.fork(parents.to(device))
            book.fork(parents.tolist())
        before = torch.stack([book.dense(0, i) for i in range(n)])
        step = token(n, heads, s, width, banks, kw, kr, dtype, gen, device)
        dense = pages.dense(0, range(n))
        assert torch.equal(dense.cpu(), before)
        y = pages.decode(0, *step, scale=s ** -0.5, routed_decay=decay)
        moves = book.write(0, step[6].tolist())
        check_step(pages, 0, step, s ** -0.5, decay, y, before)
        pool = pages.pool.cpu()
        for _, _, _, target in moves:
            book.content[target] = pool[target]
        agree(pages, book)
        if ctrl == 'fp32':
            # the dense step, bit for bit
            want = ops.decode_step(*step, dense, bank_count=banks, scale=s ** -0.5, routed_decay=decay)
            assert torch.equal(want, y)
            assert torch.equal(dense, pages.dense(0, range(n)))


def make(device, n=7, banks=11, layers=2, pages=None, heads=1, s=4, width=6, dtype=torch.bfloat16, seed=0):
    from bdm_amd import BankPages
    gen = torch.Generator().manual_seed(seed)
    cache = BankPages(n, pages or layers * n * banks + n * 2 + 3, banks=banks, heads=heads, bank_size=s, head_width=width,
                      layers=layers, dtype=dtype, device=device)
    return cache, Book(cache), gen


@pytest.mark.parametrize('shape', [(1, 4, 6, 'bf16'), (1, 1, 1, 'bf16'), (1, 3, 5, 'bf16'), (2, 8, 128, 'bf16'),
                                   (1, 1, 1, 'fp32'), (3, 5, 7, 'fp32'), (1, 8, 4, 'fp32'), (4, 8, 2048, 'bf16')],
                         ids=str)
def test_load_dense_release_compact(device, shape):
    heads, s, width, kind = shape
    print('CASE pages load', shape, flush=True)
    pages, book, gen = make(device, heads=heads, s=s, width=width, dtype=DTYPES[kind], seed=3)
    first = (torch.randn(1, 11, heads, s, width, generator=gen)).to(DTYPES[kind])
    for layer in (1, 0):
        pages.load(layer, [2], first.to(device))
        book.load(layer, [2], first)
    agree(pages, book)
    for turn in range(6):
        rows = [r for r in torch.randperm(7, generator=gen).tolist() if r != 2][:1 + turn % 4]
        states = first.expand(len(rows), -1, -1, -1, -1).clone()
        change = torch.rand(len(rows), 11, generator=gen) < 0.5
        states[change] += 1
        if turn == 1:
            states[:, :, -1, -1, -1] += 1   # differs in the last value of each page alone
        base = None if turn == 3 else 2
        layer = turn % 2
        pages.load(layer, rows, states.to(device), base=base)
        book.load(layer, rows, states, base=base)
        agree(pages, book)
        out = pages.dense(layer, rows).cpu()
        assert torch.equal(out, states)
        if turn % 2:
            gone = rows[:2]
            pages.release(gone)
            for la in (0, 1):
                for r in gone:
                    book.drop(la, r)
            agree(pages, book)
            assert not pages.dense(layer, gone).any()
            pages.compact()
            book.compact()
            agree(pages, book)
    assert torch.equal(pages.dense(0, range(7)).cpu(), torch.stack([book.dense(0, i) for i in range(7)]))
    pages.release(range(7))
    pages.compact()
    assert int(pages.used()) == 0


@pytest.mark.parametrize('n', [1, 7, 128, 129, 300, 512])
def test_fork(device, n):
    print('CASE pages fork', n, flush=True)
    pages, book, gen = make(device, n=n, banks=67, layers=2, s=1, width=8, seed=n)
    table = torch.arange(2 * n * 67).view(2, n, 67)
    pages.table.copy_(table)
    pages.references[:2 * n * 67] = 1
    from bdm_amd import BankPages
    pages = BankPages.over(pages.pool, pages.table, pages.references)
    book = Book(pages)
    choices = [torch.arange(n), torch.randint(0, n, (n,), generator=gen), torch.randint(-1, n, (n,), generator=gen),
               torch.arange(n).flip(0), torch.full((n,), n - 1), torch.randint(-9, n + 9, (n,), generator=gen),
               torch.full((n,), -1)]
    for parents in choices:
        pages.fork(parents.to(device))
        book.fork(parents.tolist())
        agree(pages, book)


def test_pool_of_many_words(device):
    """More pages than one tile of the bit map holds, allocated from the far end."""
    from bdm_amd import BankPages
    pages = 70_001
    pool = torch.zeros(pages, 1, 1, 8, dtype=torch.float32, device=device)
    references = torch.ones(pages, dtype=torch.int32, device=device)
    free = torch.tensor([3, 64, 65_535, 65_536, 69_000, 69_999, 70_000])
    references[free.to(device)] = 0
    table = torch.full((1, 4, 3), -1, dtype=torch.int32, device=device)
    cache = BankPages.over(pool, table, references)
    states = torch.arange(48, dtype=torch.float32, device=device).view(2, 3, 1, 1, 8)
    cache.load(0, [3, 1], states)
    torch.cuda.synchronize()
    assert table[0, 3].tolist() == [3, 64, 65_535] and table[0, 1].tolist() == [65_536, 69_000, 69_999]
    assert torch.equal(cache.dense(0, [3, 1]), states)
    cache.check()
    # compaction across tiles: everything else is freed but a few pages at the end
    references.zero_()
    table[0, 0] = torch.tensor([70_000, 65_537, 5], dtype=torch.int32)
    table[0, 2] = torch.tensor([69_998, 65_537, 66_000], dtype=torch.int32)
    used = table[table >= 0].long()
    references.copy_(torch.bincount(used, minlength=pages).int())
    pool.copy_(torch.randn(pages, 1, 1, 8))
    cache = BankPages.over(pool, table, references)
    book, want = Book(cache), cache.dense(0, range(4))
    cache.compact()
    book.compact()
    agree(cache, book)
    assert torch.equal(cache.dense(0, range(4)), want)
    assert int(cache.table.max()) == int(cache.used()) - 1


def test_many_new_pages_at_once(device):
    pages, book, gen = make(device, n=4, banks=3001, layers=1, s=1, width=4, dtype=torch.float32)
    first = torch.randn(1, 3001, 1, 1, 4, generator=gen)
    pages.load(0, [1], first.to(device))
    states = torch.where(torch.rand(3, 3001, 1, 1, 1, generator=gen) < 0.97, first + 1, first)
    pages.load(0, [3, 0, 2], states.to(device), base=1)
    book.load(0, [1], first)
    book.load(0, [3, 0, 2], states, base=1)
    agree(pages, book)
    pages.release([0, 1])
    book.drop(0, 0)
    book.drop(0, 1)
    pages.compact()
    book.compact()
    agree(pages, book)


def test_offsets_beyond_32_bits(device):
    """Pages behind the first 4 GiB of the pool, and behind 2^31 elements."""
    from bdm_amd import BankPages
    heads, s, width, banks = 1, 8, 2048, 12
    pages = 2 ** 32 // (s * width * 2) * 2 + 100
    pool = torch.zeros(pages, heads, s, width, dtype=torch.bfloat16, device=device)
    references = torch.zeros(pages, dtype=torch.int32, device=device)
    references[:pages - 40] = 1
    table = torch.full((1, 3, banks), -1, dtype=torch.int32, device=device)
    cache = BankPages.over(pool, table, references)
    gen = torch.Generator().manual_seed(5)
    states = (torch.randn(2, banks, heads, s, width, generator=gen) * 0.1).bfloat16()
    cache.load(0, [0, 1], states.to(device))
    assert torch.equal(cache.dense(0, [0, 1]).cpu(), states)
    cache.fork(torch.tensor([0, 1, 0], device=device))
    step = token(3, heads, s, width, banks, 8, 8, torch.bfloat16, gen, device)
    y = cache.decode(0, *step, scale=0.5, routed_decay=True)
    assert int(table.min()) >= pages - 40
    check_step(cache, 0, step, 0.5, True, y, torch.cat([states, states[:1]]))
    cache.check()
    assert not pool[:1000].any()


def test_empty_sequences_stay_empty(device):
    pages, book, gen = make(device, n=5, banks=16, layers=1, s=8, width=16, dtype=torch.float32)
    states = torch.randn(2, 16, 1, 8, 16, generator=gen)
    pages.load(0, [1, 3], states.to(device))
    book.load(0, [1, 3], states)
    before = torch.stack([book.dense(0, i) for i in range(5)])
    step = token(5, 1, 8, 16, 16, 4, 4, torch.float32, gen, device)
    step[8][:, :2] = step[6][:, :2]    # banks that are written and read
    y = pages.decode(0, *step, scale=1.0, routed_decay=True)
    book.write(0, step[6].tolist())
    assert not y[[0, 2, 4]].any() and y[[1, 3]].any()
    check_step(pages, 0, step, 1.0, True, y, before)
    agree(pages, book, contents=False)


def test_no_free_page(device):
    """A pool that is too small: nothing is written but what has pages."""
    pages, book, gen = make(device, n=4, banks=8, layers=1, pages=20, s=8, width=16, dtype=torch.float32)
    states = torch.randn(1, 8, 1, 8, 16, generator=gen)
    pages.load(0, [0], states.to(device))
    pages.fork(torch.zeros(4, dtype=torch.int64, device=device))
    before = pages.dense(0, range(4)).cpu()
    step = token(4, 1, 8, 16, 8, 4, 4, torch.float32, gen, device)
    pages.decode(0, *step, scale=1.0, routed_decay=True)   # asks for 16 pages of 12
    with pytest.raises(RuntimeError):
        pages.check()
    after = pages.dense(0, range(4)).cpu()
    wi = step[6].cpu()
    assert torch.equal(after[3], before[3])                # the last four requests
    for i in range(3):
        assert all(not torch.equal(after[i, j], before[i, j]) for j in wi[i].tolist())
    count = torch.bincount(pages.table.flatten().cpu(), minlength=20)
    assert torch.equal(count.int(), pages.references.cpu()) and int(pages.used()) == 20
    # load: the banks without a page read as zeros
    pages.status.zero_()
    other = torch.randn(1, 8, 1, 8, 16, generator=gen)
    pages.release([3])
    pages.load(0, [3], other.to(device))
    with pytest.raises(RuntimeError):
        pages.check()
    table, got = pages.table[0, 3].cpu(), pages.dense(0, [3]).cpu()[0]
    assert (table < 0).any()
    for j in range(8):
        assert torch.equal(got[j], other[0, j] if table[j] >= 0 else torch.zeros_like(other[0, j]))


def test_a_bank_twice_in_one_token_keeps_the_books(device):
    pages, book, gen = make(device, n=3, banks=8, layers=1, s=8, width=16, dtype=torch.float32)
    states = torch.randn(1, 8, 1, 8, 16, generator=gen)
    pages.load(0, [0], states.to(device))
    pages.fork(torch.zeros(3, dtype=torch.int64, device=device))
    book = Book(pages)
    step = token(3, 1, 8, 16, 8, 4, 4, torch.float32, gen, device)
    step[6][1, 2] = step[6][1, 0]
    step[6][2, :] = step[6][2, 3]
    pages.decode(0, *step, scale=1.0, routed_decay=True)
    book.write(0, step[6].tolist())
    agree(pages, book, contents=False)


def test_banks_outside_are_clamped(device):
    pages, book, gen = make(device, n=2, banks=8, layers=1, s=8, width=16, dtype=torch.float32)
    states = torch.randn(2, 8, 1, 8, 16, generator=gen)
    pages.load(0, [0, 1], states.to(device))
    step = token(2, 1, 8, 16, 8, 2, 2, torch.float32, gen, device)
    step[6][0] = torch.tensor([-7, 99])
    step[8][1] = torch.tensor([10 ** 12, -(10 ** 12)])
    same = [t.clone() for t in step]
    same[6][0] = torch.tensor([0, 7])
    same[8][1] = torch.tensor([7, 0])
    y = pages.decode(0, *step, scale=1.0, routed_decay=True)
    after = pages.dense(0, [0, 1])
    pages.load(0, [0, 1], states.to(device))
    assert torch.equal(y, pages.decode(0, *same, scale=1.0, routed_decay=True))
    assert torch.equal(after, pages.dense(0, [0, 1]))


def test_a_long_run_of_calls(device):
    """Calls in a random order, the books compared behind each."""
    pages, book, gen = make(device, n=9, banks=13, layers=3, s=8, width=16, dtype=torch.float32, seed=8)
    first = torch.randn(1, 13, 1, 8, 16, generator=gen)
    for layer in range(3):
        pages.load(layer, [0], first.to(device))
        book.load(layer, [0], first)
    for turn in range(60):
        kind = int(torch.randint(0, 6, (1,), generator=gen))
        layer = int(torch.randint(0, 3, (1,), generator=gen))
        rows = (torch.randperm(8, generator=gen)[:1 + turn % 3] + 1).tolist()
        if kind == 0:
            states = torch.where(torch.rand(len(rows), 13, 1, 1, 1, generator=gen) < 0.5, first, first + turn + 1)
            pages.load(layer, rows, states.to(device), base=0)
            book.load(layer, rows, states, base=0)
        elif kind == 1:
            parents = torch.randint(-1, 9, (9,), generator=gen)
            parents[0] = 0
            pages.fork(parents.to(device))
            book.fork(parents.tolist())
        elif kind == 2:
            pages.release(rows)
            for la in range(3):
                for r in rows:
                    book.drop(la, r)
        elif kind == 3:
            pages.compact()
            book.compact()
        else:
            step = token(9, 1, 8, 16, 13, 3, 3, torch.float32, gen, device)
            before = torch.stack([book.dense(layer, i) for i in range(9)])
            y = pages.decode(layer, *step, scale=1.0, routed_decay=True)
            moves = book.write(layer, step[6].tolist())
            check_step(pages, layer, step, 1.0, True, y, before)
            pool = pages.pool.cpu()
            for _, _, _, target in moves:
                book.content[target] = pool[target]
        agree(pages, book)


def test_graph_of_fork_and_decode(device):
    """Fork and decode captured once and replayed, eager calls between, against a cache of eager calls alone."""
    caches = []
    for _ in range(2):
        pages, _, gen = make(device, n=6, banks=16, layers=1, s=8, width=32, seed=2)
        states = torch.randn(6, 16, 1, 8, 32, generator=gen).bfloat16().to(device)
        pages.load(0, range(6), states)
        caches.append(pages)
    live, eager = caches
    step = token(6, 1, 8, 32, 16, 4, 4, torch.bfloat16, gen, device)
    parents = torch.arange(6, device=device)
    live.decode(0, *step, scale=1.0, routed_decay=True)
    eager.decode(0, *step, scale=1.0, routed_decay=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        live.fork(parents)
        y = live.decode(0, *step, scale=1.0, routed_decay=True)
        live.compact()
    for turn in range(5):
        parents.copy_(torch.randint(0, 6, (6,), generator=gen))
        for t, new in zip(step, token(6, 1, 8, 32, 16, 4, 4, torch.bfloat16, gen, device)):
            t.copy_(new)
        graph.replay()
        eager.fork(parents)
        want = eager.decode(0, *step, scale=1.0, routed_decay=True)
        eager.compact()
        torch.cuda.synchronize()
        assert torch.equal(want, y)
        assert torch.equal(live.table, eager.table) and torch.equal(live.references, eager.references)
        assert torch.equal(live.dense(0, range(6)), eager.dense(0, range(6)))
        if turn == 2:
            for cache in caches:
                cache.release([4])
                cache.load(0, [4], states[:1])


def test_the_first_sequences_alone(device):
    """A step and a fork of fewer sequences leave the others as they were."""
    pages, book, gen = make(device, n=6, banks=16, layers=1, s=8, width=16, dtype=torch.float32)
    states = torch.randn(6, 16, 1, 8, 16, generator=gen)
    pages.load(0, range(6), states.to(device))
    book.load(0, range(6), states)
    parents = torch.tensor([5, 0, 2, -1])
    pages.fork(parents.to(device))
    book.fork([5, 0, 2, -1, 4, 5])
    agree(pages, book)
    before = torch.stack([book.dense(0, i) for i in range(6)])
    step = token(3, 1, 8, 16, 16, 4, 4, torch.float32, gen, device)
    y = pages.decode(0, *step, scale=1.0, routed_decay=True)
    book.write(0, step[6].tolist())
    agree(pages, book, contents=False)
    check_step(pages, 0, step, 1.0, True, y, before[:3])
    assert torch.equal(pages.dense(0, [3, 4, 5]).cpu(), before[3:])


def test_on_a_side_stream(device):
    pages, book, gen = make(device, n=4, banks=8, layers=1, s=8, width=16, dtype=torch.float32)
    side = torch.cuda.Stream()
    states = torch.randn(4, 8, 1, 8, 16, generator=gen)
    step = token(4, 1, 8, 16, 8, 4, 4, torch.float32, gen, device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pages.load(0, range(4), states.to(device))
        pages.fork(torch.tensor([0, 0, 2, 2], device=device))
        y = pages.decode(0, *step, scale=1.0, routed_decay=True)
    side.synchronize()
    book.load(0, range(4), states)
    book.fork([0, 0, 2, 2])
    before = torch.stack([book.dense(0, i) for i in range(4)])
    book.write(0, step[6].tolist())
    agree(pages, book, contents=False)
    check_step(pages, 0, step, 1.0, True, y, before)


def test_two_caches_on_two_streams(device):
    """Steps and forks of two caches at once, each equal to the same calls alone."""
    ends = []
    for at_once in (False, True):
        caches, streams = [], []
        for n in range(2):
            pages, _, gen = make(device, n=6, banks=16, layers=1, s=8, width=32, seed=60 + n)
            states = torch.randn(6, 16, 1, 8, 32, generator=gen).bfloat16().to(device)
            steps = [token(6, 1, 8, 32, 16, 8, 8, torch.bfloat16, gen, device) for _ in range(6)]
            orders = [torch.randint(0, 6, (6,), generator=gen).to(device) for _ in steps]
            caches.append((pages, states, steps, orders, []))
            streams.append(torch.cuda.Stream() if at_once else torch.cuda.current_stream())
        torch.cuda.synchronize()
        for t in range(6):
            for (pages, states, steps, orders, out), stream in zip(caches, streams):
                with torch.cuda.stream(stream):
                    if t == 0:
                        pages.load(0, range(6), states)
                    pages.fork(orders[t])
                    out.append(pages.decode(0, *steps[t], scale=0.5, routed_decay=True))
        torch.cuda.synchronize()
        ends.append([(pages.dense(0, range(6)), pages.table.clone(), *out) for pages, _, _, _, out in caches])
    for one, two in zip(*ends):
        assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_controllers_of_any_layout(device):
    """Views that start anywhere, with strides, and one tensor in two places: the results of plain ones."""
    results = []
    for plain in (True, False):
        pages, _, gen = make(device, n=4, banks=8, layers=1, s=8, width=16, dtype=torch.float32, seed=70)
        pages.load(0, range(4), torch.randn(4, 8, 1, 8, 16, generator=gen).to(device))
        step = token(4, 1, 8, 16, 8, 4, 4, torch.float32, gen, device)
        q, k, v, g, b, w, wi, ww, ri, rw = step
        g, rw = b, ww
        if not plain:
            q = torch.cat([q.new_zeros(1), q.flatten()])[1:].view(q.shape)
            v = torch.stack([v, v], -1)[..., 0]
            b = b.transpose(0, 2).contiguous().transpose(0, 2)
            g = b
            wi = torch.cat([wi, wi], 1)[:, :4]
            ri = torch.cat([ri.new_zeros(1), ri.flatten()])[1:].view(ri.shape)
            ww = ww.t().contiguous().t()
        y = pages.decode(0, q, k, v, g, b, w, wi, ww, ri, rw, scale=1.0, routed_decay=True)
        results.append((y, pages.dense(0, range(4))))
        with pytest.raises(ValueError):  # g may be FP32 beside others, b may not
            pages.decode(0, q.bfloat16(), k.bfloat16(), v.bfloat16(), g, b, w.bfloat16(), wi, ww.bfloat16(), ri,
                         rw.bfloat16(), scale=1.0, routed_decay=True)
        with pytest.raises(ValueError):
            pages.decode(0, q, k, v.bfloat16(), g, b, w, wi, ww, ri, rw, scale=1.0, routed_decay=True)
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_one_head_caches_of_the_layer(device):
    pages, book, gen = make(device, n=2, banks=4, layers=1, s=4, width=8)
    states = torch.randn(2, 4, 4, 8, generator=gen).bfloat16()
    pages.load(0, range(2), states.to(device))
    assert torch.equal(pages.dense(0, range(2)).cpu(), states.unsqueeze(2))


def test_calls_refuse(device):
    from bdm_amd import BankPages
    pages, _, gen = make(device, n=3, banks=8, layers=2, s=8, width=16)
    states = torch.zeros(1, 8, 1, 8, 16, dtype=torch.bfloat16, device=device)
    step = token(3, 1, 8, 16, 8, 4, 4, torch.bfloat16, gen, device)
    before = pages.table.clone()

    def refused(call, *args, **options):
        with pytest.raises(ValueError):
            call(*args, **options)

    refused(pages.load, 2, [0], states)
    refused(pages.load, -1, [0], states)
    refused(pages.load, 0, [3], states)
    refused(pages.load, 0, [0, 0], states.expand(2, -1, -1, -1, -1))
    refused(pages.load, 0, [0, 1], states)
    refused(pages.load, 0, [0], states.float())
    refused(pages.load, 0, [0], states, base=0)
    refused(pages.load, 0, [0], states, base=3)
    refused(pages.load, 0, [0], states.cpu())
    refused(pages.dense, 0, [-1])
    refused(pages.release, [5])
    refused(pages.fork, torch.zeros(3, dtype=torch.int32, device=device))
    refused(pages.fork, torch.zeros(4, dtype=torch.int64, device=device))
    refused(pages.fork, torch.zeros(0, dtype=torch.int64, device=device))
    refused(pages.fork, torch.zeros(3, dtype=torch.int64))

    def changed(i, t):
        other = list(step)
        other[i] = t
        return other

    for other in (changed(0, step[0][:2]), changed(2, step[2][..., :8]), changed(1, step[1].float()),
                  changed(6, step[6].int()), changed(6, step[6][:, :3]), changed(8, step[8][:2]), changed(3, step[3].cpu())):
        refused(pages.decode, 0, *other, scale=1.0, routed_decay=True)
    refused(BankPages.over, pages.pool, pages.table.long(), pages.references)
    refused(BankPages.over, pages.pool, pages.table, pages.references[1:])
    refused(BankPages.over, pages.pool[:, :, ::2], pages.table, pages.references)
    refused(BankPages.over, pages.pool.half(), pages.table, pages.references)
    odd, _, _ = make(device, n=3, banks=8, layers=1, s=8, width=521)  # no span of a workgroup divides the head
    odd.load(0, [0], torch.zeros(1, 8, 1, 8, 521, dtype=torch.bfloat16, device=device))
    odd.fork(torch.zeros(3, dtype=torch.int64, device=device))
    with pytest.raises(NotImplementedError):
        odd.decode(0, *token(3, 1, 8, 521, 8, 4, 4, torch.bfloat16, gen, device), scale=1.0, routed_decay=True)
    assert torch.equal(odd.table[0, 0], odd.table[0, 2]) and int(odd.used()) == 8
    with pytest.raises(NotImplementedError):
        wide = [t.repeat(1, 5) if i > 5 else t for i, t in enumerate(step)]
        pages.decode(0, *wide, scale=1.0, routed_decay=True)
    torch.cuda.synchronize()
    assert torch.equal(before, pages.table)


def test_a_handle_dropped_while_a_stream_runs(device):
    """Memory of a handle goes to nobody else while a call on another stream than its own still has it."""
    pages, book, gen = make(device, n=4, banks=8, layers=1, s=8, width=16, dtype=torch.float32, seed=90)
    states = torch.randn(4, 8, 1, 8, 16, generator=gen)
    pages.load(0, range(4), states.to(device))
    book.load(0, range(4), states)
    parents = torch.tensor([0, 0, 2, 1], device=device)
    held = (pages.pool, pages.table, pages.references, pages.free_bits, pages.status, pages._tables)
    spans = [(t.data_ptr(), t.data_ptr() + t.nbytes) for t in held]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        pages.fork(parents)
        out = pages.dense(0, range(4))
    del pages, held
    others = [torch.empty(end - start, dtype=torch.uint8, device=device) for start, end in spans for _ in range(16)]
    assert not side.query(), 'the stream is done already'
    taken = [(t.data_ptr(), t.data_ptr() + t.nbytes) for t in others]
    assert not any(a < end and start < b for a, b in taken for start, end in spans)
    for t in others:
        t.zero_()
    side.synchronize()
    book.fork(parents.tolist())
    assert torch.equal(out.cpu(), torch.stack([book.dense(0, i) for i in range(4)]))


def test_load_a_part_of_the_pool(device):
    """States that are pages of the pool itself: the sequences' own, which are free behind the first kernel, and others'."""
    for turn in range(3):
        pages, book, gen = make(device, n=3, banks=64, layers=1, s=8, width=16, pages=200, dtype=torch.float32, seed=91)
        states = torch.randn(2, 64, 1, 8, 16, generator=gen)
        pages.load(0, [0, 1], states.to(device))
        book.load(0, [0, 1], states)
        first = (0, 63, 64)[turn]
        part = torch.stack(book.content[first:first + 64]).flip(0)[None]
        pages.pool[first:first + 64] = part[0].to(device)
        for i in range(64):
            book.content[first + i] = part[0, i]
        for row in (1, 2, 0):
            pages.load(0, [row], pages.pool[first:first + 64][None])
            book.load(0, [row], part)
            agree(pages, book)
            part = torch.stack(book.content[first:first + 64])[None].clone()


MANY = [
    # written banks of a step: up to 512, up to 1,024, more (in eight rounds of 1,024 at most); read banks: more than the
    # threads that look them up, with few or no written ones
    (60, 24, 1, 4, 8, 5, 3, 'bf16', 'bf16'), (64, 24, 1, 4, 8, 8, 8, 'fp32', 'fp32'), (100, 24, 1, 4, 8, 7, 2, 'fp32', 'bf16'),
    (128, 24, 1, 8, 16, 8, 8, 'bf16', 'bf16'), (129, 24, 1, 4, 8, 8, 1, 'fp32', 'fp32'), (512, 24, 1, 4, 8, 16, 16, 'fp32', 'bf16'),
    (64, 24, 1, 4, 8, 1, 16, 'fp32', 'fp32'), (64, 24, 1, 4, 8, 0, 16, 'fp32', 'bf16'), (512, 20, 1, 4, 8, 2, 16, 'bf16', 'bf16'),
    (512, 20, 1, 4, 8, 16, 0, 'bf16', 'bf16'),
]


@pytest.mark.parametrize('geometry', MANY, ids=lambda c: 'x'.join(map(str, c)))
def test_decode_of_many(device, geometry):
    test_decode(device, geometry, True)


@pytest.mark.parametrize('n', [4, 64, 129, 256, 257])
def test_fork_of_many_layers(device, n):
    """Enough layers and banks that a workgroup takes 32 columns (16 of more than 256 sequences)."""
    from bdm_amd import BankPages
    print('CASE pages fork of many layers', n, flush=True)
    layers, banks, gen = 8, 1027, torch.Generator().manual_seed(n)
    # a page of each bank for every third sequence, which the two behind it share; every seventh has none
    owner = torch.arange(n) // 3
    table = (torch.arange(layers)[:, None, None] * (n // 3 + 1) + owner[:, None]) * banks + torch.arange(banks)
    table[:, ::7] = -1
    total = layers * (n // 3 + 1) * banks

    def counted(t):
        return torch.bincount(t[t >= 0], minlength=total).int()

    pool = torch.zeros(total, 1, 1, 4, dtype=torch.float32, device=device)
    pages = BankPages.over(pool, table.int().to(device), counted(table).to(device))
    choices = [torch.randint(-1, n, (n,), generator=gen), torch.arange(n) // 4 * 4, torch.randint(-n, n, (n,), generator=gen),
               torch.arange(n - n // 2).flip(0), torch.full((n,), -1)]
    for parents in choices:
        pages.fork(parents.to(device))
        whole = torch.cat([parents, torch.arange(len(parents), n)])
        table = torch.where(whole[:, None] >= 0, table[:, whole.clamp(0)], -1)
        torch.cuda.synchronize()
        assert torch.equal(pages.table.cpu().long(), table)
        references = counted(table)
        assert torch.equal(pages.references.cpu(), references)
        free = torch.zeros((total + 63) // 64 * 64, dtype=torch.int64)
        free[:total] = references == 0
        assert torch.equal(pages.free_bits.cpu(), (free.view(-1, 64) << torch.arange(64)).sum(-1))


def test_the_count_of_used_pages_in_a_graph(device):
    from bdm_amd import BankPages
    pages = BankPages(3, 300_000, banks=64, heads=1, bank_size=1, head_width=4, device=device)
    states = torch.randn(1, 64, 1, 1, 4, generator=torch.Generator().manual_seed(1)).bfloat16().to(device)
    pages.load(0, [0], states)
    pages.used()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        used = pages.used()
    for turn in range(5):
        if turn == 1:
            pages.load(0, [1], states + 1)
        if turn == 2:
            pages.load(0, [2], states + 2)
        if turn == 3:
            pages.release([0, 1])
        torch.ones(1 << 20, device=device).sum()
        graph.replay()
        torch.cuda.synchronize()
        assert int(used) == int((pages.references > 0).sum().cpu()) == (64, 128, 192, 64, 64)[turn]
