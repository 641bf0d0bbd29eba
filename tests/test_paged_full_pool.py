"""A paged cache whose pool is short of pages: every token that a row counts is the one that was stored for it,
whoever shares its pages and whoever was refused.  The tables' functions are held against lists of token numbers,
not against the oracle, which has the same rules; on the CPU it is the oracle that is tested so."""
import random

import pytest
import torch

from oracle import paged as op


def _ints(x, dev=None):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class _OnTheOracle:
    dev = "cpu"

    @staticmethod
    def extend(table, lens, add, uses, page, most, cache):
        slots, n, t, u, c = op.extend_pages(table, lens, add, uses, page, most, cache)
        table.copy_(t)
        uses.copy_(u)
        for a, b in zip(cache[0], c[0]):
            a.copy_(b)
        return slots, n

    @staticmethod
    def reorder(table, lens, parents, uses, page):
        n, t, u = op.reorder_pages(table, lens, parents, uses, page)
        table.copy_(t)
        uses.copy_(u)
        return n


class _OnTheGpu:
    def __init__(self, dev):
        from fxlm import extend_pages, reorder_pages
        self.dev, self.extend, self.reorder = dev, extend_pages, reorder_pages


class _Rows:
    """Rows of a paged cache whose tokens are numbers, each in a pool's row as digits to base 128."""

    def __init__(self, on, R, N, P, M):
        self.on, self.P, dev = on, P, on.dev
        self.table, self.lens = torch.full((R, M), -1, dtype=torch.int32, device=dev), torch.zeros(R, dtype=torch.int32, device=dev)
        self.uses = torch.zeros(N, dtype=torch.int32, device=dev)
        self.pool = torch.zeros(2, N, P, 1, 8, device=dev).bfloat16()
        self.want, self.next = [[] for _ in range(R)], 1

    def extend(self, add, most):
        """Tokens for every row that gets its slots; returns the slots as lists."""
        slots, n = self.on.extend(self.table, self.lens, _ints(add, self.on.dev), self.uses, self.P, most, [(self.pool[0], self.pool[1])])
        self.lens.copy_(n)
        slots = slots.cpu()
        ids, at = [], []
        for r in range(len(add)):
            for j in range(min(add[r], most)):
                if int(slots[r, j]) >= 0:
                    at.append(int(slots[r, j]))
                    ids.append(self.next)
                    self.want[r] = self.want[r] + [self.next]
                    self.next += 1
        assert len(set(at)) == len(at)
        if at:
            self.pool.view(2, -1, 8)[:, torch.tensor(at, device=self.on.dev)] = self._digits(torch.tensor(ids)).to(self.on.dev)
        return slots.tolist()

    @staticmethod
    def _digits(ids):
        return torch.stack([ids >> 7 * i & 127 for i in range(8)], -1).bfloat16()

    def reorder(self, parents):
        self.lens.copy_(self.on.reorder(self.table, self.lens, _ints(parents, self.on.dev), self.uses, self.P))
        self.want = [self.want[p] if p >= 0 else [] for p in parents]

    def check(self):
        assert self.lens.tolist() == [len(w) for w in self.want]
        table, pool, P = self.table.cpu(), self.pool.cpu().view(2, -1, 8), self.P
        for r, w in enumerate(self.want):
            if w:
                at = torch.tensor([int(table[r, j // P]) * P + j % P for j in range(len(w))])
                assert torch.equal(pool[:, at], self._digits(torch.tensor(w)).expand(2, -1, -1)), r


def _longer_holder(on, R):
    # two rows of 5 tokens on one page and none free; the one that went on becomes the higher row.  The rows between them hold nothing.
    c = _Rows(on, R, 1, 16, 2)
    par, one = list(range(R)), [0] * R
    c.extend([5] + one[1:], 5)
    par[R - 1] = 0
    c.reorder(par)
    one[0] = one[R - 1] = 1
    first = c.extend(one, 1)
    assert first[0] == [5] and first[R - 1] == [-1]    # of equals the lower row keeps the page
    c.check()
    par[0], par[R - 1] = R - 1, 0
    c.reorder(par)
    slots = c.extend(one, 1)
    c.check()
    assert slots[0] == [-1] and slots[R - 1] == [6] and c.lens[[0, R - 1]].tolist() == [5, 7]
    # alone on the page, the shorter one writes where the other's token was
    par[R - 1] = -1
    par[0] = 0
    c.reorder(par)
    assert c.extend(one, 1)[0] == [5]
    c.check()


def _unlike_holders(on, R):
    # rows of unlike lengths on one page, pages for some: the longest keeps it, the others have copies in the rows' order
    c = _Rows(on, R, 3, 16, 2)
    c.extend([9] + [0] * (R - 1), 9)
    a, b, d = 1, R // 2, R - 1
    for r in (a, b, d):     # forks, a token further each; the page's other holders wait: no one is in another's way
        par = list(range(R))
        par[r] = 0
        c.reorder(par)
    c.uses[1:] = 1          # no page is free
    one = [0] * R
    one[0] = one[a] = one[b] = one[d] = 1
    c.extend(one, 1)        # row 0 alone goes on
    assert c.lens[[0, a, b, d]].tolist() == [10, 9, 9, 9]
    par = list(range(R))
    par[0], par[b] = b, 0   # and becomes row b
    c.reorder(par)
    c.uses[1:] = 0
    slots = c.extend(one, 1)
    c.check()
    assert [slots[r][0] for r in (0, a, b, d)] == [25, 41, 10, -1] and c.uses.tolist() == [2, 1, 1]


def _walk(on, R, N, P, M, seed, steps=40):
    r = random.Random(seed)
    c, refused = _Rows(on, R, N, P, M), 0
    for step in range(steps):
        most = r.choice([1, 1, 1, 3, P + 3])
        add = [(r.randint(1, most) if r.random() < 0.8 else 0) if c.want[i] or r.random() < 0.3 else 0 for i in range(R)]
        slots = c.extend(add, most)
        refused += sum(n > 0 and s[0] < 0 for n, s in zip(add, slots))
        c.check()
        c.reorder([r.choice([i, i, i, r.randrange(R), -1]) if r.random() < 0.5 else i for i in range(R)])
        c.check()
        held = torch.zeros(N, dtype=torch.int32)
        for i, w in enumerate(c.want):
            for x in c.table[i, :-(-len(w) // P)].tolist():
                held[x] += 1
        assert torch.equal(c.uses.cpu(), held)
    return refused


@pytest.mark.parametrize("R", [2, 5])
def test_the_longest_holder_keeps_a_page(R):
    _longer_holder(_OnTheOracle, R)


def test_holders_of_unlike_lengths():
    _unlike_holders(_OnTheOracle, 4)


def test_rows_of_a_short_pool():
    assert sum(_walk(_OnTheOracle, 10, 8, 16, 3, seed) for seed in range(60)) > 0


# the forms for few rows (256), for as many as one thread takes (1,024) and for more
@pytest.mark.gpu
@pytest.mark.parametrize("R", [2, 256, 257, 1024, 1025, 8192])
def test_the_longest_holder_keeps_a_page_gpu(dev, R):
    _longer_holder(_OnTheGpu(dev), R)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [4, 300, 2000])
def test_holders_of_unlike_lengths_gpu(dev, R):
    _unlike_holders(_OnTheGpu(dev), R)


@pytest.mark.gpu
@pytest.mark.parametrize("R,N,P,M,seeds", [(10, 8, 16, 3, 12), (10, 4, 64, 2, 6), (300, 150, 16, 3, 2), (1100, 600, 16, 3, 1)])
def test_rows_of_a_short_pool_gpu(dev, R, N, P, M, seeds):
    assert sum(_walk(_OnTheGpu(dev), R, N, P, M, seed, 25) for seed in range(seeds)) > 0
