"""Page bookkeeping of sequences whose `lens` the caller lowered (rejected
tokens): no page is lost, and every count is the number of table entries that
name the page."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402
from paged_util import ints  # noqa: E402


class Twin:
    """A pool and its restatement, one entry at a time, on whole table rows."""

    def __init__(self, slots, width, pages, ps):
        self.ps = ps
        self.t, self.n, self.r = np.full((slots, width), -1, np.int32), np.zeros(slots, np.int32), np.zeros(pages, np.int32)
        self.table, self.lens, self.refs = ints(self.t.ravel()).view(slots, width), ints(self.n), ints(self.r)
        self.k = torch.arange(pages).bfloat16().cuda()[None, :, None, None, None].expand(1, pages, 1, ps, 16).contiguous()
        self.v = self.k.clone()
        self.data = np.arange(pages)
        self.info = ints([0] * 4)

    def shorten(self, slot, n):
        self.n[slot] = n
        self.lens[slot] = n

    def drop(self, s):
        for p in self.t[s][self.t[s] >= 0]:
            self.r[p] -= 1
        self.t[s], self.n[s] = -1, 0

    def update(self, free=(), fork=(), extend=()):
        lst = lambda x: ints(x) if len(x) else None
        pair = lambda x: ints(np.ravel(x)).view(-1, 2) if len(x) else None
        ab.update_pages(self.k, self.v, self.table, self.lens, self.refs, free=lst(free), fork=pair(fork),
                        extend=pair(extend), info=self.info)
        for s in free:
            self.drop(s)
        for a, b in fork:
            row, n = self.t[a].copy(), self.n[a]
            self.drop(b)
            self.t[b], self.n[b] = row, n
            for p in row[row >= 0]:
                self.r[p] += 1
        together = len({s for s, _ in extend}) == len(extend)
        gone = []   # pages that entries past a length named: dropped when all is done
        used = copied = 0
        unmet = -1
        before = pool = None
        for i, (s, more) in enumerate(extend):
            if pool is None or not together:
                before, pool = self.r.copy(), [p for p in range(self.r.size) if self.r[p] == 0]
            n = int(self.n[s])
            have, want = -(-n // self.ps), -(-(n + more) // self.ps)
            cow = bool(more > 0 and n % self.ps and before[self.t[s, have - 1]] > 1)
            if want > self.t.shape[1] or want - have + cow > len(pool):
                unmet = i
                break
            if cow:
                src, dst = int(self.t[s, have - 1]), pool.pop(0)
                self.r[src] -= 1
                self.r[dst], self.t[s, have - 1], self.data[dst] = 1, dst, self.data[src]
            for e in range(have, want):
                if self.t[s, e] >= 0:
                    gone.append(int(self.t[s, e]))
                self.t[s, e] = pool.pop(0)
                self.r[self.t[s, e]] = 1
            used += want - have + cow
            copied += cow
            self.n[s] = n + more
        for p in gone:
            self.r[p] -= 1
        _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
        named = np.bincount(self.t[self.t >= 0], minlength=self.r.size)
        assert np.array_equal(named, self.r)
        assert np.array_equal(self.table.cpu().numpy(), self.t)
        assert np.array_equal(self.refs.cpu().numpy(), self.r)
        assert np.array_equal(self.lens.cpu().numpy(), self.n)
        assert self.info.tolist() == [int((self.r == 0).sum()), used, copied, unmet]
        live = np.flatnonzero(self.r)
        want = torch.tensor(self.data[live]).bfloat16().cuda()[:, None, None, None]
        at = torch.tensor(live, device="cuda")
        assert (self.k[0, at] == want).all() and (self.v[0, at] == want).all()


def test_dropping_a_shortened_sequence_drops_all_its_pages():
    p = Twin(4, 8, 20, 16)
    p.update(extend=[(0, 100), (1, 30)])
    p.shorten(0, 17)
    p.update(free=[0])
    assert int((p.refs > 0).sum()) == 2


def test_forking_to_and_from_a_shortened_sequence():
    p = Twin(4, 8, 20, 16)
    p.update(extend=[(0, 100), (1, 60)])
    p.shorten(0, 40)
    p.shorten(1, 3)
    p.update(fork=[(0, 1), (0, 2)])
    p.update(free=[0, 1])
    p.update(free=[2])
    assert int(p.refs.sum()) == 0


def test_extending_a_shortened_sequence_loses_no_page():
    p = Twin(4, 8, 20, 16)
    p.update(extend=[(0, 100), (1, 30)])
    p.shorten(0, 17)
    p.update(extend=[(0, 40)])
    p.update(fork=[(0, 2)])
    p.shorten(0, 5)
    p.update(extend=[(0, 30), (2, 1)])
    p.update(free=[0, 1, 2])
    assert int(p.refs.sum()) == 0


def test_a_page_dropped_by_an_extend_is_not_handed_out_in_the_same_call():
    """(Its contents may be the source of a copy that the call has yet to make.)"""
    p = Twin(4, 6, 8, 16)
    p.update(extend=[(0, 20)])
    p.update(fork=[(0, 1)])
    p.shorten(0, 10)
    # slot 1 copies the page that slot 0 then drops; slot 2 takes more pages after that
    p.update(extend=[(1, 1), (0, 10), (2, 16), (0, 1)])
    p.update(free=[0, 1, 2])
    assert int(p.refs.sum()) == 0


@pytest.mark.parametrize("ps", [1, 16])
@pytest.mark.parametrize("seed", range(6))
def test_random_turns(ps, seed):
    r = np.random.default_rng(seed)
    S = 40
    p = Twin(S, 40, 500, ps)
    for _ in range(12):
        for s in r.permutation(S)[:10]:
            if p.n[s]:
                p.shorten(int(s), int(r.integers(0, p.n[s] + 1)))
        order = r.permutation(S).tolist()
        n = int(r.integers(0, 6))
        fork = [(int(r.choice(order[n:n + 6])), c) for c in order[:n]]
        ext = [(int(s), int(r.integers(0, 4 * ps + 2))) for s in r.permutation(S)[:r.integers(0, 25)]]
        if seed % 2 and ext:
            ext += [ext[0], ext[-1]]
        p.update(r.permutation(S)[:r.integers(0, 4)].tolist(), fork, ext)
    p.update(free=list(range(S)))
    assert int(p.refs.sum()) == 0


def test_thousands_of_entries():
    r = np.random.default_rng(3)
    S = 2500
    p = Twin(S, 6, 16000, 16)
    p.update(extend=[(int(s), int(r.integers(40, 90))) for s in r.permutation(S)])
    for s in range(0, S, 3):
        p.n[s] = int(r.integers(0, 40))
    p.lens.copy_(ints(p.n))
    p.update(extend=[(int(s), int(r.integers(0, 6))) for s in r.permutation(S)])
    p.update(free=list(range(S)))
    assert int(p.refs.sum()) == 0
