"""Page bookkeeping against a sequential restatement: drops, forks, extends
with copy-on-write, lists that name a slot twice, a pool or a table that runs
out, compaction."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import alveare_b200 as ab  # noqa: E402
from alveare_b200 import _lib  # noqa: E402
from paged_util import ints  # noqa: E402


class Model:
    """The bookkeeping on the host, one entry at a time."""

    def __init__(self, slots, width, pages, ps):
        self.table = np.full((slots, width), -1, np.int32)
        self.lens, self.refs, self.ps = np.zeros(slots, np.int32), np.zeros(pages, np.int32), ps
        self.data = np.arange(pages) + 1000  # stands for a page's contents

    def drop(self, s):
        for e, p in enumerate(self.table[s]):
            if p >= 0:
                self.refs[p] -= 1
                self.table[s, e] = -1
        self.lens[s] = 0

    def update(self, free=(), fork=(), extend=()):
        for s in free:
            self.drop(s)
        for p, c in fork:
            if p == c:
                continue
            row, n = self.table[p].copy(), self.lens[p]
            if c != p:
                self.drop(c)
            self.table[c], self.lens[c] = row, n
            for e in row:
                if e >= 0:
                    self.refs[e] += 1
        seqs = [s for s, _ in extend]
        together = len(set(seqs)) == len(seqs)
        before = self.refs.copy()
        used, copied, unmet = 0, 0, -1
        for i, (s, more) in enumerate(extend):
            if not together:
                before = self.refs.copy()
            n, ps = int(self.lens[s]), self.ps
            have, want = -(-n // ps), -(-(n + more) // ps)
            cow = more > 0 and n % ps and before[self.table[s, have - 1]] > 1
            if together and i == 0 or not together:
                pool = [p for p in range(len(before)) if before[p] == 0]
            if want > self.table.shape[1] or want - have + bool(cow) > len(pool):
                unmet = i
                break
            if cow:
                src, dst = int(self.table[s, have - 1]), pool.pop(0)
                self.refs[src] -= 1
                self.refs[dst] = 1
                self.table[s, have - 1] = dst
                self.data[dst] = self.data[src]
                copied += 1
                used += 1
            for e in range(have, want):
                p = pool.pop(0)
                self.table[s, e], self.refs[p] = p, 1
                used += 1
            self.lens[s] = n + more
        return [int((self.refs == 0).sum()), used, copied, unmet]


class Pool:
    def __init__(self, model, layers=2, nkv=2, hd=64):
        S, W = model.table.shape
        P, ps = len(model.refs), model.ps
        self.m = model
        self.table, self.lens, self.refs = ints(model.table.ravel()).view(S, W), ints(model.lens), ints(model.refs)
        self.info = ints([9, 9, 9, 9])
        # every layer's page holds values that name the page, its layer and its side
        ids = torch.tensor(model.data, device="cuda")[None, :, None, None, None]
        lay = torch.arange(layers, device="cuda")[:, None, None, None, None]
        self.k = self.mark(ids, lay, 0).expand(layers, P, nkv, ps, hd).contiguous()
        self.v = self.mark(ids, lay, 1).expand(layers, P, nkv, ps, hd).contiguous()
        self.layers = layers

    @staticmethod
    def mark(ids, lay, side):
        return ((ids * 7 + lay * 3 + side) % 256).to(torch.bfloat16)

    def update(self, free=None, fork=None, extend=None):
        lst = lambda x: None if x is None else ints(np.asarray(x).ravel())
        pair = lambda x: None if x is None else ints(np.asarray(x, np.int32).ravel()).view(-1, 2)
        ab.update_pages(self.k, self.v, self.table, self.lens, self.refs, free=lst(free), fork=pair(fork),
                        extend=pair(extend), info=self.info)
        want = self.m.update(free or (), fork or (), extend or ())
        self.same(want)

    def same(self, info=None):
        _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
        assert np.array_equal(self.table.cpu().numpy(), self.m.table)
        assert np.array_equal(self.lens.cpu().numpy(), self.m.lens)
        assert np.array_equal(self.refs.cpu().numpy(), self.m.refs)
        if info is not None:
            assert self.info.tolist() == info
        # the pages in use hold what they should, whole and in every layer
        live = np.flatnonzero(self.m.refs)
        ids = torch.tensor(self.m.data[live], device="cuda")[None, :, None, None, None]
        lay = torch.arange(self.layers, device="cuda")[:, None, None, None, None]
        at = torch.tensor(live, device="cuda")
        assert (self.k[:, at] == self.mark(ids, lay, 0)).all()
        assert (self.v[:, at] == self.mark(ids, lay, 1)).all()


@pytest.mark.parametrize("ps", [1, 16, 48])
@pytest.mark.parametrize("seed", range(4))
def test_random_turns(ps, seed):
    r = np.random.default_rng(seed)
    S, P = 40, 300
    p = Pool(Model(S, 30, P, ps))
    for _ in range(12):
        free = r.permutation(S)[:r.integers(0, 8)].tolist()
        order = r.permutation(S).tolist()
        n = int(r.integers(0, 10))
        kids, parents = order[:n], order[n:n + 6]
        fork = [(int(r.choice(parents)), c) for c in kids]
        ext = [(int(s), int(r.integers(0, 3 * ps + 2))) for s in r.permutation(S)[:r.integers(0, 25)]]
        p.update(free, fork, ext)


def test_shared_last_page_is_copied_by_every_holder_that_extends():
    p = Pool(Model(6, 8, 40, 16))
    p.update(extend=[(0, 20)])
    p.update(fork=[(0, 1), (0, 2), (0, 3)])
    p.update(extend=[(1, 1), (2, 40), (3, 0)])   # 3 adds nothing: keeps sharing
    p.update(extend=[(0, 1), (3, 1)])
    p.update(free=[0, 1, 2, 3])
    assert int(p.refs.sum()) == 0


def test_lists_that_repeat_a_slot_are_taken_in_order():
    p = Pool(Model(6, 12, 40, 16))
    p.update(extend=[(0, 5), (0, 20), (1, 3), (0, 1)])
    p.update(free=[1, 1], fork=[(0, 1), (1, 2), (0, 1), (3, 3)])   # a child that is a parent too, and a child twice
    p.update(extend=[(2, 1), (1, 1), (2, 17)])
    p.update(free=[0, 1, 2, 0])
    assert int(p.refs.sum()) == 0


def test_pool_and_table_run_out():
    p = Pool(Model(5, 4, 6, 16))
    p.update(extend=[(0, 30), (1, 33), (2, 30), (3, 1)])      # 2 + 3, then 2 do not fit
    p.update(extend=[(3, 65), (4, 1)])                        # past the table's width
    p.update(extend=[(3, 16)])                                # the last page
    p.update(fork=[(0, 4)])
    p.update(extend=[(4, 1)])                                 # the copy finds no page
    p.update(free=[1], extend=[(4, 1)])


def test_thousands_of_entries():
    r = np.random.default_rng(3)
    S = 2500
    p = Pool(Model(S, 6, 9000, 16), layers=1, nkv=1)
    p.update(extend=[(s, int(r.integers(1, 40))) for s in r.permutation(S)])
    order = r.permutation(S)
    p.update(free=order[:1200].tolist())
    p.update(fork=[(int(order[1200 + i % 900]), int(order[i])) for i in range(1200)])
    p.update(extend=[(int(s), 1) for s in r.permutation(S)])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pages,live", [(50, 0.4), (3000, 0.3), (700, 0.0), (700, 1.0), (1, 1.0)])
def test_compact(pages, live, in_place):
    r = np.random.default_rng(pages)
    m = Model(30, max(8, pages // 5 + 2), pages, 16)
    ids = r.permutation(pages)[:int(pages * live)]
    for i, p in enumerate(ids):
        s = i % 30
        e = int((m.table[s] >= 0).sum())
        m.table[s, e] = p
        m.refs[p] += 1
    if len(ids):
        m.table[29, -1] = ids[0]
        m.refs[ids[0]] += 1
    p = Pool(m, layers=3)
    tout = p.table if in_place else torch.full_like(p.table, 5)
    rout = p.refs if in_place else torch.full_like(p.refs, 5)
    info = ints([9, 9])
    ab.compact_pages(p.k, p.v, p.table, p.refs, tout, rout, info=info)
    n = int((m.refs > 0).sum())
    src = [q for q in range(n, pages) if m.refs[q]]
    dst = [q for q in range(n) if not m.refs[q]]
    to = np.arange(pages)
    to[src] = dst
    m.data[dst] = m.data[src]
    refs = np.zeros_like(m.refs)
    refs[to[m.refs > 0]] = m.refs[m.refs > 0]
    m.refs, m.table = refs, np.where(m.table >= 0, to[m.table], -1).astype(np.int32)
    p.table, p.refs = tout, rout
    p.same()
    assert info.tolist() == [n, len(src)]


def test_large_pages_move_whole():
    """Pages of more than one copy unit, with a partial last one."""
    m = Model(2, 4, 6, 80)
    m.table[0, :2], m.table[1, 0], m.refs[[5, 1, 4]] = [5, 1], 4, 1
    p = Pool(m, layers=2, nkv=3, hd=128)
    p.k += torch.arange(128, device="cuda").to(torch.bfloat16) / 256 * 0   # contiguous copy
    g = torch.Generator(device="cuda").manual_seed(0)
    p.k.copy_(torch.randn(p.k.shape, generator=g, device="cuda").to(torch.bfloat16))
    p.v.copy_(torch.randn(p.v.shape, generator=g, device="cuda").to(torch.bfloat16))
    k0, v0 = p.k.clone(), p.v.clone()
    ab.compact_pages(p.k, p.v, p.table, p.refs, p.table, p.refs)
    to = {5: 2, 4: 0, 1: 1}   # in use 1, 4, 5; free below 3: 0, 2
    for s, d in to.items():
        assert torch.equal(p.k[:, d], k0[:, s]) and torch.equal(p.v[:, d], v0[:, s])
    assert p.table.cpu().tolist() == [[2, 1, -1, -1], [0, -1, -1, -1]]


def test_bad_slots_are_skipped_and_reported():
    p = Pool(Model(4, 4, 10, 16))
    ab.update_pages(p.k, p.v, p.table, p.lens, p.refs, free=ints([7]), fork=ints([0, -1]).view(1, 2),
                    extend=ints([99, 3, 1, 5, 2, -1]).view(3, 2), info=p.info)
    with pytest.raises(_lib.AlvError):
        _lib.context(0).sync_status(torch.cuda.current_stream().cuda_stream)
    p.m.update(extend=[(1, 5)])
    p.same()


def test_refusals():
    p = Pool(Model(4, 4, 10, 16))
    up = lambda **kw: ab.update_pages(p.k, p.v, p.table, p.lens, p.refs, **kw)
    with pytest.raises(TypeError):
        up(free=ints([1]).cpu())
    with pytest.raises(TypeError):
        up(free=ints([1]).long())
    with pytest.raises(ValueError):
        up(fork=ints([1, 2]))
    with pytest.raises(ValueError):
        up(extend=ints([1, 2, 3]).view(1, 3))
    with pytest.raises(ValueError):
        up(info=ints([1]))
    with pytest.raises(ValueError):
        ab.update_pages(p.k, p.v[:1], p.table, p.lens, p.refs)
    with pytest.raises(ValueError):
        ab.update_pages(p.k, p.v, p.table, p.lens, p.refs[:5])
    with pytest.raises(ValueError):
        ab.update_pages(p.k.transpose(2, 3), p.v.transpose(2, 3), p.table, p.lens, p.refs)
    with pytest.raises(ValueError):
        ab.compact_pages(p.k, p.v, p.table, p.refs, p.table[:2], p.refs)
    with pytest.raises(_lib.AlvError):   # renumbered in place, but not contiguous
        wide = torch.full((4, 9), -1, dtype=torch.int32, device="cuda")
        pool = ab.paged._pool(0, p.k, p.v, wide[:, :4], None, p.refs)
        ctx = _lib.context(0)
        ctx.check(ctx.lib.alv_pages_compact(ctx.ptr, pool, wide.data_ptr(), p.refs.data_ptr(), None, None),
                  "alv_pages_compact")


def test_cache_class_round_trip():
    c = ab.PagedKVCache(2, 2, 64, 32, page_size=16, slots=4, max_len=100)
    c.update(extend=[(0, 20), (2, 5)])
    assert c.check() == dict(free_pages=29, handed_out=3, copied=0, first_unmet=-1)
    c.update(fork=[(0, 1)], extend=[(1, 1)])
    assert c.check()["copied"] == 1
    b = c.batch([2, 1], [5, 1])
    assert b["kv_lens"].tolist() == [5, 21] and b["q_start"].tolist() == [0, 5, 6]
    assert torch.equal(b["page_table"], c.table[[2, 1]])
    c.update(free=[0])
    c.compact()
    assert int((c.refs > 0).sum()) == int((c.refs[:3] > 0).sum()) == 3
