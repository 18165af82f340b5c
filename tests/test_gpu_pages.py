"""Page calls against a plain bookkeeping of them: bit for bit, data and statuses."""
import numpy as np
import pytest
import torch

from qengine_amd import kvcache
from tests import _paged8 as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


class Pool:
    """Both sides' tables, counts and planes."""

    def __init__(self, n_slots, max_blocks, n_pages, bt, plane_bytes=(1024, 20, 7), seed=0):
        rng = np.random.default_rng(seed)
        self.bt = bt
        self.tables = np.full((n_slots, max_blocks), -1, np.int32)
        self.refs = np.zeros(n_pages, np.int32)
        self.data = [rng.integers(0, 256, (n_pages, b)).astype(np.uint8) for b in plane_bytes]
        self.rng = rng

    def fill(self, lens):
        order = list(self.rng.permutation(len(self.refs)))
        for s, n in enumerate(lens):
            for b in range(-(-n // self.bt)):
                p = order.pop()
                self.tables[s, b] = p
                self.refs[p] = 1

    def put(self):
        self.t, self.r = i32(self.tables), i32(self.refs)
        self.d = [torch.from_numpy(x.copy()).to(DEV) for x in self.data]
        self.planes = kvcache.page_planes(self.d)

    def copied(self, pairs):
        src = [x.copy() for x in self.data]
        for a, b in pairs:
            if a >= 0:
                for x, y in zip(self.data, src):
                    x[b] = y[a]

    def check(self):
        assert np.array_equal(self.t.cpu().numpy(), self.tables)
        assert np.array_equal(self.r.cpu().numpy(), self.refs)
        for x, y in zip(self.d, self.data):
            assert np.array_equal(x.cpu().numpy(), y)


@pytest.mark.parametrize("bt", [1, 16, 48])
def test_fork_reserve_release(bt):
    """Parents forked, every slot's next tokens reserved, children cut back and released."""
    p = Pool(12, 40, 300, bt, seed=bt)
    lens = [bt * 5 + bt // 2, bt * 3, 1, bt * 30 + 1, 0]
    p.fill(lens)
    p.put()
    parents, children = [0, 0, 3, 1, 2], [5, 6, 7, 8, 9]
    tok = [lens[0], bt * 2, lens[3], lens[1], lens[2]]
    st = i32([9] * 5)
    want = R.fork(p.tables, p.refs, parents, children, tok, bt)
    kvcache.pages_fork(p.t, p.r, i32(parents), i32(children), i32(tok), st, block_tokens=bt)
    assert st.tolist() == want == [0] * 5
    p.check()

    slots = [0, 5, 6, 3, 7, 4, 8, 9]
    pos = [lens[0], lens[0], bt * 2, lens[3], lens[3], 0, lens[1], lens[2]]
    new = [3, 3, 1, 2 * bt + 1, 1, 4 * bt, 0, 2]
    st = i32([9] * 8)
    want, pairs = R.reserve(p.tables, p.refs, slots, pos, new, 4 * bt + 3, bt)
    scratch = torch.zeros(10000, dtype=torch.int32, device=DEV)
    kvcache.pages_reserve(p.t, p.r, i32(slots), i32(pos), i32(new), st, p.planes, block_tokens=bt, max_new=4 * bt + 3,
                          scratch=scratch)
    p.copied(pairs)
    assert st.tolist() == want
    assert scratch[:16].view(8, 2).tolist() == [list(x) for x in pairs]
    p.check()

    slots, keep = [5, 7, 0, 9, 4], [0, bt * 3 + 1, 1, 0, 10 ** 9]
    st = i32([9] * 5)
    want = R.release(p.tables, p.refs, slots, keep, bt)
    kvcache.pages_release(p.t, p.r, i32(slots), i32(keep), st, block_tokens=bt)
    assert st.tolist() == want
    p.check()


def test_entries_that_are_refused_change_nothing():
    p = Pool(6, 4, 40, 16, seed=3)
    p.fill([60, 20, 5])
    p.tables[3, 1] = 99   # past the pool
    p.put()
    par, chi, tok = [0, 1, 0, -1, 0, 6, 0, 3, 2], [4, 4, 0, 5, 1, 5, 5, 5, 3], [60, 20, 5, 5, 3, 1, 65, 20, 5]
    n = 6   # (a list is at most as long as there are slots)
    for lo in (0, 3):
        a, b, c = par[lo:lo + n], chi[lo:lo + n], tok[lo:lo + n]
        st = i32([9] * n)
        want = R.fork(p.tables, p.refs, a, b, c, 16)
        kvcache.pages_fork(p.t, p.r, i32(a), i32(b), i32(c), st, block_tokens=16)
        assert st.tolist() == want and R.INVALID in want
        p.check()
    st = i32([9] * 6)
    args = [0, 0, -1, 6, 3, 2], [60, 10, 0, 0, 16, 5], [4, 1, 1, 1, 1, 99]
    want, pairs = R.reserve(p.tables, p.refs, *args, 8, 16)
    kvcache.pages_reserve(p.t, p.r, *map(i32, args), st, p.planes, block_tokens=16, max_new=8)
    assert st.tolist() == want == [0, -1, -1, -1, -1, -1]
    p.copied(pairs)
    p.check()
    st = i32([9] * 5)
    want = R.release(p.tables, p.refs, [2, 2, 7, 0, -1], [0, 0, 0, -1, 0], 16)
    kvcache.pages_release(p.t, p.r, i32([2, 2, 7, 0, -1]), i32([0, 0, 0, -1, 0]), st, block_tokens=16)
    assert st.tolist() == want
    p.check()


def test_reserve_when_pages_run_out():
    """Served in list order while the pages last, and a slot that wants none is always served."""
    p = Pool(5, 8, 12, 16, seed=4)
    p.fill([40, 40, 40])   # 9 of 12 pages
    p.put()
    args = [0, 3, 1, 4, 2], [40, 0, 48, 0, 40], [8, 40, 8, 1, 4]
    st = i32([9] * 5)
    want, pairs = R.reserve(p.tables, p.refs, *args, 40, 16)
    kvcache.pages_reserve(p.t, p.r, *map(i32, args), st, p.planes, block_tokens=16, max_new=40)
    assert st.tolist() == want == [0, 0, -9, -9, 0]
    p.check()


def test_every_sharer_writes():
    """All sharers of a page reserve at once: each gets a copy and the page is free again."""
    p = Pool(4, 4, 20, 16, seed=5)
    p.fill([21])
    p.put()
    R.fork(p.tables, p.refs, [0, 0, 0], [1, 2, 3], [21, 21, 21], 16)
    kvcache.pages_fork(p.t, p.r, i32([0] * 3), i32([1, 2, 3]), i32([21] * 3), block_tokens=16)
    args = [0, 1, 2, 3], [21] * 4, [1] * 4
    want, pairs = R.reserve(p.tables, p.refs, *args, 1, 16)
    kvcache.pages_reserve(p.t, p.r, *map(i32, args), None, p.planes, block_tokens=16, max_new=1)
    p.copied(pairs)
    assert sum(a >= 0 for a, _ in pairs) == 4 and (p.refs == 0).sum() == 20 - 5
    p.check()


@pytest.mark.parametrize("n", [1, 7, 1024])
def test_reserve_of_many_slots(n):
    p = Pool(n, 5, 6000, 16, plane_bytes=(32,), seed=n)
    lens = list(p.rng.integers(0, 60, n))
    p.fill(lens)
    p.put()
    slots = list(p.rng.permutation(n))
    pos = [int(lens[s]) for s in slots]
    new = [int(x) for x in p.rng.integers(0, 18, n)]
    st = i32([9] * n)
    want, pairs = R.reserve(p.tables, p.refs, slots, pos, new, 17, 16)
    kvcache.pages_reserve(p.t, p.r, i32(slots), i32(pos), i32(new), st, p.planes, block_tokens=16, max_new=17)
    p.copied(pairs)
    assert st.tolist() == want
    p.check()


@pytest.mark.parametrize("n_pages,keep", [(1, 1.0), (50, 0.5), (3000, 0.3), (5000, 0.9), (2100, 0.0)])
def test_compact(n_pages, keep):
    p = Pool(9, n_pages // 8 + 1, n_pages, 16, plane_bytes=(64, 3, 40000) if n_pages <= 50 else (48, 4), seed=n_pages)
    for page in np.flatnonzero(p.rng.random(n_pages) < keep):
        s, b = int(p.rng.integers(0, 9)), int(p.rng.integers(0, p.tables.shape[1]))
        if p.tables[s, b] < 0:
            p.tables[s, b] = page
            p.refs[page] = 1
    if p.refs.any():   # shared pages
        s = int(np.argmax((p.tables >= 0).any(1)))
        b = int(np.argmax(p.tables[s] >= 0))
        free = np.argwhere(p.tables < 0)
        if len(free):
            p.tables[tuple(free[0])] = p.tables[s, b]
            p.refs[p.tables[s, b]] += 1
    p.put()
    moved, used = i32([7] * n_pages), i32([7])
    want, n = R.compact(p.tables, p.refs)
    kvcache.pages_compact(p.t, p.r, moved, used, p.planes)
    src = [x.copy() for x in p.data]
    for a, b in enumerate(want):
        if b >= 0 and a != b:
            for x, y in zip(p.data, src):
                x[b] = y[a]
    assert np.array_equal(moved.cpu().numpy(), want) and used.item() == n
    p.check()


def test_copy_planes_of_every_alignment():
    """16-, 4- and 1-byte planes, more than one chunk, pairs out of range left out."""
    p = Pool(1, 1, 9, 16, plane_bytes=(16384 * 2 + 48, 16388, 33, 16), seed=6)
    p.put()
    pairs = [(0, 8), (3, 1), (-1, 2), (2, -1), (9, 2), (4, 4), (5, 7)]
    kvcache.pages_copy(p.planes, i32(pairs))
    p.copied([x for x in pairs if x in ((0, 8), (3, 1), (5, 7))])
    p.check()


def test_offsets_past_four_gigabytes():
    """A plane of more than 2^32 bytes: its last page."""
    n, b = 4200, 1 << 20
    big = torch.zeros(n, b, dtype=torch.uint8, device=DEV)
    big[4195] = 77
    kvcache.pages_copy(kvcache.page_planes([big]), i32([(4195, 4199)]))
    assert (big[4199] == 77).all() and (big[4194] == 0).all() and (big[3] == 0).all()


def test_scratch_on_a_given_stream():
    """With stream= and no scratch the plan lies in that stream's memory, not in a block that the current stream
    gave back and may still write; the calls' results are the same."""
    s = torch.cuda.Stream()
    lent = torch.empty(10000, dtype=torch.int32, device=DEV)   # a block for the current stream to have at hand
    del lent
    t = kvcache._scratch(40000, torch.device(DEV), s)
    owner = [x["stream"] for x in torch.cuda.memory_snapshot() if x["address"] <= t.data_ptr() < x["address"] + x["total_size"]]
    assert owner == [s.cuda_stream]

    p = Pool(6, 20, 200, 16, plane_bytes=(4096, 20), seed=11)
    p.fill([100, 37, 5, 0, 0, 0])
    p.put()
    st = i32([9] * 3)
    calls = [i32(x) for x in ([0, 1, 0], [3, 4, 5], [100, 37, 90])], [i32(x) for x in ([0, 3, 4], [100, 100, 37], [1, 40, 3])]
    back, keep, moved, used = i32([0, 5]), i32([0, 33]), i32([0] * 200), i32([0])
    R.fork(p.tables, p.refs, [0, 1, 0], [3, 4, 5], [100, 37, 90], 16)
    s.wait_stream(torch.cuda.current_stream())
    kvcache.pages_fork(p.t, p.r, *calls[0], block_tokens=16, stream=s)
    kvcache.pages_reserve(p.t, p.r, *calls[1], st, p.planes, block_tokens=16, max_new=40, stream=s)
    want, pairs = R.reserve(p.tables, p.refs, [0, 3, 4], [100, 100, 37], [1, 40, 3], 40, 16)
    p.copied(pairs)
    kvcache.pages_release(p.t, p.r, back, keep, block_tokens=16, stream=s)
    R.release(p.tables, p.refs, [0, 5], [0, 33], 16)
    kvcache.pages_compact(p.t, p.r, moved, used, p.planes, stream=s)
    to, n = R.compact(p.tables, p.refs)
    src = [x.copy() for x in p.data]
    for a, b in enumerate(to):
        if b >= 0 and a != b:
            for x, y in zip(p.data, src):
                x[b] = y[a]
    s.synchronize()
    assert st.tolist() == want == [0] * 3 and used.item() == n and np.array_equal(moved.cpu().numpy(), to)
    p.check()


def test_captured_without_scratch():
    """Release, reserve and compact in one graph, their scratch out of the graph's own memory: every replay, with
    eager calls and other allocations between, as the bookkeeping."""
    p = Pool(5, 30, 120, 16, plane_bytes=(4096, 20), seed=12)
    p.fill([100, 37, 5, 0, 60])
    p.put()
    slots, pos, new = list(range(5)), np.array([100, 37, 5, 0, 60]), [3, 17, 1, 2, 0]
    back, keep = i32([4]), i32([9])
    sl, at, nw, moved, used, st = i32(slots), i32(pos), i32(new), i32([0] * 120), i32([0]), i32([9] * 5)

    def step():
        kvcache.pages_release(p.t, p.r, back, keep, block_tokens=16)
        kvcache.pages_reserve(p.t, p.r, sl, at, nw, st, p.planes, block_tokens=16, max_new=20)
        kvcache.pages_compact(p.t, p.r, moved, used, p.planes)

    def plain():
        R.release(p.tables, p.refs, [4], [9], 16)
        want, pairs = R.reserve(p.tables, p.refs, slots, [int(x) for x in pos], new, 20, 16)
        p.copied(pairs)
        to, n = R.compact(p.tables, p.refs)
        src = [x.copy() for x in p.data]
        for a, b in enumerate(to):
            if b >= 0 and a != b:
                for x, y in zip(p.data, src):
                    x[b] = y[a]
        return want, n
    R.fork(p.tables, p.refs, [0], [3], [100], 16)
    kvcache.pages_fork(p.t, p.r, i32([0]), i32([3]), i32([100]), block_tokens=16)
    pos[3] = 100
    at.copy_(i32(pos))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    p.check()   # (capturing runs nothing)
    for turn in range(9):
        junk = [torch.full((n,), -7, dtype=torch.int32, device=DEV) for n in (16, 34, 122, 500)]
        if turn % 3 == 1:
            step()
        else:
            g.replay()
        want, n = plain()
        assert st.tolist() == want and used.item() == n, turn
        p.check()
        del junk
        pos[:4] += new[:4]
        pos[4] = 9
        at.copy_(i32(pos))
