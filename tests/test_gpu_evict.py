"""Eviction from the paged 8-bit cache against the definition: byte for byte."""
import numpy as np
import pytest
import torch

from qengine_amd import kvcache
from tests import _loop as L
from tests import _paged8 as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _t(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def _cache(rng, lens, bt, kv, hd, ties=False):
    tables, _, _, n_pages = R.layout(rng, lens, [0] * len(lens), bt, kv, hd, max_blocks=max(-(-max(lens) // bt), 1) + 1)
    kp, ke = R.random_pool(rng, n_pages, bt, kv, hd)
    vp, ve = R.random_pool(rng, n_pages, bt, kv, hd)
    w = rng.random((n_pages, kv, bt)) ** 8 if not ties else rng.integers(0, 4, (n_pages, kv, bt))
    return tables, [kp, vp], [ke, ve], w.astype(np.float32)


def _run(tables, pools, exps, w, lens, keep, max_ctx, max_keep, sink=0, recent=0, stream=None, ws=None):
    d = [_t(x) for x in (*pools, *exps, w)]
    kept = torch.full((len(lens), w.shape[1], max_keep), 99, dtype=torch.int32, device=DEV)
    bt = w.shape[2]
    ws = kvcache.evict_f8_paged_workspace(len(lens), w.shape[1], bt, max_ctx, max_keep, DEV) if ws is None else ws
    kvcache.evict_f8_paged(*d, _t(tables), _t(np.array(lens, np.int32)), _t(np.array(keep, np.int32)), kept, ws,
                           max_ctx=max_ctx, sink=sink, recent=recent, stream=stream)
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in d] + [kept.cpu().numpy()]


def _check(tables, pools, exps, w, lens, keep, max_ctx, max_keep, sink=0, recent=0, **kw):
    got = _run(tables, pools, exps, w, lens, keep, max_ctx, max_keep, sink, recent, **kw)
    before = [x.copy() for x in (*pools, *exps, w)]
    kept = L.evict(pools, exps, w, tables, lens, keep, max_ctx, max_keep, sink, recent)
    for a, b, what in zip(got, (*pools, *exps, w, kept), ("k", "v", "k_exp", "v_exp", "weights", "kept")):
        assert np.array_equal(a, b, equal_nan=what == "weights"), what
    return before, kept


@pytest.mark.parametrize("hd,kv,bt", [(128, 4, 16), (256, 4, 64), (128, 1, 256), (256, 2, 16), (128, 8, 48), (256, 1, 512)])
def test_against_the_definition(hd, kv, bt):
    rng = np.random.default_rng(hd + bt)
    lens = [700, 1, 0, 33, 512, 1500, 64, 17]
    keep = [300, 1, 0, 40, 511, 64, 1, 0]
    for sink, recent in ((0, 0), (4, 20), (1000, 3), (5, 1000)):
        _check(*_cache(rng, lens, bt, kv, hd), lens, keep, 1500, 600, sink, recent)


@pytest.mark.parametrize("bt", [16, 64])
def test_ties_go_to_the_lowest_row(bt):
    rng = np.random.default_rng(bt)
    lens = [900, 130, 2000]
    _check(*_cache(rng, lens, bt, 2, 128, ties=True), lens, [333, 100, 1999], 2048, 2000, 2, 7)
    c = _cache(rng, lens, bt, 2, 128)
    c[3][:] = 0   # all the same
    _, kept = _check(*c, lens, [10, 129, 500], 2048, 500, 0, 4)
    assert (kept[0, 0, :6] == np.arange(6)).all() and (kept[0, 0, 6:10] == np.arange(896, 900)).all()


def test_weights_of_every_kind():
    """Negative ones, both zeros, infinities, NaN, subnormals and the largest."""
    rng = np.random.default_rng(3)
    lens = [640]
    c = _cache(rng, lens, 16, 1, 128)
    kinds = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 1e-45, -1e-45, 3.4e38, -3.4e38, 1.0, -1.0, 2.0], np.float32)
    c[3][:] = kinds[rng.integers(0, len(kinds), c[3].shape)]
    for k in (1, 60, 200, 350, 500, 600, 639):
        _check(*[x.copy() if isinstance(x, np.ndarray) else [y.copy() for y in x] for x in c], lens, [k], 640, 640)


@pytest.mark.parametrize("hd", [128, 256])
def test_long_slots(hd):
    """Past what a workgroup's registers hold, many chunks a head."""
    rng = np.random.default_rng(hd)
    lens = [40000, 20000, 16385]
    c = _cache(rng, lens, 64, 1, hd)
    _check(*c, lens, [15000, 19990, 3], 40000, 20000, 4, 100)


def test_long_slots_ties_and_kinds():
    """More equal weights than a stretch of rows holds, NaN and infinities among them; every number kept."""
    rng = np.random.default_rng(11)
    lens = [30000, 17000, 4096 + 30, 4097, 100, 0]
    for sink, recent in ((0, 0), (30, 1)):
        c = _cache(rng, lens, 256, 1, 128, ties=True)
        kinds = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 1e-45, 3.4e38, -1.0], np.float32)
        c[3][:c[3].shape[0] // 2] = kinds[rng.integers(0, len(kinds), c[3][:c[3].shape[0] // 2].shape)]
        _check(*c, lens, [29000, 1, 4096, 2000, 99, 5], 30000, 29000, sink, recent)
    c = _cache(rng, lens, 256, 1, 128)
    c[3][:] = 1
    _, kept = _check(*c, lens, [12345, 16999, 10, 4096, 0, 0], 30000, 17000)
    assert (kept[0, 0, :12345] == np.arange(12345)).all()


def test_almost_all_stays_and_next_to_nothing():
    rng = np.random.default_rng(5)
    lens = [5000, 5000, 5000]
    c = _cache(rng, lens, 32, 2, 128)
    c[3][c[0][1][0], :, 0] = 0
    c[3][c[0][1][0], :, 0] -= 1    # the slot's first row goes: everything moves by one
    _check(*c, lens, [4999, 4999, 1], 5000, 5000)


def test_raised_exponents_and_rows_that_stay():
    """Rows that do not move are requantized where a louder row joins their page; pages ahead of the first that changes are
    not written."""
    rng = np.random.default_rng(6)
    bt, lens = 16, [160]
    tables, pools, exps, w = _cache(rng, lens, bt, 1, 128)
    w[:] = 1
    w[tables[0][1], 0, 10:] = 0       # rows 26 .. 31 go, in whose place quieter or louder rows come
    for e in exps:
        e[tables[0][:2]] = 100
        e[tables[0][2:]] = 106
    before, kept = _check(tables, pools, exps, w, lens, [154], 160, 160)
    assert (kept[0, 0] == np.r_[0:26, 32:160, [-1] * 6]).all()
    for a, b in zip(before[:2], pools):
        assert np.array_equal(a[tables[0][0]], b[tables[0][0]]) and not np.array_equal(a[tables[0][1], :10], b[tables[0][1], :10])


def test_slots_that_are_left_alone():
    rng = np.random.default_rng(7)
    lens = [100, 100, 100, 100, 100, 100, 100]
    c = _cache(rng, lens, 16, 2, 128)
    c[0][4][3] = -1
    c[0][5][6] = 10 ** 6
    lens[1], lens[2] = -1, 101
    before, kept = _check(*c, lens, [50, 50, 50, -1, 50, 50, 60], 100, 55)
    assert (kept[1:] == -1).all() and (kept[0, :, :50] >= 0).all()
    # a length past the table, and one past max_keep that would not move
    _, kept = _check(*_cache(rng, [64, 64], 16, 1, 128), [90, 64], [10, 64], 100, 50)
    assert (kept == -1).all()


def test_shared_first_pages():
    """Slots that share the pages of a protected beginning: those are not written, each keeps its own rest."""
    rng = np.random.default_rng(8)
    bt = 16
    tables, pools, exps, w = _cache(rng, [200, 200], bt, 2, 128)
    tables[1, :4] = tables[0, :4]
    for e in exps:
        e[:] = 110
    before, kept = _check(tables, pools, exps, w, [200, 200], [120, 90], 200, 120, sink=64, recent=8)
    for a, b in zip(before[:2], pools):
        assert np.array_equal(a[tables[0, :4]], b[tables[0, :4]])


def test_captured_and_on_a_stream_with_a_larger_workspace():
    rng = np.random.default_rng(9)
    lens, keep = [1000, 300], [400, 299]
    c = _cache(rng, lens, 16, 2, 128)
    ws = kvcache.evict_f8_paged_workspace(8, 4, 16, 4096, 2048, DEV)
    ws.fill_(255)
    copy = lambda: [x.copy() if isinstance(x, np.ndarray) else [y.copy() for y in x] for x in c]  # noqa: E731
    _check(*copy(), lens, keep, 1000, 500, 2, 3, ws=ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    _check(*copy(), lens, keep, 1000, 500, 2, 3, ws=ws, stream=s)
    tables, pools, exps, w = copy()
    fresh = [_t(x) for x in (*pools, *exps, w)]
    d = [x.clone() for x in fresh]
    kept = torch.zeros(2, 2, 500, dtype=torch.int32, device=DEV)
    args = (_t(tables), _t(np.array(lens, np.int32)), _t(np.array(keep, np.int32)), kept, ws)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        kvcache.evict_f8_paged(*d, *args, max_ctx=1000, sink=2, recent=3)
    want = L.evict(pools, exps, w, tables, lens, keep, 1000, 500, 2, 3)
    for _ in range(4):
        for a, b in zip(d, fresh):
            a.copy_(b)
        kept.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((*d, kept), (*pools, *exps, w, want)):
            assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("max_ctx", [16384, 16385])
def test_lengths_around_what_one_workgroup_holds(max_ctx):
    """The longest slots of the one kind of selection and the shortest of the other, and whole stretches of rows."""
    rng = np.random.default_rng(max_ctx)
    lens = [16384, min(16385, max_ctx), 8192, 4096, 4095, 1]
    for sink, recent in ((0, 0), (1, 1)):
        _check(*_cache(rng, lens, 128, 1, 128), lens, [16383, 8000, 4096, 1, 4094, 1], max_ctx, 16384, sink, recent)


def test_many_slots_of_many_heads():
    """More chunks than workgroups are at work at a time, whole and partial, of heads that keep other rows."""
    rng = np.random.default_rng(17)
    lens = [int(x) for x in rng.integers(0, 900, 64)]
    keep = [int(x) for x in rng.integers(0, 900, 64)]
    _check(*_cache(rng, lens, 32, 16, 256), lens, keep, 900, 900, 4, 30)


@pytest.mark.parametrize("hd,bt", [(128, 4096), (256, 8192), (128, 2064)])
def test_pages_of_thousands_of_rows(hd, bt):
    """Many chunks of rows a page, each of which needs the exponents of all of the page's rows; slots of one page too."""
    rng = np.random.default_rng(bt)
    lens = [20000, 9000, 300, bt]
    _check(*_cache(rng, lens, bt, 1, hd), lens, [12000, 8999, 299, bt - 1], 20000, 12000, 4, 50)
    _check(*_cache(rng, lens, bt, 1, hd, ties=True), lens, [bt, 100, 300, 1], 20000, 12000)
