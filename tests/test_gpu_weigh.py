"""Accumulated attention weights of the paged 8-bit cache against the 64-bit definition: batches of single tokens,
blocks and prompts, windows, absent pages, recycled memory, many splits, graphs and streams."""
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


def _batch(rng, lens, new, bt, kv, hd, nq, scale=1.0):
    tables, starts, positions, n_pages = R.layout(rng, lens, new, bt, kv, hd)
    kp, ke = R.random_pool(rng, n_pages, bt, kv, hd, scale)
    q = rng.standard_normal((int(starts[-1]) + 2, nq, hd)).astype(np.float16)
    return dict(q=q, kp=kp, ke=ke, w=rng.random((n_pages, kv, bt)).astype(np.float32), tables=tables, starts=starts,
                positions=positions)


def _run(b, max_tok, max_ctx, scale, weighed=None, ws=None, stream=None, **kw):
    w = _t(b["w"])
    nq, hd = b["q"].shape[1:]
    kv, slots = b["kp"].shape[2], len(b["positions"])
    if ws is None:
        ws = kvcache.weigh_f8_paged_workspace(nq, kv, slots, b["q"].shape[0], max_tok, max_ctx, DEV, head_dim=hd)
        ws.fill_(255)
    kvcache.weigh_f8_paged(_t(b["q"]), _t(b["kp"]), _t(b["ke"]), w, ws, _t(b["tables"]), _t(b["starts"]), _t(b["positions"]),
                           max_tok=max_tok, max_ctx=max_ctx, scale=scale,
                           weighed=None if weighed is None else _t(np.array(weighed, np.int32)), stream=stream, **kw)
    torch.cuda.synchronize()
    return w.cpu().numpy().astype(np.float64)


def _check(b, max_tok=None, max_ctx=None, scale=None, weighed=None, ws=None, stream=None, **kw):
    new = np.diff(b["starts"])
    max_tok = int(max(new.max(), 1)) if max_tok is None else max_tok
    max_ctx = int(max((b["positions"] + new).max(), 1)) if max_ctx is None else max_ctx
    scale = b["q"].shape[2] ** -0.5 if scale is None else scale
    got = _run(b, max_tok, max_ctx, scale, weighed, ws, stream, **kw)
    ref, tol = L.weigh(b["q"], b["kp"], b["ke"], b["w"], b["tables"], b["starts"], b["positions"], scale, weighed,
                       max_ctx=max_ctx, **kw)
    assert (np.abs(got - ref) <= tol).all(), np.nanmax(np.abs(got - ref) - tol)
    return got


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("nq,kv", [(16, 4), (8, 8), (8, 1), (15, 3)])
@pytest.mark.parametrize("bt", [16, 64, 48])
def test_single_tokens_and_blocks(hd, nq, kv, bt):
    rng = np.random.default_rng(hd + nq + bt)
    _check(_batch(rng, [0, 1, 15, 300, 777, 31], [1, 1, 1, 1, 1, 1], bt, kv, hd, nq))
    _check(_batch(rng, [5, 0, 40, 1000], [3, 8, 0, 1], bt, kv, hd, nq), decay=0.5)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("nq,kv", [(16, 4), (6, 6), (8, 1), (10, 2)])
def test_prompts(hd, nq, kv):
    rng = np.random.default_rng(hd + nq)
    _check(_batch(rng, [0], [700], 16, kv, hd, nq))
    _check(_batch(rng, [130, 0, 50, 999], [257, 33, 1, 64], 32, kv, hd, nq), decay=0.25)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("new", [[1, 1, 1], [9, 16, 3], [300, 65, 1]])
@pytest.mark.parametrize("window,sink", [(1, 0), (40, 0), (40, 7), (200, 64), (33, 500), (64, 33), (10000, 3)])
def test_windows(hd, new, window, sink):
    rng = np.random.default_rng(window + sink)
    _check(_batch(rng, [500, 90, 1300], new, 16, 2, hd, 8), window=window, sink=sink, decay=0.75)


@pytest.mark.parametrize("new", [[1, 2], [100, 90]])
def test_absent_pages_and_short_tables(new):
    rng = np.random.default_rng(len(new))
    b = _batch(rng, [200, 333], new, 16, 2, 128, 8)
    b["tables"][0, [0, 3, 4]] = -1
    b["tables"][1, 5] = 10 ** 6
    b["tables"] = b["tables"][:, :14]
    b["ke"][0] = 255      # (what an absent page's lookup reads)
    b["kp"][0] = 0x7f
    b["tables"][b["tables"] == 0] = -5
    _check(b)


def test_rows_that_see_nothing_and_slots_without_rows():
    rng = np.random.default_rng(4)
    for new in ([2, 0, 1], [90, 0, 70]):
        b = _batch(rng, [20, 100, 30], new, 16, 2, 128, 4)
        b["tables"][0, :] = -1                       # no key at all
        _check(b)
        b["positions"][2] = -1                       # left alone
        _check(b, max_ctx=200)
        b = _batch(rng, [20, 100, 30], new, 16, 2, 128, 4)
        before = b["w"].copy()
        got = _check(b, window=5, decay=1.0)
        page = b["tables"][1, :6]
        assert np.array_equal(got[page].astype(np.float32), before[page])


@pytest.mark.parametrize("new", [[1, 3], [80, 70]])
def test_weighed_and_recycled_memory(new):
    """Weights past `weighed` hold anything before; with decay 0 all do."""
    rng = np.random.default_rng(5)
    b = _batch(rng, [100, 60], new, 16, 1, 128, 4)
    b["w"][:] = np.nan
    for s, n in enumerate((50, 0)):
        for j in range(n):
            b["w"][b["tables"][s, j // 16], 0, j % 16] = 2.0
    got = _run(b, max(new), 200, 0.1, weighed=[50, 0])
    ref, tol = L.weigh(b["q"], b["kp"], b["ke"], b["w"], b["tables"], b["starts"], b["positions"], 0.1, [50, 0])
    live = tol > 0
    assert live.sum() == sum(new) + 160 and (np.abs(got - ref)[live] <= tol[live]).all() and np.isnan(got[~live]).all()
    got = _run(b, max(new), 200, 0.1, decay=0.0)
    ref, tol = L.weigh(b["q"], b["kp"], b["ke"], b["w"], b["tables"], b["starts"], b["positions"], 0.1, decay=0.0)
    assert (np.abs(got - ref)[live] <= tol[live]).all()


@pytest.mark.parametrize("new", [[1], [40], [130]])
def test_context_limits_and_max_tok(new):
    rng = np.random.default_rng(6)
    b = _batch(rng, [300], new, 16, 2, 256, 8)
    for max_ctx in (1, 31, 300, 301, 4000):
        _check(b, max_ctx=max_ctx)
    if new[0] > 1:
        got = _run(b, new[0] - 1, 500, 0.0625)
        ref, tol = L.weigh(b["q"], b["kp"], b["ke"], b["w"], b["tables"], b["starts"], b["positions"], 0.0625,
                           max_tok=new[0] - 1)
        assert (np.abs(got - ref) <= tol).all()


@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
def test_scales(scale):
    rng = np.random.default_rng(7)
    for new in ([2], [150]):
        _check(_batch(rng, [250], new, 16, 2, 128, 8), scale=scale)


def test_weights_sum_to_the_rows():
    """A long context in many chunks, one token and many: each row's weights are one in all."""
    rng = np.random.default_rng(8)
    for new in ([1, 1], [200, 3]):
        b = _batch(rng, [40000, 9000], new, 64, 1, 128, 4)
        b["w"][:] = 0
        got = _run(b, max(new), 40200, 128 ** -0.5, decay=0.0)
        for s in range(2):
            assert abs(got[b["tables"][s][b["tables"][s] >= 0]].sum() - new[s] * 4) <= new[s] * 4 * 2e-5


@pytest.mark.parametrize("hd", [128, 256])
def test_long_contexts(hd):
    rng = np.random.default_rng(9)
    _check(_batch(rng, [9000, 2000], [1, 1], 64, 1, hd, 8))
    _check(_batch(rng, [5000, 300], [70, 2], 64, 1, hd, 4))


def test_a_query_that_is_not_finite():
    rng = np.random.default_rng(10)
    for new in ([2, 1], [90, 100]):
        b = _batch(rng, [50, 40], new, 16, 2, 128, 4)
        clean = _run(b, max(new), 200, 0.1)
        b["q"][0, 0, 5] = np.nan                     # slot 0, head 0 of KV head 0
        got = _run(b, max(new), 200, 0.1)
        mine = b["tables"][0][b["tables"][0] >= 0]
        assert np.isnan(got[mine[0], 0, 0]) and np.array_equal(got[:, 1], clean[:, 1])
        other = b["tables"][1][b["tables"][1] >= 0]
        assert np.array_equal(got[other], clean[other])


def test_the_same_bits_every_time():
    rng = np.random.default_rng(11)
    for new in ([1, 1], [120, 70], [300, 1]):
        b = _batch(rng, [3000, 800], new, 16, 2, 128, 8)
        a = [_run(b, max(new), 4000, 0.09) for _ in range(3)]
        assert np.array_equal(a[0], a[1]) and np.array_equal(a[0], a[2])


def test_many_slots():
    """More (slot, KV head) pairs than one launch dimension's old limit of 65,535, and slots without rows between."""
    rng = np.random.default_rng(12)
    n = 9000
    new = [(1 if i % 3 else 0) for i in range(n)]
    b = _batch(rng, [int(x) for x in rng.integers(1, 30, n)], new, 16, 8, 128, 8)
    _check(b)


def test_a_workspace_of_larger_numbers_a_stream_and_a_graph():
    rng = np.random.default_rng(13)
    ws = kvcache.weigh_f8_paged_workspace(8, 2, 8, 400, 256, 3000, DEV, head_dim=128)
    ws.fill_(255)
    st = torch.cuda.Stream()
    for new in ([1, 1, 1], [4, 0, 9], [200, 1, 65], [256]):
        b = _batch(rng, [500, 90, 1300][:len(new)], new, 16, 2, 128, 8)
        _check(b, ws=ws)
        st.wait_stream(torch.cuda.current_stream())
        _check(b, ws=ws, stream=st)
    for new in ([1, 2], [150, 3]):
        b = _batch(rng, [700, 90], new, 16, 2, 128, 8)
        args = [_t(b[k]) for k in ("q", "kp", "ke", "w")] + [ws] + [_t(b[k]) for k in ("tables", "starts", "positions")]
        fresh = args[3].clone()
        kw = dict(max_tok=160, max_ctx=1000, scale=0.1, decay=0.5)
        kvcache.weigh_f8_paged(*args, **kw)
        torch.cuda.synchronize()
        want = args[3].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kvcache.weigh_f8_paged(*args, **kw)
        for _ in range(3):
            args[3].copy_(fresh)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(args[3], want)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("nq,kv", [(12, 4), (14, 2), (7, 1)])
def test_groups_that_do_not_divide_a_tile(hd, nq, kv):
    rng = np.random.default_rng(hd + nq)
    _check(_batch(rng, [60, 700, 0], [301, 45, 90], 16, kv, hd, nq), decay=0.5)
    _check(_batch(rng, [60, 700, 0], [301, 45, 90], 16, kv, hd, nq), window=100, sink=9)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("new", [[1], [12], [300]])
@pytest.mark.parametrize("step", [0.5, 7.0, 28.0, -28.0])
def test_scores_that_rise_and_fall(hd, new, step):
    """Scores that change by `step` every 64 keys: what has been summed so far becomes next to nothing, many times, or what
    follows does."""
    rng = np.random.default_rng(13)
    b = _batch(rng, [900], new, 16, 1, hd, 4)
    j = np.arange(900 + new[0])
    level = j // 64 + 1 if step > 0 else 15 - j // 64
    page = b["tables"][0][j // 16]
    b["kp"][page, j % 16] = R.e4m3_encode(level.astype(np.float64))[:, None, None]   # (exact up to 16)
    b["ke"][:] = 127
    b["q"][:] = 1 + rng.integers(-3, 4, b["q"].shape) / 64
    _check(b, scale=abs(step) / hd)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("few", [True, False])
def test_many_rows_of_many_slots(hd, few):
    """More slots than a workgroup walks at a time, with runs of more than 64 that have no rows, beside single tokens (taken
    by the kernels for few rows) or where the call's rows say that all slots are alike."""
    rng = np.random.default_rng(hd + few)
    n, tok = 620, 40 if few else 20
    new = [0] * n
    for s in (0, 1, 75, 76, 160, 255, 256, 257, 400, 511, 512, 619):
        new[s] = int(rng.integers(17, tok + 1))
    if few:
        new[3] = new[80] = new[300] = new[618] = 1
    lens = [int(x) for x in rng.integers(0, 300, n)]
    b = _batch(rng, lens, new, 16, 2, hd, 8)
    if not few:   # rows behind the last slot's
        b["q"] = np.concatenate([b["q"], rng.standard_normal((n * tok // 2, 8, hd)).astype(np.float16)])
    _check(b, max_tok=tok, decay=0.5)
    _check(b, max_tok=tok, window=70, sink=20)


@pytest.mark.parametrize("hd", [128, 256])
def test_more_tiles_than_a_workgroup_walks_at_a_time(hd):
    """More than 256 tiles of 256 keys of one slot, of several, and more than 256 tiles of rows."""
    rng = np.random.default_rng(hd)
    _check(_batch(rng, [65700], [70], 64, 1, hd, 4), decay=0.5)
    _check(_batch(rng, [40000, 0, 30000, 5], [40, 0, 70, 90], 64, 1, hd, 4), decay=0.0)
    _check(_batch(rng, [66000, 100], [33, 40], 64, 1, hd, 4), window=3000, sink=70)
    b = _batch(rng, [10, 7], [8300, 9], 64, 1, hd, 8)
    _check(b, max_ctx=300)
    _check(b, max_ctx=300, window=150, sink=33)


def test_a_query_of_minus_infinity():
    """Products that are all -infinity are those of keys that are not seen: the row adds nothing."""
    rng = np.random.default_rng(15)
    for new in (1, 90):
        b = _batch(rng, [50], [new], 16, 1, 128, 1)
        b["kp"][:] = np.abs(rng.integers(1, 120, b["kp"].shape)).astype(np.uint8)   # (positive codes)
        b["ke"][:] = 127
        b["q"][:, :, 7] = -np.inf
        got = _run(b, new, 200, 0.1)
        page, at = b["tables"][0][np.arange(50 + new) // 16], np.arange(50 + new) % 16
        want = np.where(np.arange(50 + new) < 50, b["w"][page, 0, at], 0)
        assert np.array_equal(got[page, 0, at].astype(np.float32), want)
