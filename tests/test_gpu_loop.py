"""Decoding loops of the operators together, as they are used, each step against the 64-bit references on what the
device holds: a bounded cache (prompt, weighing, eviction, more tokens, a captured step) and a beam search."""
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


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _np(x):
    return x.cpu().numpy()


class Cache:
    """A paged 8-bit cache with weights, on the device and as the references keep it."""

    def __init__(self, slots, blocks, pages, bt, kv, hd):
        self.bt, self.kv, self.hd = bt, kv, hd
        shape = (pages, bt, kv, hd)
        self.pools = [torch.zeros(shape, dtype=torch.uint8, device=DEV) for _ in range(2)]
        self.exps = [torch.zeros(pages, kv, dtype=torch.uint8, device=DEV) for _ in range(2)]
        self.w = kvcache.f8_weights(pages, bt, kv, DEV)
        self.t, self.r = torch.full((slots, blocks), -1, dtype=torch.int32, device=DEV), torch.zeros(pages, dtype=torch.int32, device=DEV)
        self.planes = kvcache.page_planes([*self.pools, *self.exps, self.w])
        self.ref = [_np(x).copy() for x in (*self.pools, *self.exps, self.w)]
        self.tables, self.refs = _np(self.t).copy(), _np(self.r).copy()

    def reserve(self, slots, positions, n_new):
        want, pairs = R.reserve(self.tables, self.refs, slots, positions, n_new, max(n_new), self.bt)
        st = i32([9] * len(slots))
        kvcache.pages_reserve(self.t, self.r, i32(slots), i32(positions), i32(n_new), st, self.planes, block_tokens=self.bt,
                              max_new=max(n_new))
        assert st.tolist() == want == [0] * len(slots)
        for a, b in pairs:
            if a >= 0:
                for x in self.ref:
                    x[b] = x[a]
        assert np.array_equal(_np(self.t), self.tables) and np.array_equal(_np(self.r), self.refs)

    def release(self, slots, keep):
        R.release(self.tables, self.refs, slots, keep, self.bt)
        kvcache.pages_release(self.t, self.r, i32(slots), i32(keep), block_tokens=self.bt)
        assert np.array_equal(_np(self.t), self.tables) and np.array_equal(_np(self.r), self.refs)

    def append(self, k, v, starts, positions):
        for x, pool, exp in ((k, 0, 2), (v, 1, 3)):
            R.append(self.ref[pool], self.ref[exp], _np(x), self.tables, starts, positions)
        kvcache.f8_append_kv_paged(k, v, *self.pools, *self.exps, self.t, i32(starts), i32(positions),
                                   max_tok=int(np.diff(starts).max()))
        self.check()

    def check(self):
        for x, y in zip((*self.pools, *self.exps), self.ref):
            assert np.array_equal(_np(x), y)


def _close(got, want, tol):
    assert (np.abs(got - want) <= tol).all(), np.nanmax(np.abs(got - want) - tol)


@pytest.mark.parametrize("hd,nq,kv,bt", [(128, 8, 2, 16), (256, 8, 8, 48)])
def test_a_bounded_cache(hd, nq, kv, bt):
    """Prompts whose last queries weigh the keys, an eviction to a budget, pages given back, then tokens at their true
    positions in the rows behind, each weighed, with another eviction on the way."""
    rng = np.random.default_rng(hd)
    lens, budget, scale, rot, tail = [150, 1, 77, 230], 64, hd ** -0.5, hd // 2, 8
    slots = len(lens)
    c = Cache(slots, 260 // bt + 1, 80, bt, kv, hd)
    table = kvcache.rope_table(rot, base=1e5, device=DEV)
    weights = [rng.standard_normal(hd).astype(np.float32) for _ in range(2)]
    dev_weights = [_t(x) for x in weights]
    aws = kvcache.attn_f8_paged_workspace(nq, kv, slots, 500, 230, 400, DEV, head_dim=hd)
    wws = kvcache.weigh_f8_paged_workspace(nq, kv, slots, 500, 230, 400, DEV, head_dim=hd)
    ews = kvcache.evict_f8_paged_workspace(slots, kv, bt, 400, budget, DEV)

    def step(new, rows, positions, weighing):
        """new[s] tokens at `positions` go to rows rows[s] on; the last of them weigh the keys (weighing[s] rows)."""
        starts = np.cumsum([0] + new).astype(np.int32)
        n = int(starts[-1])
        qkv = (rng.standard_normal((n, nq + 2 * kv, hd)) * 3).astype(np.float16)
        buf = _t(qkv)
        q, k, v = buf[:, :nq], buf[:, nq:nq + kv], buf[:, nq + kv:]
        kvcache.norm_rope(q, k, *dev_weights, i32(positions), table)
        for x, y, w in ((q, qkv[:, :nq], weights[0]), (k, qkv[:, nq:nq + kv], weights[1])):
            _close(_np(x), *L.norm_rope(y, w, np.array(positions), rot, "half", base=1e5))
        assert np.array_equal(_np(v), qkv[:, nq + kv:])
        c.reserve(list(range(slots)), rows, new)
        c.append(k, v, starts, np.array(rows, np.int32))
        q = q.contiguous()
        out = torch.empty_like(q)
        kvcache.attn_f8_paged(q, *c.pools, *c.exps, out, aws, c.t, i32(starts.tolist()), i32(rows), max_tok=max(new), max_ctx=400,
                              scale=scale)
        _close(_np(out), *R.attention(_np(q), *c.ref[:4], c.tables, starts, np.array(rows), scale))
        # the last rows weigh; the weights of the keys before this step's stand
        last = np.cumsum([0] + weighing).astype(np.int32)
        pick = np.concatenate([np.arange(b - m, b) for b, m in zip(starts[1:], weighing)])
        at = [r + a - m for r, a, m in zip(rows, new, weighing)]
        ql = q[_t(pick)].contiguous()
        before = _np(c.w).copy()
        kvcache.weigh_f8_paged(ql, c.pools[0], c.exps[0], c.w, wws, c.t, i32(last.tolist()), i32(at), max_tok=max(weighing),
                               max_ctx=400, scale=scale, decay=0.75, weighed=i32(rows))
        _close(_np(c.w), *L.weigh(_np(ql), c.ref[0], c.ref[2], before, c.tables, last, np.array(at), scale, rows, 0.75))
        c.ref[4][:] = _np(c.w)

    def evict(rows):
        kept = torch.full((slots, kv, budget), 7, dtype=torch.int32, device=DEV)
        want = L.evict(c.ref[:2], c.ref[2:4], c.ref[4], c.tables, rows, [budget] * slots, 400, budget, 4, 16)
        kvcache.evict_f8_paged(*c.pools, *c.exps, c.w, c.t, i32(rows), i32([budget] * slots), kept, ews, max_ctx=400, sink=4,
                               recent=16)
        assert np.array_equal(_np(kept), want)
        rows = [min(n, budget) for n in rows]
        for s in range(slots):   # (rows past the new length hold anything)
            j = np.arange(rows[s])
            page, at = c.tables[s][j // bt], j % bt
            for x, y in zip(c.pools, c.ref):
                assert np.array_equal(_np(x)[page, at], y[page, at])
            for x, y in zip(c.exps, c.ref[2:4]):
                assert np.array_equal(_np(x)[page], y[page])
            assert np.array_equal(_np(c.w)[page, :, at], c.ref[4][page, :, at])
        for x, y in zip((*c.pools, *c.exps, c.w), c.ref):
            y[:] = _np(x)
        c.release(list(range(slots)), rows)
        return rows

    step(lens, [0] * slots, np.concatenate([np.arange(n) for n in lens]).tolist(), [min(n, tail) for n in lens])
    rows, true = evict(lens), list(lens)
    for i in range(6):
        new = [1, 1, 1, 1] if i != 3 else [3, 1, 5, 2]
        step(new, rows, np.concatenate([np.arange(p, p + n) for p, n in zip(true, new)]).tolist(), new)
        rows, true = [a + b for a, b in zip(rows, new)], [a + b for a, b in zip(true, new)]
        if i == 4:
            rows = evict(rows)


def test_a_captured_step():
    """Norms, append, attention and weighing of single tokens in one graph, replayed with the lengths moved on from
    outside and eager work between: every replay against the same calls run eagerly on a copy."""
    slots, nq, kv, hd, bt, rot, scale = 5, 16, 4, 128, 16, 64, 0.1
    rng = np.random.default_rng(3)
    tables = _t(rng.permutation(slots * 20).astype(np.int32).reshape(slots, 20))
    table = kvcache.rope_table(rot, device=DEV)
    w = _t(rng.standard_normal(hd).astype(np.float32))
    ones = torch.arange(slots + 1, dtype=torch.int32, device=DEV)
    aws = kvcache.attn_f8_paged_workspace(nq, kv, slots, slots, 1, 320, DEV, head_dim=hd)
    wws = kvcache.weigh_f8_paged_workspace(nq, kv, slots, slots, 1, 320, DEV, head_dim=hd)

    def fresh():
        return [torch.zeros(slots * 20, bt, kv, hd, dtype=torch.uint8, device=DEV) for _ in range(2)] + \
               [torch.zeros(slots * 20, kv, dtype=torch.uint8, device=DEV) for _ in range(2)] + [kvcache.f8_weights(slots * 20, bt, kv, DEV)]

    def run(state, buf, pos, out):
        kp, vp, ke, ve, wt = state
        q, k, v = buf[:, :nq], buf[:, nq:nq + kv], buf[:, nq + kv:]
        qo = out[0]
        kvcache.norm_rope(q, k, w, None, pos, table, q_out=qo)
        kvcache.f8_append_kv_paged(k, v, kp, vp, ke, ve, tables, ones, pos, max_tok=1)
        kvcache.attn_f8_paged(qo, kp, vp, ke, ve, out[1], aws, tables, ones, pos, max_tok=1, max_ctx=320, scale=scale)
        kvcache.weigh_f8_paged(qo, kp, ke, wt, wws, tables, ones, pos, max_tok=1, max_ctx=320, scale=scale, decay=0.9)

    a, b = fresh(), fresh()
    buf = torch.zeros(slots, nq + 2 * kv, hd, dtype=torch.float16, device=DEV)
    pos = torch.zeros(slots, dtype=torch.int32, device=DEV)
    outs = [[torch.empty(slots, nq, hd, dtype=torch.float16, device=DEV) for _ in range(2)] for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(a, buf, pos, outs[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(a, buf, pos, outs[0])
    for x, y in zip(a, fresh()):
        x.copy_(y)
    for i in range(40):
        new = _t(rng.standard_normal(buf.shape).astype(np.float16))
        pos.copy_(_t((np.arange(slots) * 3 + i).astype(np.int32)))
        buf.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        run(b, new, pos, outs[1])
        torch.cuda.synchronize()
        for x, y in zip((*a, *outs[0]), (*b, *outs[1])):
            assert torch.equal(x, y), i


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_a_beam_search(dtype):
    """Requests of several beams over shared prompts: selection, reordering of pages and token histories, pages of
    their own for the next tokens, the append; beams end on the way and one request runs out of candidates."""
    n, beams, vocab, bt, kv, hd, end, steps = 3, 4, 50, 16, 2, 128, 7, 8
    rng = np.random.default_rng(5)
    c = Cache(n * beams, 6, 120, bt, kv, hd)
    slots = list(range(n * beams))
    prompts = [20, 33, 5]
    # the prompt of a request once, its pages shared by the other beams
    first = [r * beams for r in range(n)]
    c.reserve(first, [0] * n, prompts)
    starts = np.zeros(n * beams + 1, np.int32)
    for r in range(n):
        starts[r * beams + 1:] += prompts[r]
    kv_rows = rng.standard_normal((2, int(starts[-1]), kv, hd)).astype(np.float16)
    c.append(_t(kv_rows[0]), _t(kv_rows[1]), starts, np.zeros(n * beams, np.int32))
    par = [s for s in first for _ in range(beams - 1)]
    chi = [s + b for s in first for b in range(1, beams)]
    lens = [prompts[s // beams] for s in slots]
    assert R.fork(c.tables, c.refs, par, chi, [lens[s] for s in par], bt) == [0] * len(par)
    kvcache.pages_fork(c.t, c.r, i32(par), i32(chi), i32([lens[s] for s in par]), block_tokens=bt)

    history = torch.full((n * beams, steps), -1, dtype=torch.int32, device=DEV)
    ref_history = _np(history).copy()
    states = kvcache.page_planes([history])
    scores = torch.full((n, beams), -torch.inf, device=DEV)
    scores[:, 0] = 0
    done = torch.zeros(n, beams, dtype=torch.int32, device=DEV)
    parents, tokens = (torch.empty(n, beams, dtype=torch.int32, device=DEV) for _ in range(2))
    top = torch.empty(n, beams, device=DEV)
    ws = kvcache.beam_select_workspace(n, beams, vocab, beams, DEV)
    for i in range(steps):
        logits = rng.standard_normal((n * beams, vocab)) * 2
        logits[:, end] += 2.5                       # (beams end)
        if i == 0:
            logits[2 * beams, 2:] = -np.inf         # (two candidates of the last request's one beam)
        logits = torch.from_numpy(logits).to(dtype)
        sc, dn = _np(scores).copy(), _np(done).copy()
        kvcache.beam_select(logits.to(DEV), scores, parents, tokens, top, ws, done=done, end_token=end)
        p, t, s = _np(parents), _np(tokens), _np(top)
        L.beam_check(logits.float().numpy(), sc, beams, p, t, s, dn, end)
        st = i32([9] * (n * beams))
        kvcache.pages_reorder(c.t, c.r, i32(slots), parents.view(-1), i32(lens), st, states, block_tokens=bt)
        want = L.reorder(c.tables, c.refs, slots, p.reshape(-1).tolist(), lens, bt, (ref_history,))
        assert st.tolist() == want and (np.array(want) == R.INVALID).sum() == (p == -1).sum()
        assert np.array_equal(_np(c.t), c.tables) and np.array_equal(_np(c.r), c.refs)
        # (the same calls a loop makes on the device: done of the parent, or the token)
        was = torch.where(parents >= 0, done.view(-1)[parents.clamp(min=0).long()], 0)
        done = (was.bool() | (tokens == end)).int()
        scores = top.clone()
        history[:, i] = tokens.view(-1)
        ref_history[:, i] = t.reshape(-1)
        assert np.array_equal(_np(history), ref_history)
        # the tokens' rows, in pages of their own
        c.reserve(slots, lens, [1] * (n * beams))
        rows = rng.standard_normal((2, n * beams, kv, hd)).astype(np.float16)
        c.append(_t(rows[0]), _t(rows[1]), np.arange(n * beams + 1, dtype=np.int32), np.array(lens, np.int32))
        lens = [x + 1 for x in lens]
        used = c.tables[c.tables >= 0]
        assert np.array_equal(np.bincount(used, minlength=len(c.refs)), c.refs)
    assert done.any()


@pytest.mark.parametrize("new", [[1, 1, 1], [90, 5, 1]])
def test_pages_past_four_billion_bytes(new):
    """The same pages at the front of a small pool and past 2^32 bytes of a large one: the same bits, and nothing else is
    touched of the large one's first pages."""
    rng = np.random.default_rng(23)
    bt, kv, hd, nq, far, lens = 64, 4, 256, 16, 70000, [700, 64, 1500]
    tables, starts, positions, n = R.layout(rng, lens, new, bt, kv, hd)
    pools = [R.random_pool(rng, n, bt, kv, hd) for _ in range(2)]
    w = rng.random((n, kv, bt)).astype(np.float32)
    q = _t(rng.standard_normal((int(starts[-1]), nq, hd)).astype(np.float16))
    keep, rows = [300, 10, 900], [a + b for a, b in zip(lens, new)]
    out = []
    for at in (0, far):
        big = []
        for x in (pools[0][0], pools[1][0], pools[0][1], pools[1][1], w):
            y = torch.zeros((at + n, *x.shape[1:]), dtype=torch.float32 if x.dtype == np.float32 else torch.uint8, device=DEV)
            y[at:].copy_(_t(x))
            big.append(y)
        kp, vp, ke, ve, wt = big
        t = _t(np.where(tables >= 0, tables + at, -1).astype(np.int32))
        ws = kvcache.weigh_f8_paged_workspace(nq, kv, 3, q.shape[0], max(new), 1700, DEV, head_dim=hd)
        kvcache.weigh_f8_paged(q, kp, ke, wt, ws, t, _t(starts), _t(positions), max_tok=max(new), max_ctx=1700, scale=hd ** -0.5)
        weighed = wt[at:].clone()
        kept = torch.zeros(3, kv, 900, dtype=torch.int32, device=DEV)
        ews = kvcache.evict_f8_paged_workspace(3, kv, bt, 1700, 900, DEV)
        kvcache.evict_f8_paged(kp, vp, ke, ve, wt, t, i32(rows), i32(keep), kept, ews, max_ctx=1700, sink=2, recent=9)
        if at:
            assert not any(x[:n].any() for x in big)
        out.append([weighed, kept] + [x[at:] for x in big])
    for a, b in zip(*out):
        assert torch.equal(a, b)
    assert (out[0][1] >= 0).any()


def test_two_streams_at_once():
    """Weighing and eviction of two caches on two streams, with a workspace each: as one after the other."""
    rng = np.random.default_rng(29)
    bt, kv, hd, nq, lens = 16, 8, 128, 16, [3000, 17, 1200, 2500]
    tables, starts, positions, n = R.layout(rng, lens, [1] * 4, bt, kv, hd)
    rows, keep = [a + 1 for a in lens], [1000, 17, 1100, 2000]
    pools = [R.random_pool(rng, n, bt, kv, hd) for _ in range(2)]
    w = rng.random((n, kv, bt)).astype(np.float32)
    q = [_t(rng.standard_normal((4, nq, hd)).astype(np.float16)) for _ in range(2)]
    t, st, pos, r, k = _t(tables), _t(starts), _t(positions), i32(rows), i32(keep)

    def state():
        return [_t(x) for x in (pools[0][0], pools[1][0], pools[0][1], pools[1][1], w)] + \
               [torch.zeros(4, kv, 2000, dtype=torch.int32, device=DEV), kvcache.weigh_f8_paged_workspace(nq, kv, 4, 4, 1, 3100, DEV, head_dim=hd),
                kvcache.evict_f8_paged_workspace(4, kv, bt, 3100, 2000, DEV)]

    def run(s, q, stream):
        kvcache.weigh_f8_paged(q, s[0], s[2], s[4], s[6], t, st, pos, max_tok=1, max_ctx=3100, scale=0.1, stream=stream)
        kvcache.evict_f8_paged(*s[:5], t, r, k, s[5], s[7], max_ctx=3100, sink=4, recent=30, stream=stream)

    want = [state(), state()]
    for s, x in zip(want, q):
        run(s, x, None)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = [state(), state()]
        torch.cuda.synchronize()
        for s, x, stream in zip(got, q, streams):
            run(s, x, stream)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a[:6], b[:6]))
