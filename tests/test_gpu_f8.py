"""The paged 8-bit cache: append bit for bit, attention against 64 bits, and the calls
together."""
import numpy as np
import pytest
import torch

from qengine_amd import kvcache
from tests import _paged8 as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def _append_case(rng, lens, new, bt, kv, hd, x=None, **kw):
    tables, starts, pos, n_pages = R.layout(rng, lens, new, bt, kv, hd, **kw)
    (kp, ke), (vp, ve) = R.random_pool(rng, n_pages, bt, kv, hd), R.random_pool(rng, n_pages, bt, kv, hd)
    rows = int(starts[-1]) + 2
    k = rng.standard_normal((rows, kv, hd)).astype(np.float16) if x is None else x
    v = (rng.standard_normal((rows, kv, hd)) * 8.0 ** rng.integers(-2, 3, (rows, 1, 1))).astype(np.float16)
    return tables, starts, pos, kp, ke, vp, ve, k, v


def _check_append(case, max_tok=None, table_edit=None):
    tables, starts, pos, kp, ke, vp, ve, k, v = case
    if table_edit:
        table_edit(tables, pos)
    g = [dev(x) for x in (kp, vp, ke, ve)]
    new = int(max(np.diff(starts).max(), 1))
    kvcache.f8_append_kv_paged(dev(k), dev(v), *g, dev(tables), dev(starts), dev(pos), max_tok=max_tok or new)
    for x, pool, exp in ((k, kp, ke), (v, vp, ve)):
        R.append(pool, exp, x, tables, starts.tolist(), pos.tolist(), max_tok or new)
    for got, want, what in zip(g, (kp, vp, ke, ve), ("k", "v", "ke", "ve")):
        assert np.array_equal(got.cpu().numpy(), want), what


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("bt,lens,new", [
    (16, [0, 5, 15, 16, 100], [1, 1, 1, 1, 1]),              # a decode step: fresh pages, continued ones, a page's last row
    (64, [63, 0, 1], [2, 130, 64]),                           # over page ends
    (16, [7, 3, 0], [40, 0, 17]),                             # a slot without rows
    (48, [47, 100, 95], [49, 3, 1]),                          # pages that are no power of two
    (256, [200, 0], [300, 5]),                                # more rows than a thread keeps
])
def test_append_bit_exact(hd, bt, lens, new):
    rng = np.random.default_rng(bt * 7 + hd + len(new))
    _check_append(_append_case(rng, lens, new, bt, 3, hd))


def test_append_special_values():
    """NaN, infinities, the range's ends, subnormals, zeros, and pages whose older rows are requantized."""
    rng = np.random.default_rng(1)
    lens, new = [4, 0, 9, 3, 15], [1, 3, 2, 1, 1]
    n = sum(new) + 2
    x = rng.standard_normal((n, 2, 128)).astype(np.float16)
    x[0, 0, 3], x[0, 1, :] = np.nan, np.inf
    x[1, 0, :] = 0.0
    x[1, 1, :], x[2, 1, :], x[3, 1, :] = 0.0, 0.0, 0.0          # a page of zeros
    x[2, 0, 5], x[3, 0, 6] = 65504, -61440
    x[4, 0, :] = np.float16(6e-8) * rng.integers(0, 4, 128)      # subnormal fp16
    x[4, 1, 7] = -np.inf
    x[6, :, :] = 448.0                                           # exactly the largest code
    x[7, 0, :] = 448.25
    x[7, 1, :] = np.float16(-np.nan)
    _check_append(_append_case(rng, lens, new, 16, 2, 128, x=x))


def test_append_bad_pages_and_short_max_tok():
    """Rows without a page, past the table or past max_tok are dropped, everything else is as it was."""
    rng = np.random.default_rng(2)

    def edit(tables, pos):
        tables[0, 1], tables[1, 0], tables[2, 2] = -1, 10 ** 6, -5
        pos[3] = -1
        pos[4] = 16 * tables.shape[1] - 2   # runs past the table
    _check_append(_append_case(rng, [3, 4, 5, 6, 7], [30, 20, 60, 4, 9], 16, 2, 128), table_edit=edit)
    _check_append(_append_case(rng, [3, 4], [30, 20], 16, 2, 128), max_tok=7)


def test_slots_out_of_range():
    """A slot whose position is negative or past 2^30 is left alone: cache, rotated queries and outputs."""
    rng = np.random.default_rng(3)
    tables, starts, pos, kp, ke, vp, ve, k, v = _append_case(rng, [3, 4, 5], [2, 3, 4], 16, 2, 128)
    pos[0], pos[2] = -1, (1 << 30) + 1
    g = [dev(x) for x in (kp, vp, ke, ve)]
    q = torch.full((len(k), 8, 128), 1.0, dtype=torch.float16, device=DEV)
    got = torch.full_like(q, 5.0)
    kvcache.f8_append_kv_paged(dev(k), dev(v), *g, dev(tables), dev(starts), dev(pos), max_tok=4, q=q, q_out=got,
                               rope=kvcache.rope_table(128, device=DEV))
    assert (got[:2] == 5).all() and (got[5:] == 5).all() and (got[2:5] != 5).all()
    own = set(tables[1].tolist())
    for x, y in zip(g, (kp, vp, ke, ve)):
        x = x.cpu().numpy()
        assert all(np.array_equal(x[i], y[i]) for i in range(len(y)) if i not in own)
    out = torch.full_like(q, 5.0)
    ws = kvcache.attn_f8_paged_workspace(8, 2, 3, len(k), 4, 64, DEV, head_dim=128)
    kvcache.attn_f8_paged(q, g[0], g[1], g[2], g[3], out, ws, dev(tables), dev(starts), dev(pos), max_tok=4, max_ctx=64, scale=0.1)
    assert (out[:2] == 5).all() and (out[5:] == 5).all() and (out[2:5] != 5).any()


@pytest.mark.parametrize("layout,rot", [("half", 64), ("interleaved", 256), ("half", 256), ("interleaved", 16)])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [70, 0, 3, 20]])
def test_rope_in_the_append(layout, rot, new):
    """q, k and v as views of one buffer: the same bits as rope, then the append; q apart and in place."""
    rng = np.random.default_rng(rot)
    tables, starts, pos, kp, ke, vp, ve, _, _ = _append_case(rng, [0, 5, 77, 31], new, 16, 2, 256)
    rows = int(starts[-1]) + 2
    buf = dev(rng.standard_normal((rows, 6 + 2 + 2, 256)).astype(np.float16))
    q, k, v = buf[:, :6], buf[:, 6:8], buf[:, 8:]
    t = kvcache.rope_table(rot, device=DEV)
    at = np.zeros(rows, np.int32)
    for s in range(4):
        at[starts[s]:starts[s + 1]] = pos[s] + np.arange(new[s])
    ko, qo = torch.empty_like(k, memory_format=torch.contiguous_format), torch.empty_like(q, memory_format=torch.contiguous_format)
    kvcache.rope(q, k, dev(at), t, layout=layout, q_out=qo, k_out=ko)
    a, b = [dev(x) for x in (kp, vp, ke, ve)], [dev(x) for x in (kp, vp, ke, ve)]
    rest = (dev(tables), dev(starts), dev(pos))
    kvcache.f8_append_kv_paged(ko, v, *a, *rest, max_tok=max(new))
    got = torch.full_like(qo, 5.0)
    kvcache.f8_append_kv_paged(k, v, *b, *rest, max_tok=max(new), q=q, q_out=got, rope=t, layout=layout)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    n = int(starts[-1])
    assert torch.equal(got[:n], qo[:n]) and (got[n:] == 5).all()
    keep = buf[n:].clone()
    kvcache.f8_append_kv_paged(k, v, *b, *rest, max_tok=max(new), q=q, rope=t, layout=layout)
    assert torch.equal(buf[:n, :6], qo[:n]) and torch.equal(buf[n:], keep)


def test_append_of_a_long_prompt_beside_many_slots():
    """255 single tokens beside a prompt of 65,536 in 16-row pages: more than 2^32 threads. The same bits as the two apart."""
    slots, prompt, bt, kv, hd, nq = 256, 65536, 16, 8, 256, 8
    g = torch.Generator(device=DEV).manual_seed(5)
    n, blocks = prompt + slots - 1, prompt // bt
    q, k, v = (torch.randn(n, heads, hd, device=DEV, generator=g, dtype=torch.float16) for heads in (nq, kv, kv))
    tables = torch.full((slots, blocks), -1, dtype=torch.int32, device=DEV)
    tables[slots // 2] = torch.arange(blocks, device=DEV)
    own = torch.cat([torch.arange(slots // 2), torch.arange(slots // 2 + 1, slots)])
    tables[own, 0] = blocks + torch.arange(slots - 1, dtype=torch.int32, device=DEV)
    new = [1] * slots
    new[slots // 2] = prompt
    starts = torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device=DEV)
    pos = torch.zeros(slots, dtype=torch.int32, device=DEV)
    t = kvcache.rope_table(64, device=DEV)
    a = [*kvcache.f8_pool(blocks + slots - 1, bt, kv, hd, DEV), *kvcache.f8_pool(blocks + slots - 1, bt, kv, hd, DEV)]
    b = [x.clone() for x in a]
    got, want = torch.zeros_like(q), torch.zeros_like(q)

    def call(c, out, lo, hi, most):
        kvcache.f8_append_kv_paged(k, v, c[0], c[2], c[1], c[3], tables[lo:hi], starts[lo:hi + 1], pos[lo:hi], max_tok=most,
                                   q=q, q_out=out, rope=t)
    call(a, got, 0, slots, prompt)
    for lo, hi, most in ((0, slots // 2, 1), (slots // 2, slots // 2 + 1, prompt), (slots // 2 + 1, slots, 1)):
        call(b, want, lo, hi, most)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(got, want)
    assert (a[1] > 0).all() and (a[3] > 0).all()   # (every page was written)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _attend(q, kp, vp, ke, ve, tables, starts, pos, scale, window=0, sink=0, max_tok=None, max_ctx=None, alias=False):
    nq, kv, hd = q.shape[1], kp.shape[2], q.shape[2]
    mt = max_tok or int(max(np.diff(starts).max(), 1))
    mc = max_ctx or int(max((pos + np.diff(starts)).max(), 1))
    qd = dev(q)
    out = qd if alias else torch.full_like(qd, 9.0)
    ws = kvcache.attn_f8_paged_workspace(nq, kv, len(pos), q.shape[0], mt, mc, DEV, head_dim=hd)
    assert not ws.any()
    ws[4096:] = 0xff   # (past the counts nothing in it is trusted)
    kvcache.attn_f8_paged(qd, dev(kp), dev(vp), dev(ke), dev(ve), out, ws, dev(tables), dev(starts), dev(pos), max_tok=mt,
                          max_ctx=mc, scale=scale, window=window, sink=sink)
    assert not ws[:4096].any()   # ready for the next call
    return out.cpu().numpy()


def _attn_case(seed, lens, new, bt, kv, gqa, hd, scale=1.0, spare_rows=2):
    rng = np.random.default_rng(seed)
    tables, starts, pos, n_pages = R.layout(rng, lens, new, bt, kv, hd)
    (kp, ke), (vp, ve) = R.random_pool(rng, n_pages, bt, kv, hd, scale), R.random_pool(rng, n_pages, bt, kv, hd)
    # what a page holds past its slot's last key is anything, NaN codes among it
    for s, (a, b) in enumerate(zip(lens, new)):
        end = a + b
        if end % bt and tables[s, end // bt] >= 0:
            kp[tables[s, end // bt], end % bt:] = 0x7f
            vp[tables[s, end // bt], end % bt:] = 0xff
    q = rng.standard_normal((int(starts[-1]) + spare_rows, kv * gqa, hd)).astype(np.float16)
    return q, kp, vp, ke, ve, tables, starts, pos


def _check_attn(case, scale, window=0, sink=0, rows_left=True, **kw):
    q, kp, vp, ke, ve, tables, starts, pos = case
    got = _attend(*case, scale, window, sink, **kw).astype(np.float64)
    ref, tol = R.attention(q, kp, vp, ke, ve, tables, starts.tolist(), pos.tolist(), scale, window, sink,
                           kw.get("max_ctx") or 1 << 30)
    own = ~np.isnan(ref)
    err = np.where(own, np.abs(got - np.where(own, ref, 0)), 0)
    assert (err <= tol).all(), (err.max(), (err / np.maximum(tol, 1e-30)).max())
    if not kw.get("alias"):
        assert (got[~own] == 9.0).all()   # rows behind the last slot's
    return got


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("bt,lens,gqa,kv", [
    (64, [0], 4, 2), (16, [1, 14, 15, 16], 1, 1), (16, [700], 8, 2), (64, [31, 32, 33, 127, 128, 129], 6, 1),
    (256, [3000, 5, 0, 260], 4, 2), (64, [2047, 1500, 100], 4, 2), (16, [1023], 8, 1), (48, [1000, 47], 3, 3), (16, [0] * 20 + [2000], 5, 1)])
def test_decode(hd, bt, lens, gqa, kv):
    """One query a slot, from no earlier key to several parts of a workgroup's line."""
    _check_attn(_attn_case(hd + bt + len(lens), lens, [1] * len(lens), bt, kv, gqa, hd), hd ** -0.5)


@pytest.mark.parametrize("hd,gqa,new", [(256, 4, [8, 5, 0, 1]), (128, 8, [4, 3]), (256, 4, [16, 16]), (128, 6, [10, 2, 7]),
                                        (256, 1, [64, 33]), (256, 8, [2, 1])])
def test_verify(hd, gqa, new):
    """Blocks of up to 64 (token, head) rows, slots without rows among them."""
    lens = [300, 17, 40, 0][:len(new)]
    _check_attn(_attn_case(hd + gqa, lens, new, 16, 2, gqa, hd), hd ** -0.5)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("bt,lens,new,gqa", [
    (64, [0], [65], 1), (16, [0, 0, 0], [100, 1, 33], 4), (32, [500, 0], [20, 150], 6), (64, [130], [300], 2),
    (48, [77, 3, 0], [1, 90, 0], 8)])
def test_prompts(hd, bt, lens, new, gqa):
    """More than 64 rows a slot, with one-token slots and empty ones in the batch."""
    _check_attn(_attn_case(hd + bt + gqa, lens, new, bt, 2, gqa, hd), hd ** -0.5)


@pytest.mark.parametrize("hd,gqa", [(128, 4), (256, 4), (128, 1), (256, 6), (128, 8)])
@pytest.mark.parametrize("lens,new", [
    ([500, 3, 0, 300, 64, 1000], [1, 200, 1, 2, 0, 1]),       # single tokens beside a prompt
    ([500, 3, 90, 300, 64, 10], [5, 400, 17, 2, 3, 9]),       # on both sides of the bound
    ([10, 20, 30], [80, 90, 100]), ([0], [130])])             # none to take apart
def test_prompts_with_single_tokens(lens, new, hd, gqa):
    """Slots of few tokens go to a launch of their own where contexts may be long; two of them share the workspace."""
    _check_attn(_attn_case(hd + gqa, lens, new, 16, 2, gqa, hd), hd ** -0.5, max_ctx=1 << 20)


@pytest.mark.parametrize("new", [[1, 1, 1], [6, 1, 9], [70, 3, 100]])
@pytest.mark.parametrize("window,sink", [(1, 0), (20, 0), (64, 4), (100, 33), (5000, 1), (7, 2**31 - 1), (2**31 - 1, 2**31 - 1)])
def test_window_and_sinks(new, window, sink):
    """Exact to the key; pages out of every query's window are given back first."""
    case = _attn_case(window + sum(new), [400, 30, 999], new, 16, 2, 4, 128)
    tables, pos = case[5], case[7]
    for s in range(3):
        for b in range(tables.shape[1]):
            lo, hi = b * 16, b * 16 + 15
            if lo >= sink and hi <= pos[s] - window:
                tables[s, b] = -1
    _check_attn(case, 128 ** -0.5, window, sink)


@pytest.mark.parametrize("new", [[1, 1], [5, 12], [90, 2]])
@pytest.mark.parametrize("hd", [128, 256])
def test_absent_pages(new, hd):
    """Keys of pages outside the pool are not seen, wherever they are; a query that sees none gets zeros."""
    case = _attn_case(7 + hd, [200, 40], new, 16, 2, 4, hd)
    tables = case[5]
    tables[0, 3], tables[0, 4], tables[0, 9] = -1, 10 ** 6, -7
    tables[1, :] = -1
    got = _check_attn(case, 0.1)
    n0 = int(case[6][1])
    assert (got[n0:int(case[6][2])] == 0).all()


@pytest.mark.parametrize("new", [[1, 1], [5, 12], [90, 2]])
@pytest.mark.parametrize("hd", [128, 256])
def test_pages_that_were_never_written(new, hd):
    """Pages in no table hold anything, exponents too: absent pages do not bring in those of another."""
    q, kp, vp, ke, ve, tables, starts, pos = _attn_case(8 + hd, [200, 40], new, 16, 2, 4, hd)
    tables[0, 3], tables[0, 5], tables[1, 1] = -1, len(kp) + 1, -2
    if 0 in tables:   # page 0 is in no table: its own content goes to a new last page
        kp, vp, ke, ve = (np.concatenate([x, x[:1]]) for x in (kp, vp, ke, ve))
        tables[tables == 0] = len(kp) - 1
    for free in sorted(set(range(len(kp))) - set(tables.ravel().tolist())):
        kp[free], vp[free], ke[free], ve[free] = 0x7f, 0xff, 255, 255
    _check_attn((q, kp, vp, ke, ve, tables, starts, pos), 0.1)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 12, 2], [90, 1, 33], [70, 100, 8]])
@pytest.mark.parametrize("bt", [16, 32, 48])
@pytest.mark.parametrize("hd", [128, 256])
def test_pages_reserved_ahead(new, bt, hd):
    """Pages of a slot's table past its last key were never written and hold anything, exponents too: a tile that
    reaches into one is not touched by it."""
    rng = np.random.default_rng(bt + hd + sum(new))
    lens = [200, 40, 7]
    blocks = -(-max(a + b for a, b in zip(lens, new)) // bt) + 6
    tables, starts, pos, n_pages = R.layout(rng, lens, new, bt, 2, hd, spare=blocks, max_blocks=blocks)
    (kp, ke), (vp, ve) = R.random_pool(rng, n_pages, bt, 2, hd), R.random_pool(rng, n_pages, bt, 2, hd)
    free = sorted(set(range(n_pages)) - set(tables.ravel().tolist()))
    kp[free], vp[free], ke[free], ve[free] = 0x7f, 0xff, 255, 255
    for s in range(3):
        ahead = np.flatnonzero(tables[s] < 0)
        tables[s, ahead] = free[:len(ahead)]
    q = rng.standard_normal((int(starts[-1]) + 2, 8, hd)).astype(np.float16)
    _check_attn((q, kp, vp, ke, ve, tables, starts, pos), 0.1)


@pytest.mark.parametrize("new", [[1, 1, 1], [4, 9, 2], [80, 1, 40]])
def test_extreme_scores(new):
    """Peaked rows (one weight is all), a negative scale, and a scale of zero (the mean)."""
    for scale in (6.0, -2.0, 0.0):
        _check_attn(_attn_case(31, [150, 0, 77], new, 32, 1, 4, 128), scale)


def test_exponent_range():
    """Pages of every exponent that the append writes, tiny ones (subnormal fp16 values) and the largest."""
    for new in ([1], [70]):
        rng = np.random.default_rng(4)
        lens, bt, kv, hd = [41 * 16], 16, 1, 128
        tables, starts, pos, n_pages = R.layout(rng, lens, new, bt, kv, hd)
        pools = []
        for which in range(2):
            e = np.full((n_pages, kv), 120, np.uint8)
            e[tables[0, :41], 0] = 95 + np.arange(41)
            code = rng.integers(0, 0x70, (n_pages, bt, kv, hd)).astype(np.uint8) | (rng.integers(0, 2, (n_pages, bt, kv, hd)).astype(np.uint8) << 7)
            # values that fp16 holds, as the append's are: multiples of 2^-24
            val = np.round(R.CODES[code] * 2.0 ** (e[:, None, :, None].astype(float) - 127) * 2.0 ** 24) / 2.0 ** 24
            pools += [R.e4m3_encode(val * 2.0 ** (127 - e[:, None, :, None].astype(float))), e]
        q = (rng.standard_normal((int(starts[-1]), 4, hd)) * 1e-3).astype(np.float16)
        _check_attn((q, pools[0], pools[2], pools[1], pools[3], tables, starts, pos), 1e-3)


def test_output_in_place_of_the_queries():
    for lens, new in (([500, 3], [1, 1]), ([200, 0], [70, 150])):
        case = _attn_case(5, lens, new, 16, 2, 4, 128, spare_rows=0)
        _check_attn(case, 0.09, alias=True)


@pytest.mark.parametrize("lens,new", [([20], [1]), ([900, 5], [1, 1]), ([9000], [1]), ([2000], [12]), ([3000, 4], [90, 7])])
def test_queries_that_are_not_finite(lens, new):
    """A NaN in a query row makes that row NaN, whole or joined from parts, and no other."""
    q, *rest = _attn_case(17, lens, new, 16, 2, 4, 128, spare_rows=0)
    want = _attend(q, *rest, 0.09)
    q[0, 5, 77] = np.nan
    got = _attend(q, *rest, 0.09)
    assert np.isnan(got[0, 5]).all()
    got[0, 5] = want[0, 5]
    assert np.array_equal(got, want)


def test_context_limit():
    """Keys at or past max_ctx are not seen, and a larger table is not read."""
    case = _attn_case(6, [300, 100], [1, 1], 16, 1, 4, 128)
    _check_attn(case, 0.09, max_ctx=200)


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 9, 2], [16, 1, 12], [70, 300, 5]])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("max_ctx,window,sink", [(200, 50, 40), (200, 1, 200), (333, 64, 100), (33, 20, 1)])
def test_sinks_past_the_context_limit(new, hd, max_ctx, window, sink):
    """Queries whose window lies past max_ctx see the sinks, all of them, and nothing else."""
    got = _check_attn(_attn_case(hd + sum(new) + sink, [400, 30, 1000], new, 16, 2, 4, hd), 0.09, window, sink, max_ctx=max_ctx)
    assert np.abs(got[0]).max() > 0   # (the first slot's queries are past the limit by more than the window)


def test_starts_out_of_order():
    """Starts that decrease name the same rows again and again: 2^32 key tiles of a head here, which is no call
    that can be carried out (nothing is), and a few, which is."""
    rows, slots, ctx = 16384, 64, 1 << 24
    q = torch.zeros((rows, 4, 128), dtype=torch.float16, device=DEV)
    pool, exp = torch.zeros((2, 16384, 1, 128), dtype=torch.uint8, device=DEV), torch.full((2, 1), 120, dtype=torch.uint8, device=DEV)
    tables = torch.full((slots, ctx // 16384), -1, dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, rows] * (slots // 2) + [0], dtype=torch.int32, device=DEV)
    ws = kvcache.attn_f8_paged_workspace(4, 1, slots, rows, rows, ctx, DEV, head_dim=128)
    for pos, want in ((ctx - rows, 5.0), (0, 0.0)):
        out = torch.full_like(q, 5.0)
        at = torch.full((slots,), pos, dtype=torch.int32, device=DEV)
        kvcache.attn_f8_paged(q, pool, pool, exp, exp, out, ws, tables, starts, at, max_tok=rows, max_ctx=ctx, scale=0.1)
        assert (out == want).all()


def test_more_than_four_billion_merge_threads():
    """32,771 slots of 64 rows of eight heads, some of them cut between parts: each slot's rows as the one slot's
    of the reference."""
    slots, kv, gqa, tok, bt, hd = 32771, 8, 8, 8, 16, 128
    one = _attn_case(77, [140], [tok], bt, kv, gqa, hd, spare_rows=0)
    q, kp, vp, ke, ve, tables, _, _ = one
    ref, tol = R.attention(*one[:6], [0, tok], [140], 0.09)
    qd = dev(q).repeat(slots, 1, 1)
    out = torch.zeros_like(qd)
    starts = torch.arange(0, slots * tok + 1, tok, dtype=torch.int32, device=DEV)
    pos = torch.full((slots,), 140, dtype=torch.int32, device=DEV)
    ws = kvcache.attn_f8_paged_workspace(kv * gqa, kv, slots, slots * tok, tok, 148, DEV, head_dim=hd)
    kvcache.attn_f8_paged(qd, dev(kp), dev(vp), dev(ke), dev(ve), out, ws, dev(tables).repeat(slots, 1), starts, pos,
                          max_tok=tok, max_ctx=148, scale=0.09)
    del qd
    rd, td = dev(ref), dev(tol)
    for part in out.view(slots, tok, kv * gqa, hd).split(1024):
        assert ((part.double() - rd).abs() <= td).all()


def test_same_result_every_time_and_on_another_stream():
    case = _attn_case(8, [3000, 10, 700], [1, 1, 1], 64, 2, 4, 256)
    a = _attend(*case, 0.06)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = _attend(*case, 0.06)
    assert np.array_equal(a, b)
    case = _attn_case(8, [300, 0], [90, 300], 64, 2, 4, 256)
    assert np.array_equal(_attend(*case, 0.06), _attend(*case, 0.06))


def test_one_workspace_for_calls_of_every_shape():
    """Short and long contexts, single tokens and prompts in turn on one workspace, without a reset."""
    cases = [(_attn_case(11, [300, 900, 5], [1, 1, 1], 16, 2, 4, 128), 0.09), (_attn_case(12, [3000], [1], 64, 2, 4, 128), 0.09),
             (_attn_case(13, [20, 0], [70, 130], 16, 2, 4, 128), 0.09), (_attn_case(14, [700] * 9, [1] * 9, 16, 2, 4, 128), 0.09),
             (_attn_case(15, [64, 300], [9, 16], 16, 2, 4, 128), 0.09)]
    want = [_attend(*c, f) for c, f in cases]
    ws = kvcache.attn_f8_paged_workspace(8, 2, 9, 1000, 200, 4000, DEV, head_dim=128)
    for turn in range(3):
        for (c, f), w in zip(cases, want):
            q, kp, vp, ke, ve, tables, starts, pos = map(dev, c)
            n = np.diff(c[6])
            out = torch.full_like(q, 9.0)
            kvcache.attn_f8_paged(q, kp, vp, ke, ve, out, ws, tables, starts, pos, max_tok=int(n.max()),
                                  max_ctx=int((c[7] + n).max()), scale=f)
            assert np.array_equal(out.cpu().numpy(), w), turn


def test_offsets_past_four_gigabytes():
    """A pool of more than 2^32 bytes, the slot in its last pages: the same bits as in a small pool."""
    case = _attn_case(9, [900], [1], 64, 4, 4, 256, spare_rows=0)
    q, kp, vp, ke, ve, tables, starts, pos = case
    small = _attend(*case, 0.06)
    n = (1 << 32) // (64 * 4 * 256) + 40
    kb, vb = (torch.zeros((n, 64, 4, 256), dtype=torch.uint8, device=DEV) for _ in range(2))
    keb, veb = (torch.zeros((n, 4), dtype=torch.uint8, device=DEV) for _ in range(2))
    m = len(kp)
    for big, x in ((kb, kp), (vb, vp), (keb, ke), (veb, ve)):
        big[n - m:] = dev(x)
    far = np.where(tables >= 0, tables + n - m, tables).astype(np.int32)
    out = torch.empty_like(dev(q))
    ws = kvcache.attn_f8_paged_workspace(16, 4, 1, 1, 1, 901, DEV, head_dim=256)
    kvcache.attn_f8_paged(dev(q), kb, vb, keb, veb, out, ws, dev(far), dev(starts), dev(pos), max_tok=1, max_ctx=901, scale=0.06)
    assert np.array_equal(out.cpu().numpy(), small)
    # and the append there
    k = dev(np.ones((1, 4, 256), np.float16))
    kvcache.f8_append_kv_paged(k, k, kb, vb, keb, veb, dev(far), dev(starts), dev(pos), max_tok=1)
    page = int(far[0, 900 // 64])
    e = keb[page].cpu().numpy().astype(float)
    assert (R.CODES[kb[page, 900 % 64].cpu().numpy()] * 2.0 ** (e - 127)[:, None] == 1).all()


def _check_many_slots(case, order, scale, max_ctx=None):
    """A batch whose slot i is slot order[i] of `case`: every row as the reference's of that slot."""
    q, kp, vp, ke, ve, tables, starts, pos = case
    ref, tol = R.attention(q, kp, vp, ke, ve, tables, starts.tolist(), pos.tolist(), scale)
    n = np.diff(starts)
    rows = np.concatenate([np.arange(starts[s], starts[s + 1]) for s in order])
    first = np.cumsum([0] + [n[s] for s in order]).astype(np.int32)
    big = np.concatenate([q[rows], q[:3]])   # (and rows behind the last slot)
    got = _attend(big, kp, vp, ke, ve, tables[order], first, pos[order], scale, max_ctx=max_ctx)
    assert (got[len(rows):] == 9.0).all()
    err = np.abs(got[:len(rows)].astype(np.float64) - ref[rows])
    bad = np.flatnonzero((err > tol[rows]).any((1, 2)))
    assert not len(bad), (len(bad), bad[:5], err.max())


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("max_ctx", [None, 1 << 17])   # (by the contexts; prompts and the others in launches of their own)
@pytest.mark.parametrize("slots", [64, 65, 130, 600])
@pytest.mark.parametrize("new,gqa", [
    ([1, 1, 0, 1, 1], 4), ([5, 9, 0, 2, 1], 4), ([5, 8, 0, 2, 3], 8), ([40, 33, 0, 65, 1], 8)])
def test_many_slots(new, gqa, slots, max_ctx, hd):
    """More slots than a wave or a workgroup takes up at a time, runs of slots without rows among them, and more row
    tiles than slots at a time."""
    rng = np.random.default_rng(slots + hd + gqa)
    order = rng.integers(0, 5, slots)
    order[20:min(160, slots - 10)] = np.where(rng.random(min(160, slots - 10) - 20) < 0.02, 1, 2)
    if slots > 300:
        order[200:420] = 2
    if max(new) > 64:   # (few of the longest)
        order = np.where((order == 3) & (rng.random(slots) < 0.8), 0, order)
    _check_many_slots(_attn_case(slots, [40, 300, 10, 5, 700], new, 16, 2, gqa, hd), order, hd ** -0.5, max_ctx)


@pytest.mark.parametrize("hd", [128, 256])
def test_prompts_beside_many_slots(hd):
    """A few prompts among 600 single tokens, in one launch and in two."""
    rng = np.random.default_rng(hd)
    order = rng.integers(0, 3, 600)
    order[[0, 77, 511, 512, 599]] = 3
    for max_ctx in (None, 1 << 17):
        _check_many_slots(_attn_case(hd, [90, 3, 10, 50], [1, 1, 0, 300], 32, 1, 4, hd), order, hd ** -0.5, max_ctx)


@pytest.mark.parametrize("new", [[1, 1], [5, 12], [16, 3], [90, 300]])
@pytest.mark.parametrize("hd", [128, 256])
def test_context_limit_of_every_kernel(new, hd):
    """As test_context_limit, for up to 16 rows, up to 64 and more, with the limit inside a slot's new rows and ahead
    of them."""
    for max_ctx in (100, 310, 200):
        _check_attn(_attn_case(hd + max_ctx, [300, 30], new, 16, 2, 4, hd), 0.09, max_ctx=max_ctx)


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("lens,new,gqa", [([20000], [1], 4), ([9000, 12000], [1, 1], 1), ([20000], [12], 2), ([17000, 3], [10, 9], 6)])
def test_merges_of_many_records(lens, new, gqa, hd):
    """Row tiles in more than 64 parts, the records that the merge takes up at a time."""
    _check_attn(_attn_case(hd + gqa, lens, new, 64, 1, gqa, hd), hd ** -0.5)


@pytest.mark.parametrize("new", [[1, 1, 1], [6, 1, 9], [16, 3, 12], [70, 3, 100]])
@pytest.mark.parametrize("window,sink", [(1, 0), (20, 0), (64, 4), (100, 33), (300, 70), (5000, 1), (7, 2**31 - 1)])
def test_window_and_sinks_of_wide_heads(new, window, sink):
    """As test_window_and_sinks, at head_dim 256, with every page that no query sees given back."""
    case = _attn_case(window + sum(new), [400, 30, 999], new, 16, 2, 4, 256)
    tables, pos = case[5], case[7]
    for s in range(3):
        for b in range(tables.shape[1]):
            if b * 16 >= sink and b * 16 + 15 <= pos[s] - window:
                tables[s, b] = -1
    _check_attn(case, 256 ** -0.5, window, sink)


def test_calls_on_a_given_stream():
    """Rotation, append and attention with stream=: what they give on the current stream."""
    rng = np.random.default_rng(12)
    s = torch.cuda.Stream()
    tables, starts, pos, n_pages = R.layout(rng, [30, 100, 0], [1, 20, 90], 16, 2, 128)
    rows = int(starts[-1])
    q, k, v = (dev(rng.standard_normal((rows, h, 128)).astype(np.float16)) for h in (8, 2, 2))
    at = dev(np.concatenate([pos[i] + np.arange(starts[i + 1] - starts[i]) for i in range(3)]).astype(np.int32))
    idx = [dev(x) for x in (tables, starts, pos)]
    t = kvcache.rope_table(64, device=DEV)
    pools = [dev(x) for x in (*R.random_pool(rng, n_pages, 16, 2, 128), *R.random_pool(rng, n_pages, 16, 2, 128))]
    ws = [kvcache.attn_f8_paged_workspace(8, 2, 3, rows, 90, 128, DEV, head_dim=128) for _ in range(2)]

    def run(stream, w):
        kp, ke, vp, ve = [x.clone() for x in pools]
        qr, qa, out = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        kvcache.rope(q, None, at, t, q_out=qr, stream=stream)
        kvcache.f8_append_kv_paged(k, v, kp, vp, ke, ve, *idx, max_tok=90, q=q, q_out=qa, rope=t, stream=stream)
        kvcache.attn_f8_paged(qr, kp, vp, ke, ve, out, w, *idx, max_tok=90, max_ctx=128, scale=0.09, stream=stream)
        if stream is not None:
            stream.synchronize()
        return qr, qa, kp, vp, ke, ve, out
    for x, y in zip(run(None, ws[0]), run(s, ws[1])):
        assert torch.equal(x, y)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

class Server:
    """A layer's state, its buffers and one decode step of all slots over them."""

    def __init__(self, seed, slots=6, bt=16, kv=2, gqa=4, hd=128, n_pages=80):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.bt, self.kv, self.nq, self.hd, self.slots = bt, kv, kv * gqa, hd, slots
        self.kp, self.ke = kvcache.f8_pool(n_pages, bt, kv, hd, DEV)
        self.vp, self.ve = kvcache.f8_pool(n_pages, bt, kv, hd, DEV)
        self.tables = torch.full((slots, 20), -1, dtype=torch.int32, device=DEV)
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
        self.planes = kvcache.page_planes([self.kp, self.vp, self.ke, self.ve])
        self.table = kvcache.rope_table(64, device=DEV)
        self.i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        self.all, self.one = self.i(list(range(slots))), self.i([1] * slots)
        self.starts, self.pos = self.i(list(range(slots + 1))), self.i([0] * slots)
        self.status = self.i([0] * slots)
        self.qkv = torch.zeros(slots, self.nq + 2 * kv, hd, dtype=torch.float16, device=DEV)
        self.q = torch.zeros(slots, self.nq, hd, dtype=torch.float16, device=DEV)
        self.out = torch.zeros_like(self.q)
        self.ws = kvcache.attn_f8_paged_workspace(self.nq, kv, slots, slots, 1, 320, DEV, head_dim=hd)
        self.scratch = torch.zeros(1000, dtype=torch.int32, device=DEV)
        self.g = g

    def rows(self, n):
        return torch.randn(n, self.nq + 2 * self.kv, self.hd, device=DEV, generator=self.g).half()

    def prompt(self, slot, n):
        """A prompt's rows: reserved, appended, attended."""
        x = self.rows(n)
        q, k, v = x[:, :self.nq], x[:, self.nq:self.nq + self.kv], x[:, self.nq + self.kv:]
        t = self.tables[slot:slot + 1]
        kvcache.pages_reserve(self.tables, self.refs, self.i([slot]), self.i([0]), self.i([n]), self.status[:1], self.planes,
                              block_tokens=self.bt, max_new=n)
        starts, pos = self.i([0, n]), self.i([0])
        qr = torch.empty(n, self.nq, self.hd, dtype=torch.float16, device=DEV)
        kvcache.f8_append_kv_paged(k, v, self.kp, self.vp, self.ke, self.ve, t, starts, pos, max_tok=n, q=q, q_out=qr,
                                   rope=self.table)
        out = torch.empty_like(qr)
        ws = kvcache.attn_f8_paged_workspace(self.nq, self.kv, 1, n, n, n, DEV, head_dim=self.hd)
        kvcache.attn_f8_paged(qr, self.kp, self.vp, self.ke, self.ve, out, ws, t, starts, pos, max_tok=n, max_ctx=n, scale=0.1)
        self.pos[slot] = n
        return qr, out

    def step(self):
        kv, nq = self.kv, self.nq
        kvcache.pages_reserve(self.tables, self.refs, self.all, self.pos, self.one, self.status, self.planes,
                              block_tokens=self.bt, max_new=1, scratch=self.scratch)
        kvcache.f8_append_kv_paged(self.qkv[:, nq:nq + kv], self.qkv[:, nq + kv:], self.kp, self.vp, self.ke, self.ve,
                                   self.tables, self.starts, self.pos, max_tok=1, q=self.qkv[:, :nq], q_out=self.q,
                                   rope=self.table)
        kvcache.attn_f8_paged(self.q, self.kp, self.vp, self.ke, self.ve, self.out, self.ws, self.tables, self.starts,
                              self.pos, max_tok=1, max_ctx=320, scale=0.1)
        self.pos.add_(1)

    def reference(self, q, rows_pos):
        """64-bit attention of q over what the pools hold."""
        a = [x.cpu().numpy() for x in (q, self.kp, self.vp, self.ke, self.ve, self.tables)]
        return R.attention(*a, list(range(len(rows_pos) + 1)), list(rows_pos), 0.1)


def test_prompts_forks_steps_and_release():
    """Prompts, forked children, decode steps that copy shared pages, a slot given back, the pool compacted."""
    s = Server(1)
    qr, out = s.prompt(0, 37)
    s.prompt(1, 100)
    a = [x.cpu().numpy() for x in (qr, s.kp, s.vp, s.ke, s.ve, s.tables[:1])]
    ref, tol = R.attention(*a, [0, 37], [0], 0.1)
    assert (np.abs(out.cpu().numpy() - ref) <= tol).all()
    kvcache.pages_fork(s.tables, s.refs, s.i([0, 1, 0]), s.i([2, 3, 4]), s.i([37, 100, 32]), s.status[:3], block_tokens=s.bt)
    s.pos.copy_(s.i([37, 100, 37, 100, 32, 0]))
    before = s.kp[s.tables[0, 0].item()].clone()
    for step in range(20):
        s.qkv.copy_(s.rows(s.slots))
        pos = s.pos.tolist()
        s.step()
        assert s.status.tolist() == [0] * 6
        ref, tol = s.reference(s.q, pos)
        assert (np.abs(s.out.cpu().numpy() - ref) <= tol).all(), step
    # the shared prompt pages were left alone, the written ones belong to one slot each
    assert torch.equal(s.kp[s.tables[0, 0].item()], before) and s.tables[0, 0] == s.tables[2, 0]
    assert s.tables[0, 2] != s.tables[2, 2] and s.tables[1, 6] != s.tables[3, 6]
    counts = np.bincount(s.tables[s.tables >= 0].cpu().numpy(), minlength=80)
    assert np.array_equal(counts, s.refs.cpu().numpy())
    kvcache.pages_release(s.tables, s.refs, s.i([1, 0]), s.i([0, 40]), block_tokens=s.bt)
    s.pos.copy_(s.i([-1, -1] + s.pos.tolist()[2:]))
    moved, used = s.i([0] * 80), s.i([0])
    kvcache.pages_compact(s.tables, s.refs, moved, used, s.planes)
    assert (s.refs[:used.item()] > 0).all() and (s.refs[used.item():] == 0).all()
    live = s.pos.tolist()[2:]
    q = s.rows(4)[:, :s.nq].contiguous()
    got = torch.empty_like(q)
    t = s.tables[2:].contiguous()
    ws = kvcache.attn_f8_paged_workspace(s.nq, s.kv, 4, 4, 1, 320, DEV, head_dim=s.hd)
    kvcache.attn_f8_paged(q, s.kp, s.vp, s.ke, s.ve, got, ws, t, s.i([0, 1, 2, 3, 4]), s.i([p - 1 for p in live]), max_tok=1,
                          max_ctx=320, scale=0.1)
    a = [x.cpu().numpy() for x in (q, s.kp, s.vp, s.ke, s.ve, t)]
    ref, tol = R.attention(*a, [0, 1, 2, 3, 4], [p - 1 for p in live], 0.1)
    assert (np.abs(got.cpu().numpy() - ref) <= tol).all()


def test_captured_steps():
    """Two graphs of the whole decode step over one workspace, replayed in turn with eager steps between:
    every step's output, tables and pools equal an eager server's."""
    a, b = Server(2), Server(2)
    for s in (a, b):
        s.prompt(0, 30)
        s.prompt(1, 63)
        kvcache.pages_fork(s.tables, s.refs, s.i([0, 1]), s.i([2, 3]), s.i([30, 63]), block_tokens=s.bt)
        s.pos.copy_(s.i([30, 63, 30, 63, 0, 0]))
    a.qkv.copy_(a.rows(6))
    b.qkv.copy_(b.rows(6))
    a.step()
    b.step()
    keep = [x.clone() for x in (a.kp, a.vp, a.ke, a.ve, a.tables, a.refs, a.pos)]
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a.step()
        graphs.append(g)
    for x, y in zip((a.kp, a.vp, a.ke, a.ve, a.tables, a.refs, a.pos), keep):
        x.copy_(y)
    for step in range(12):
        x = a.rows(6)
        b.rows(6)
        a.qkv.copy_(x)
        b.qkv.copy_(x)
        if step % 3 == 2:
            a.step()
        else:
            graphs[step % 3].replay()
        b.step()
        for p, q in ((a.out, b.out), (a.kp, b.kp), (a.ve, b.ve), (a.tables, b.tables), (a.refs, b.refs), (a.pos, b.pos)):
            assert torch.equal(p, q), step


def test_captured_prompts_and_two_streams():
    """A captured batch of prompts and single tokens (two launches and both merges), replayed with new queries and
    eager calls on the same workspace between; and the same batches on two streams at once."""
    cases = [_attn_case(41, [3000, 0, 900, 700], [1, 300, 1, 2], 16, 2, 4, 128), _attn_case(42, [0, 2500], [500, 1], 64, 2, 4, 256)]
    calls = []
    for case in cases:
        q, kp, vp, ke, ve, tables, starts, pos = map(dev, case)
        mt, rows = int(np.diff(case[6]).max()), q.shape[0]
        ws = [kvcache.attn_f8_paged_workspace(8, 2, len(pos), rows, mt, 1 << 17, DEV, head_dim=q.shape[2]) for _ in range(2)]

        def call(out, w, q=q, rest=(kp, vp, ke, ve), idx=(tables, starts, pos), mt=mt):
            kvcache.attn_f8_paged(q, *rest, out, w, *idx, max_tok=mt, max_ctx=1 << 17, scale=0.09)
        calls.append((q, ws, call))
    for q, ws, call in calls:
        out, want = torch.full_like(q, 9.0), torch.full_like(q, 9.0)
        call(out, ws[0])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(out, ws[0])
        for step in range(5):
            q.copy_(torch.randn(q.shape, device=DEV).half())
            out.fill_(9.0)
            g.replay()
            call(want, ws[0] if step % 2 else ws[1])
            assert torch.equal(out, want), step
    # at once: each stream with its own workspace
    want = []
    for q, ws, call in calls:
        want.append(torch.full_like(q, 9.0))
        call(want[-1], ws[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[torch.full_like(q, 9.0) for q, _, _ in calls] for _ in streams]
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            for _ in range(4):
                for out, (q, ws, call) in zip(got[i], calls):
                    call(out, ws[i])
    torch.cuda.synchronize()
    for outs in got:
        for out, w in zip(outs, want):
            assert torch.equal(out, w)
