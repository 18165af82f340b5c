"""Refusals of the operators around the paged 8-bit cache in a decoding loop before anything is launched, their
workspace queries, and the references that the GPU tests use against plain ones."""
import ctypes

import numpy as np
import pytest
import torch

from qengine_amd import _lib, kvcache
from tests import _loop as R

OK, INVALID, NULL, UNSUPPORTED, ALIGN, WORKSPACE = 0, -1, -2, -3, -4, -7


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(1 << 16)
    test_buf.append(buf)
    return (ctypes.addressof(buf) + 255) & ~255


test_buf = []


def _each(f, code, **calls):
    """f of each keyword alone gives the code"""
    for k, values in calls.items():
        for v in values:
            assert f(**{k: v}) == code, (k, v, f(**{k: v}))


# ---- the C entry points -----------------------------------------------------

def test_norm_refusals(L, p):
    def f(**kw):
        a = dict(q=p, qs=512, qo=p, qos=512, qw=p, k=p + 64, ks=256, ko=p + 64, kos=256, kw=None, eps=1e-6, pos=p, t=p, n=4,
                 nq=4, nk=2, hd=128, rot=64, lay=0)
        a.update(kw)
        return L.qkv_norm_rope(a["q"], a["qs"], a["qo"], a["qos"], a["qw"], a["k"], a["ks"], a["ko"], a["kos"], a["kw"],
                               a["eps"], a["pos"], a["t"], 1.0, a["n"], a["nq"], a["nk"], a["hd"], a["rot"], a["lay"], None)
    assert f(n=0) == OK
    nan = float("nan")
    _each(f, INVALID, n=[-1], nq=[-1, 1025], nk=[-1, 1025], hd=[0, -16], rot=[-2, 63, 130], lay=[-1, 2],
          eps=[0.0, -1e-6, nan, float("inf"), 1e-60], qs=[511], ks=[255], qos=[1024], kos=[512])
    assert f(nq=0, nk=0) == f(ko=p) == INVALID
    _each(f, UNSUPPORTED, hd=[1025, 4096], n=[2**31 - 1])
    _each(f, NULL, q=[None], qo=[None], k=[None], ko=[None], pos=[None], t=[None])
    _each(f, ALIGN, qw=[p + 2], kw=[p + 1], pos=[p + 2], t=[p + 4])
    assert f(q=p + 1, qo=p + 1) == ALIGN
    # a side without heads is not looked at, nor are a rotation's tables without one
    assert f(n=0, nq=0, q=None, qo=None) == f(n=0, rot=0, pos=None, t=None) == OK


def test_norm_refuses_more_rows_than_workgroups_are_counted(L, p):
    """2^34 rows and 2,048 more, of a size that takes a wave a row."""
    assert L.qkv_norm_rope(p, 2048, p, 2048, None, p + 64, 2048, p + 64, 2048, None, 1e-6, p, p, 1.0, 8388609, 1024, 1024, 2, 2,
                           0, None) == UNSUPPORTED


def test_norm_gradient_refusals(L, p):
    ws = L.qkv_norm_rope_grad_workspace_bytes(4, 4, 2, 128)
    assert ws > 0

    def f(**kw):
        a = dict(q=p, qs=512, qd=p + 4096, qds=512, qx=p + 4096, qxs=512, qw=p, qg=p, k=p + 64, ks=256, kd=p + 8192, kds=256,
                 kx=p + 8192, kxs=256, kw=None, kg=p + 1024, eps=1e-6, pos=p, t=p, n=4, nq=4, nk=2, hd=128, rot=64, lay=0,
                 ws=p, wb=ws)
        a.update(kw)
        return L.qkv_norm_rope_grad(a["q"], a["qs"], a["qd"], a["qds"], a["qx"], a["qxs"], a["qw"], a["qg"], a["k"], a["ks"],
                                    a["kd"], a["kds"], a["kx"], a["kxs"], a["kw"], a["kg"], a["eps"], a["pos"], a["t"], 1.0,
                                    a["n"], a["nq"], a["nk"], a["hd"], a["rot"], a["lay"], a["ws"], a["wb"], None)
    assert f(n=0, qg=None, kg=None) == OK
    _each(f, INVALID, n=[-1], nq=[-1, 1025], nk=[-1], hd=[0], rot=[-2, 63, 130], lay=[-1, 2], eps=[0.0, float("nan")],
          qs=[511], qds=[511], qxs=[511, 1024], ks=[255], kds=[255, 512], kg=[p], kx=[p + 4096])
    _each(f, UNSUPPORTED, hd=[1025], n=[2**31 - 1])
    _each(f, NULL, q=[None], qd=[None], qx=[None], k=[None], kd=[None], kx=[None], pos=[None], t=[None])
    _each(f, ALIGN, q=[p + 1], qw=[p + 2], qg=[p + 2], kg=[p + 2], pos=[p + 1], t=[p + 4], ws=[p + 2])
    _each(f, WORKSPACE, ws=[None], wb=[0, ws - 1])
    w = L.qkv_norm_rope_grad_workspace_bytes
    assert w(4, 0, 0, 128) == w(4, -1, 2, 128) == w(-1, 4, 2, 128) == w(4, 4, 2, 0) == w(4, 4, 2, 1025) == 0
    # the workspace of more tokens, heads and elements serves fewer
    for hd in (10, 128, 1024):
        sizes = [[w(n, nq, 2, hd) for nq in (0, 1, 8, 64)] for n in (0, 1, 33, 1000, 40000)]
        assert (np.diff(sizes, axis=0) >= 0).all() and (np.diff(sizes, axis=1) >= 0).all()


def test_weighing_refusals(L, p):
    ws = L.qkv_weigh_f8_paged_workspace_bytes(8, 2, 128, 2, 4, 2, 100)
    assert ws > 0

    def f(**kw):
        a = dict(q=p, kp=p, ke=p, w=p, rows=4, nq=8, kv=2, hd=128, slots=2, mt=2, mc=100, bt=p, mb=8, bl=16, np=8, st=p, pos=p,
                 wd=None, d=1.0, win=0, s=0, ws=p, wb=ws)
        a.update(kw)
        return L.qkv_weigh_f8_paged(a["q"], a["kp"], a["ke"], a["w"], a["rows"], a["nq"], a["kv"], a["hd"], a["slots"],
                                    a["mt"], a["mc"], a["bt"], a["mb"], a["bl"], a["np"], a["st"], a["pos"], a["wd"],
                                    a["d"], 0.1, a["win"], a["s"], a["ws"], a["wb"], None)
    assert f(rows=0) == f(slots=0) == f(mt=0) == OK
    _each(f, INVALID, rows=[-1], slots=[-1], mt=[-1], mc=[0, -1], nq=[7, 0], kv=[0], np=[0], mb=[0], bl=[0], win=[-1],
          s=[-1], d=[float("nan"), float("inf")])
    _each(f, UNSUPPORTED, nq=[18, 1026], hd=[64, 192], bl=[8, 1 << 23], mc=[(1 << 30) + 1])
    _each(f, NULL, q=[None], kp=[None], ke=[None], w=[None], bt=[None], st=[None], pos=[None])
    _each(f, ALIGN, q=[p + 8], kp=[p + 8], w=[p + 2], bt=[p + 2], st=[p + 1], pos=[p + 2], wd=[p + 2], ws=[p + 16])
    # (the query counts the largest of the smaller calls too: this one's own need is a part of it)
    _each(f, WORKSPACE, ws=[None], wb=[0, 1024])
    w = L.qkv_weigh_f8_paged_workspace_bytes
    assert w(8, 3, 128, 2, 4, 2, 100) == w(8, 2, 64, 2, 4, 2, 100) == w(8, 2, 128, 0, 4, 2, 100) == 0
    assert w(8, 2, 128, 2, 4, 100, 100) == w(8, 2, 128, 2, 4, 4, 100)   # no slot has more rows than the call
    # the stated limit suffices, and far past it nothing is taken
    for slots, kv, tok, ctx in ((1, 4, 1 << 20, 1 << 15), (64, 8, 4096, 1 << 16), (1 << 12, 8, 1, 1 << 20), (1, 8, 1, 1 << 30),
                                (40, 1, 1, 1 << 30), (1, 1, 1 << 20, 2000000), (10600, 8, 1, 1 << 20), (1, 8, 4096, 130000000)):
        assert slots * max(kv, 2) * (tok * 4 / 32 + 6) * (ctx / 256 + 6) < 2.0 ** 31
        assert w(4 * kv, kv, 256, slots, slots * tok if slots * tok < 2**31 else 2**31 - 1, tok, ctx) > 0
    assert w(32, 8, 256, 1 << 16, 1 << 16, 1, 1 << 30) == w(32, 8, 256, 1, 1 << 24, 1 << 24, 1 << 26) == 0


@pytest.mark.parametrize("head_dim", [128, 256])
@pytest.mark.parametrize("num_q,num_kv", [(8, 8), (9, 3), (16, 4), (20, 4), (14, 2), (32, 4)])
def test_weighing_workspace_serves_smaller_calls(num_q, num_kv, head_dim):
    """The size never falls as any of the numbers grows."""
    size = _lib.lib().qkv_weigh_f8_paged_workspace_bytes
    grid = [(1, 2, 4, 33, 64, 65, 300), (1, 4, 17, 64, 300, 5000), (1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 32, 33, 64, 65, 257, 3000),
            (1, 31, 64, 65, 127, 129, 511, 1025, 2048, 2049, 65536, 1 << 20)]
    need = {}
    for slots in grid[0]:
        for rows in grid[1]:
            for tok in grid[2]:
                for ctx in grid[3]:
                    need[slots, rows, tok, ctx] = size(num_q, num_kv, head_dim, slots, rows, tok, ctx)
    assert min(need.values()) > 0
    for at, n in need.items():
        for i in range(4):
            up = grid[i].index(at[i]) + 1
            if up < len(grid[i]):
                more = at[:i] + (grid[i][up],) + at[i + 1:]
                assert need[more] >= n, (at, more)


def test_eviction_refusals(L, p):
    ws = L.qkv_evict_f8_paged_workspace_bytes(2, 2, 16, 100, 50)
    assert ws > 0

    def f(**kw):
        a = dict(kp=p, vp=p, ke=p, ve=p, w=p, slots=2, kv=2, hd=128, mc=100, mk=50, bt=p, mb=8, bl=16, np=8, ln=p, kn=p, s=0,
                 r=0, kept=p, ws=p, wb=ws)
        a.update(kw)
        return L.qkv_evict_f8_paged(a["kp"], a["vp"], a["ke"], a["ve"], a["w"], a["slots"], a["kv"], a["hd"], a["mc"], a["mk"],
                                    a["bt"], a["mb"], a["bl"], a["np"], a["ln"], a["kn"], a["s"], a["r"], a["kept"],
                                    a["ws"], a["wb"], None)
    assert f(slots=0) == f(mk=0) == OK
    _each(f, INVALID, slots=[-1], kv=[0], mc=[-1], mk=[-1], mb=[0], bl=[0], np=[0], s=[-1], r=[-1])
    _each(f, UNSUPPORTED, hd=[64, 192], bl=[24, 1 << 23], mc=[(1 << 30) + 1], mk=[(1 << 30) + 1], slots=[1 << 23])
    _each(f, NULL, kp=[None], vp=[None], ke=[None], ve=[None], w=[None], bt=[None], ln=[None], kn=[None], kept=[None])
    _each(f, ALIGN, kp=[p + 8], vp=[p + 4], w=[p + 2], bt=[p + 1], ln=[p + 2], kn=[p + 2], kept=[p + 2], ws=[p + 2])
    _each(f, WORKSPACE, ws=[None], wb=[0, ws - 1])
    w = L.qkv_evict_f8_paged_workspace_bytes
    assert w(0, 2, 16, 100, 50) == w(-1, 2, 16, 100, 50) == w(2, 0, 16, 100, 50) == w(2, 2, 0, 100, 50) == 0
    assert w(2, 2, 16, -1, 50) == w(2, 2, 16, 100, -1) == w(2, 2, 16, (1 << 30) + 1, 50) == 0
    # n_slots * num_kv * (max_ctx / 4096 + 1) up to 2^22, and * (max_keep / 64 + 1) up to 2^24
    assert w(1 << 10, 8, 16, 4096 * 510, 64) > 0 == w(1 << 10, 8, 16, 4096 * 511, 64)
    assert w(1 << 10, 8, 16, 4096, 64 * 2046) > 0 == w(1 << 10, 8, 16, 4096, 64 * 2047)
    # larger numbers serve smaller ones (a context's stretches are of a long one only)
    grid = [(1, 2, 24), (1, 4, 8), (0, 1, 4096, 16384, 16385, 40000, 1 << 20), (1, 63, 64, 5000, 1 << 17)]
    sizes = np.array([[[[w(s, kv, 16, c, k) for k in grid[3]] for c in grid[2]] for kv in grid[1]] for s in grid[0]], np.int64)
    assert sizes.min() > 0 and all((np.diff(sizes, axis=i) >= 0).all() for i in range(4))


def test_beam_refusals(L, p):
    ws = L.qkv_beam_select_workspace_bytes(3, 4, 1000, 8)
    assert ws > 0

    def f(**kw):
        a = dict(l=p, ty=0, st=1000, s=p, d=None, e=0, n=3, b=4, v=1000, t=8, pa=p, to=p, top=p, ws=p, wb=ws)
        a.update(kw)
        return L.qkv_beam_select(a["l"], a["ty"], a["st"], a["s"], a["d"], a["e"], a["n"], a["b"], a["v"], a["t"], a["pa"],
                                 a["to"], a["top"], a["ws"], a["wb"], None)
    assert f(n=0) == OK
    _each(f, INVALID, n=[-1], b=[0], v=[0], t=[0], ty=[-1, 3], st=[999, 0, -1000])
    assert f(d=p, e=-1) == f(d=p, e=1000) == INVALID
    assert f(n=0, e=-1) == OK     # (no beam has ended: the token is not read)
    _each(f, UNSUPPORTED, b=[65], t=[65], v=[1 << 30], n=[(1 << 22) + 1])
    _each(f, NULL, l=[None], s=[None], pa=[None], to=[None], top=[None])
    _each(f, ALIGN, l=[p + 1], s=[p + 2], d=[p + 2], pa=[p + 1], to=[p + 2], top=[p + 2], ws=[p + 4])
    assert f(ty=1, l=p + 2) == ALIGN
    _each(f, WORKSPACE, ws=[None], wb=[0, ws - 1])
    w = L.qkv_beam_select_workspace_bytes
    assert w(0, 4, 1000, 8) == w(3, 0, 1000, 8) == w(3, 65, 1000, 8) == w(3, 4, 0, 8) == w(3, 4, 1000, 65) == 0
    grid = [(1, 2, 64), (1, 4, 64), (1, 1000, 8191, 131072, 1 << 20), (1, 8, 64)]
    sizes = np.array([[[[w(n, b, v, t) for t in grid[3]] for v in grid[2]] for b in grid[1]] for n in grid[0]], np.int64)
    assert sizes.min() > 0 and all((np.diff(sizes, axis=i) >= 0).all() for i in range(4))


def test_reorder_refusals(L, p):
    planes = (kvcache._Plane * 2)(kvcache._Plane(p, 64), kvcache._Plane(p + 4096, 3))
    pl = ctypes.addressof(planes)

    def f(**kw):
        a = dict(t=p, ns=2000, mb=8, bl=16, r=p, np=8, a=p, b=p, c=p, n=2, st=p, pl=pl, npl=2)
        a.update(kw)
        return L.qkv_pages_reorder(a["t"], a["ns"], a["mb"], a["bl"], a["r"], a["np"], a["a"], a["b"], a["c"], a["n"], a["st"],
                                   a["pl"], a["npl"], None)
    assert f(n=0) == f(n=0, pl=None, npl=0) == OK
    _each(f, INVALID, n=[-1, 2001], ns=[0], mb=[0], bl=[0], np=[0], npl=[-1])
    _each(f, UNSUPPORTED, n=[1025], npl=[129])
    _each(f, NULL, t=[None], r=[None], a=[None], b=[None], c=[None], pl=[None])
    _each(f, ALIGN, t=[p + 2], r=[p + 1], a=[p + 2], b=[p + 2], c=[p + 1], st=[p + 2])
    bad = (kvcache._Plane * 1)(kvcache._Plane(p, 0))
    assert f(pl=ctypes.addressof(bad), npl=1) == INVALID
    bad[0] = kvcache._Plane(0, 16)
    assert f(pl=ctypes.addressof(bad), npl=1) == NULL


# ---- the wrappers -------------------------------------------------------------

def test_wrappers_refuse_before_the_launch():
    """Shapes, types and devices, on CPU tensors: every call raises ValueError."""
    x, w = torch.zeros(3, 4, 128, dtype=torch.float16), torch.ones(128)
    t = kvcache.rope_table(64, device="cpu")
    i = torch.zeros(3, dtype=torch.int32)
    pool, exp = torch.zeros(2, 16, 4, 128, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8)
    table, ws = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(64, dtype=torch.uint8)
    planes = kvcache.f8_weights(2, 16, 4, "cpu")
    assert planes.shape == (2, 4, 16) and planes.dtype is torch.float32 and not planes.any()
    logits, scores = torch.zeros(6, 50), torch.zeros(3, 2)
    out = [torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4)]
    bad = [
        lambda: kvcache.norm_rope(None, None, w, w, i, t),
        lambda: kvcache.norm_rope(None, x, w, w, i, t, q_out=x),
        lambda: kvcache.norm_rope(x, x[:2], w, w, i, t),
        lambda: kvcache.norm_rope(x[0], None, w, None, i, t),
        lambda: kvcache.norm_rope(x, None, w, None, i, t),                   # not on a device
        lambda: kvcache.norm_rope_grad(None, None, None, None, w, w, i, t),
        lambda: kvcache.norm_rope_grad(x, None, None, None, w, None, i, t),
        lambda: kvcache.weigh_f8_paged(x, pool, exp, planes, ws, table, i, i, max_tok=1, max_ctx=10, scale=1.0),
        lambda: kvcache.evict_f8_paged(pool, pool, exp, exp, planes, table, i, i, table, ws, max_ctx=10),
        lambda: kvcache.beam_select(logits, scores, *out, ws),
        lambda: kvcache.pages_reorder(table, i, i, i, i, block_tokens=16),
        lambda: kvcache.norm_rope_grad_workspace(4, 0, 0, 128, "cpu"),
        lambda: kvcache.norm_rope_grad_workspace(4, 4, 2, 2048, "cpu"),
        lambda: kvcache.weigh_f8_paged_workspace(8, 3, 2, 4, 2, 100, "cpu"),
        lambda: kvcache.weigh_f8_paged_workspace(8, 2, 2, 4, 2, 100, "cpu", head_dim=64),
        lambda: kvcache.evict_f8_paged_workspace(2, 2, 16, -1, 50, "cpu"),
        lambda: kvcache.beam_select_workspace(3, 65, 1000, 8, "cpu"),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    assert kvcache.weigh_f8_paged_workspace(8, 2, 0, 4, 2, 100, "cpu").numel() == 0
    assert kvcache.evict_f8_paged_workspace(0, 2, 16, 100, 50, "cpu").numel() == 0
    assert kvcache.beam_select_workspace(0, 4, 1000, 8, "cpu").numel() == 0


# ---- the references -----------------------------------------------------------

@pytest.mark.parametrize("layout,rot", [("half", 16), ("interleaved", 8), ("half", 0)])
def test_norm_gradient_is_the_differences(layout, rot):
    """The formula's gradient against central differences of the forward formula in 64 bits: their error is h^2 of the
    third derivative and 2^-52 / h of the values, 1e-8 of the values' size at h = 1e-5."""
    rng = np.random.default_rng(rot)
    x, dy, w = rng.standard_normal((3, 2, 16)), rng.standard_normal((3, 2, 16)), rng.standard_normal(16)
    pos = np.array([0, 7, 100])
    f = lambda x, w: (R.norm_rope(x, w, pos, rot, layout, eps=1e-3)[0] * dy).sum()
    dx, _, dw, _ = R.norm_rope_grad(x, dy, w, pos, rot, layout, eps=1e-3)
    h = 1e-5
    for a, g, at in ((x, dx, (1, 0, 3)), (x, dx, (2, 1, 15)), (x, dx, (0, 0, 0)), (w, dw, (4,)), (w, dw, (12,))):
        up, down = a.copy(), a.copy()
        up[at] += h
        down[at] -= h
        d = (f(up, w) - f(down, w) if a is x else f(x, up) - f(x, down)) / (2 * h)
        assert abs(d - g[at]) <= 1e-8 * 100


def test_beam_reference_is_a_search():
    """The selection's reference against a plain sort of log-softmax scores."""
    rng = np.random.default_rng(0)
    logits, scores = rng.standard_normal((6, 30)), rng.standard_normal((2, 3)).astype(np.float32)
    lp = torch.log_softmax(torch.from_numpy(logits), -1).numpy().reshape(2, 3, 30) + scores[:, :, None]
    assert np.allclose(R.beam_scores(logits, scores)[0].reshape(lp.shape), lp, rtol=0, atol=1e-12)


def test_weighing_reference_is_a_softmax():
    """Weights of keys against torch's softmax over a slot's dense keys, summed."""
    rng = np.random.default_rng(1)
    kp, ke = rng.integers(0, 100, (3, 16, 2, 128)).astype(np.uint8), np.full((3, 2), 121, np.uint8)
    q = rng.standard_normal((5, 4, 128)).astype(np.float16)
    out, _ = R.weigh(q, kp, ke, np.zeros((3, 2, 16), np.float32), np.array([[2, 0, 1]], np.int32), [0, 5], [30], 0.05)
    k = R.R.CODES[kp[[2, 0, 1]].reshape(48, 2, 128)[:35]] * 2.0 ** -6
    for h in range(2):
        s = torch.from_numpy(np.einsum("rgd,kd->rgk", q[:, 2 * h:2 * h + 2].astype(np.float64), k[:, h]) * 0.05)
        mask = torch.arange(35)[None, None] > torch.arange(30, 35)[:, None, None]
        want = torch.softmax(s.masked_fill(mask, -torch.inf), -1).sum((0, 1)).numpy()
        got = out[[2, 0, 1], h].reshape(48)
        assert np.allclose(got[:35], want, rtol=1e-12, atol=1e-14) and not got[35:].any()
