"""Refusals of the rotary, paged 8-bit and page calls before anything is launched, the host
side of the rotary table, and the references that the GPU tests use against each other."""
import ctypes

import numpy as np
import pytest
import torch

from qengine_amd import _lib, kvcache
from tests import _paged8 as R


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(1 << 16)
    test_buf.append(buf)
    return (ctypes.addressof(buf) + 255) & ~255


test_buf = []


# ---- rotary table ----------------------------------------------------------

def _table(L, rot, base=10000.0, kind=0, args=(1.0, 1.0, 32.0, 1.0)):
    turns, amp = (ctypes.c_uint64 * max(1, rot // 2))(), ctypes.c_float()
    st = L.qkv_rope_table(rot, base, kind, *args, ctypes.addressof(turns), ctypes.addressof(amp))
    return st, np.array(turns[:], dtype=object), amp.value


@pytest.mark.parametrize("rot", [2, 10, 64, 128, 256])
@pytest.mark.parametrize("scaling", [None, ("linear", 3.0), ("ntk", 4.0), ("yarn", 8.0, 4096), ("yarn", 2.0, 100, 20.0, 2.0)])
def test_rope_table_is_the_formula(L, rot, scaling):
    if scaling and scaling[0] == "ntk" and rot < 4:
        return
    t = kvcache.rope_table(rot, base=123456.0, scaling=scaling, device="cpu")
    f, amp = R.frequencies(rot, 123456.0, scaling)
    got = np.array([int(x) % 2 ** 64 for x in t.turns.tolist()], dtype=np.float64) / 2.0 ** 64
    # the 64-bit formula's own error, a few roundings of 2^-53, and the fixed point's rounding:
    # half of its unit of 2^-64
    assert np.all(np.abs(got - f / (2 * np.pi)) <= f / (2 * np.pi) * 64 * 2.0 ** -53 + 2.0 ** -65)
    assert abs(t.amplitude - amp) <= 2.0 ** -23 * amp and t.rot_dim == rot


def test_a_table_from_a_models_own_frequencies():
    """Made by hand from 64-bit frequencies, the table is rope_table's to the rounding of those: f by 4 of 2^-53
    (the power, the division and the two products), and half a unit."""
    f, amp = R.frequencies(128, 1e6)
    t = kvcache.RopeTable(torch.tensor([round(x / (2 * np.pi) * 2.0 ** 64) for x in f]), 1.25, 128)
    want = kvcache.rope_table(128, base=1e6, device="cpu")
    err = np.abs(np.array([int(a) - int(b) for a, b in zip(t.turns, want.turns)], np.float64)) / 2.0 ** 64
    # (the exponent of the power is rounded too: 2^-53 of ln f, at most 14)
    assert (err <= f / (2 * np.pi) * (4 + 14) * 2.0 ** -53 + 2.0 ** -64).all()
    assert t.amplitude == 1.25 and t.rot_dim == 128 and t.turns.dtype is torch.int64


def test_rope_table_refusals(L):
    assert _table(L, 64)[0] == 0
    assert _table(L, 0)[0] == _table(L, 7)[0] == _table(L, -2)[0] == -1
    assert _table(L, 64, base=0.0)[0] == _table(L, 64, base=float("nan"))[0] == -1
    assert _table(L, 64, kind=4)[0] == _table(L, 64, kind=-1)[0] == -1
    assert _table(L, 64, kind=1, args=(0.5, 1, 1, 1))[0] == _table(L, 2, kind=2, args=(2.0, 1, 1, 1))[0] == -1
    assert _table(L, 64, kind=3, args=(2.0, 0.0, 32.0, 1.0))[0] == -1
    assert _table(L, 64, kind=3, args=(2.0, 100.0, 1.0, 1.0))[0] == -1
    assert L.qkv_rope_table(64, 10000.0, 0, 1.0, 1.0, 1.0, 0.0, None, None) == -2
    for bad in (("cubic", 2.0), ("linear",), ("yarn", 2.0), ("linear", 2.0, 3.0)):
        with pytest.raises(ValueError):
            kvcache.rope_table(64, scaling=bad, device="cpu")
    t = kvcache.rope_table(64, device="cpu")
    for turns in (t.turns[:31], t.turns.double()):   # (the kernels read rot_dim / 2 of them)
        with pytest.raises(ValueError):
            kvcache.RopeTable(turns, 1.0, 64)


# ---- the C entry points -----------------------------------------------------

def test_rope_refusals(L, p):
    def f(**kw):
        a = dict(q=p, qs=512, qo=p, qos=512, k=p + 64, ks=256, ko=p + 64, kos=256, pos=p, t=p, n=4, nq=4, nk=2, hd=128, rot=64,
                 lay=0)
        a.update(kw)
        return L.qkv_rope(a["q"], a["qs"], a["qo"], a["qos"], a["k"], a["ks"], a["ko"], a["kos"], a["pos"], a["t"], 1.0,
                          a["n"], a["nq"], a["nk"], a["hd"], a["rot"], a["lay"], 0, None)
    assert f(n=0) == 0
    assert f(n=-1) == f(nq=0, nk=0) == f(nq=-1) == f(rot=0) == f(rot=63) == f(rot=130) == f(lay=2) == f(hd=0) == -1
    assert f(qs=500) == f(ks=100) == -1            # strides shorter than a token's heads
    assert f(qos=1024) == -1                       # in place with another stride
    assert f(k=p, ko=p) == f(ko=p) == -1           # one memory for both outputs
    assert f(q=None) == f(qo=None) == f(k=None) == f(pos=None) == f(t=None) == -2
    assert f(q=p + 1, qo=p + 1) == f(pos=p + 2) == f(t=p + 4) == -4
    assert f(nq=2000) == -1


def test_append_refusals(L, p):
    def f(**kw):
        a = dict(k=p, ks=512, v=p, vs=512, kp=p, vp=p, ke=p, ve=p, rows=4, slots=2, mt=2, kv=4, hd=128, bt=p, mb=4, bl=16,
                 np=8, st=p, pos=p, q=None, qs=0, qo=None, qos=0, nq=0, t=None, rot=0, lay=0)
        a.update(kw)
        return L.qkv_f8_append_kv_paged(a["k"], a["ks"], a["v"], a["vs"], a["kp"], a["vp"], a["ke"], a["ve"], a["rows"],
                                        a["slots"], a["mt"], a["kv"], a["hd"], a["bt"], a["mb"], a["bl"], a["np"],
                                        a["st"], a["pos"], a["q"], a["qs"], a["qo"], a["qos"], a["nq"], a["t"], 1.0,
                                        a["rot"], a["lay"], None)
    assert f(rows=0) == f(slots=0) == f(mt=0) == 0
    assert f(rows=-1) == f(slots=-1) == f(mt=-1) == f(kv=0) == f(mb=0) == f(bl=0) == f(np=0) == -1
    assert f(hd=64) == f(bl=24) == f(rot=40) == -3
    assert f(bl=1 << 22) == f(kv=1 << 20) == f(bl=0x7ffffff0, kv=0x7fffffff) == -3   # pages of 2 GiB and more
    assert f(rot=-16) == f(rot=256) == f(lay=3) == f(nq=4) == -1    # (queries without a rotation)
    assert f(k=None) == f(v=None) == f(kp=None) == f(ve=None) == f(bt=None) == f(st=None) == f(pos=None) == -2
    assert f(rot=64) == -2 and f(rot=64, t=p, nq=4) == -2           # no table; no queries
    assert f(ks=256) == f(rot=64, t=p, nq=4, q=p, qs=256, qo=p, qos=256) == -1
    assert f(k=p + 8) == f(ks=516) == f(kp=p + 8) == f(st=p + 2) == f(rot=64, t=p + 4) == -4


def test_attention_refusals(L, p):
    ws = L.qkv_attn_f8_paged_workspace_bytes(8, 2, 128, 2, 4, 2, 100)
    assert ws > 0

    def f(**kw):
        a = dict(q=p, kp=p, vp=p, ke=p, ve=p, out=p, rows=4, nq=8, kv=2, hd=128, slots=2, mt=2, mc=100, bt=p, mb=8, bl=16,
                 np=8, st=p, pos=p, w=0, s=0, ws=p, wb=ws)
        a.update(kw)
        return L.qkv_attn_f8_paged(a["q"], a["kp"], a["vp"], a["ke"], a["ve"], a["out"], a["rows"], a["nq"], a["kv"],
                                   a["hd"], a["slots"], a["mt"], a["mc"], a["bt"], a["mb"], a["bl"], a["np"], a["st"],
                                   a["pos"], 0.1, a["w"], a["s"], a["ws"], a["wb"], None)
    assert f(rows=0) == f(slots=0) == f(mt=0) == 0
    assert f(rows=-1) == f(slots=-1) == f(mt=-1) == f(mc=0) == f(nq=7) == f(kv=0) == f(np=0) == -1
    assert f(nq=18) == f(hd=192) == f(bl=8) == f(mc=(1 << 30) + 1) == -3
    assert f(bl=1 << 23) == f(bl=0x7ffffff0) == -3      # pages of 2 GiB and more
    assert f(w=-1) == f(s=-1) == -1
    assert f(q=None) == f(ke=None) == f(out=None) == f(bt=None) == f(st=None) == -2
    assert f(q=p + 8) == f(vp=p + 4) == f(pos=p + 1) == f(ws=p + 16) == -4
    assert f(wb=ws - 1) == f(ws=None) == -7
    w = L.qkv_attn_f8_paged_workspace_bytes
    assert w(8, 3, 128, 2, 4, 2, 100) == w(8, 2, 64, 2, 4, 2, 100) == w(8, 2, 128, 0, 4, 2, 100) == 0
    # the call with the most rows that the numbers allow never needs more than the query says
    assert w(8, 2, 128, 2, 4, 100, 100) == w(8, 2, 128, 2, 4, 4, 100)


def test_page_refusals(L, p):
    planes = (kvcache._Plane * 2)(kvcache._Plane(p, 64), kvcache._Plane(p + 4096, 3))
    pl = ctypes.addressof(planes)

    def fork(**kw):
        a = dict(t=p, ns=4, mb=8, bl=16, r=p, np=8, a=p, b=p, c=p, n=2, st=p)
        a.update(kw)
        return L.qkv_pages_fork(a["t"], a["ns"], a["mb"], a["bl"], a["r"], a["np"], a["a"], a["b"], a["c"], a["n"], a["st"],
                                None)

    def release(**kw):
        a = dict(t=p, ns=4, mb=8, bl=16, r=p, np=8, a=p, b=p, n=2, st=p)
        a.update(kw)
        return L.qkv_pages_release(a["t"], a["ns"], a["mb"], a["bl"], a["r"], a["np"], a["a"], a["b"], a["n"], a["st"], None)

    def reserve(**kw):
        a = dict(t=p, ns=4, mb=8, bl=16, r=p, np=8, a=p, b=p, c=p, n=2, mn=5, st=p, pl=pl, npl=2, sc=p, sb=4096)
        a.update(kw)
        return L.qkv_pages_reserve(a["t"], a["ns"], a["mb"], a["bl"], a["r"], a["np"], a["a"], a["b"], a["c"], a["n"],
                                   a["mn"], a["st"], a["pl"], a["npl"], a["sc"], a["sb"], None)

    for f in (fork, release, reserve):
        assert f(n=0) == 0
        assert f(n=-1) == f(ns=0) == f(mb=0) == f(bl=0) == f(np=0) == -1
        assert f(t=None) == f(r=None) == f(a=None) == f(b=None) == -2
        assert f(t=p + 2) == f(r=p + 1) == f(a=p + 2) == f(st=p + 2) == -4
    assert fork(n=5) == release(n=5) == -1           # longer than there are slots
    assert reserve(n=1025) == reserve(npl=129) == -3
    assert reserve(mn=0) == 0 and reserve(mn=-1) == -1
    assert reserve(sb=4 * (3 * 2 + 2 * 2 * 2) - 1) == reserve(sc=None) == -7
    assert reserve(pl=None) == -2 and reserve(npl=-1) == -1
    bad = (kvcache._Plane * 1)(kvcache._Plane(p, 0))
    assert reserve(pl=ctypes.addressof(bad), npl=1) == -1
    bad[0] = kvcache._Plane(0, 16)
    assert reserve(pl=ctypes.addressof(bad), npl=1) == -2
    assert L.qkv_pages_copy(pl, 2, 8, p, 0, None) == L.qkv_pages_copy(None, 0, 8, p, 4, None) == 0
    assert L.qkv_pages_copy(pl, 2, 0, p, 1, None) == L.qkv_pages_copy(pl, 2, 8, p, -1, None) == -1
    assert L.qkv_pages_copy(pl, 2, 8, None, 1, None) == -2 and L.qkv_pages_copy(pl, 2, 8, p + 2, 1, None) == -4

    def compact(**kw):
        a = dict(t=p, ns=4, mb=8, r=p, np=8, m=p, u=p, pl=pl, npl=2, sc=p, sb=40)
        a.update(kw)
        return L.qkv_pages_compact(a["t"], a["ns"], a["mb"], a["r"], a["np"], a["m"], a["u"], a["pl"], a["npl"], a["sc"],
                                   a["sb"], None)
    assert compact(np=0) == compact(ns=-1) == -1
    assert compact(m=None) == compact(u=None) == compact(t=None) == -2
    assert compact(sb=39) == compact(sc=None) == -7 and compact(m=p + 2) == -4


# ---- the references ---------------------------------------------------------

def test_e4m3_reference():
    """Codes are torch's of the same type, the nearest with ties to even."""
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(np.nan_to_num(t, nan=9e9), np.nan_to_num(R.CODES, nan=9e9))
    x = np.concatenate([np.random.default_rng(0).standard_normal(20000) * 60, np.linspace(-0.05, 0.05, 4001),
                        (R._POS[1:] + R._POS[:-1]) / 2])
    x = np.clip(x, -448, 448).astype(np.float32)
    assert np.array_equal(R.e4m3_encode(x.astype(np.float64)), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_append_reference_holds_its_rows():
    """Every stored value is within half a step of e4m3 (2^-4 relative, 2^-10 of the exponent's unit below
    its normal range) of its row, over pages that are continued twice."""
    rng = np.random.default_rng(1)
    pool, exp = np.zeros((3, 16, 2, 128), np.uint8), np.zeros((3, 2), np.uint8)
    tables = np.array([[2, 0, 1]], np.int32)
    rows, at = np.zeros((40, 2, 128), np.float16), 0
    for n in (5, 1, 20, 14):
        rows[at:at + n] = rng.standard_normal((n, 2, 128))
        R.append(pool, exp, rows[at:at + n], tables, [0, n], [at])
        at += n
    j = np.arange(40)
    page = tables[0][j // 16]
    unit = 2.0 ** (exp[page].astype(float) - 127)[..., None]
    got = R.CODES[pool[page, j % 16]] * unit
    x = rows.astype(np.float64)
    # (a row requantized once rounds twice: its codes only change below the normal range)
    assert (np.abs(got - x) <= np.abs(x) * 2.0 ** -4 + 2 * unit * 2.0 ** -10).all()


def test_page_references_keep_the_counts():
    rng = np.random.default_rng(2)
    tables, refs = np.full((6, 10), -1, np.int32), np.zeros(60, np.int32)
    lens = [0] * 6
    for step in range(60):
        kind = rng.integers(0, 4)
        if kind == 0:
            n = [int(x) for x in rng.integers(0, 9, 6)]
            n = [min(x, 160 - 16 - a) if a < 140 else 0 for x, a in zip(n, lens)]
            st, _ = R.reserve(tables, refs, list(range(6)), lens, n, 9, 16)
            lens = [a + (b if s == 0 else 0) for a, b, s in zip(lens, n, st)]
        elif kind == 1:
            a, b = rng.permutation(6)[:2]
            R.release(tables, refs, [b], [0], 16)
            assert R.fork(tables, refs, [a], [b], [lens[a]], 16) == [0]
            lens[b] = lens[a]
        elif kind == 2:
            a = int(rng.integers(0, 6))
            lens[a] = int(rng.integers(0, lens[a] + 1))
            R.release(tables, refs, [a], [lens[a]], 16)
        else:
            _, n = R.compact(tables, refs)
            assert (refs[:n] > 0).all() and (refs[n:] == 0).all()
        assert np.array_equal(np.bincount(tables[tables >= 0], minlength=60), refs)
        assert all((tables[s, :-(-lens[s] // 16)] >= 0).all() for s in range(6))


def test_wrappers_refuse_before_the_launch():
    """Shapes, types and devices, on CPU tensors: every call raises ValueError."""
    x = torch.zeros(3, 4, 128, dtype=torch.float16)
    t = kvcache.rope_table(64, device="cpu")
    i = torch.zeros(3, dtype=torch.int32)
    bad = [
        lambda: kvcache.rope(None, None, i, t),
        lambda: kvcache.rope(x.float(), None, i, t),
        lambda: kvcache.rope(x, None, i, t),                       # not on a device
        lambda: kvcache.rope(x, x[:2], i, t),
        lambda: kvcache.rope(x, None, i, t, k_out=x),
        lambda: kvcache.rope(x, None, i, t, layout="both"),
        lambda: kvcache.f8_append_kv_paged(x, x, *[torch.zeros(2, 16, 4, 128)] * 2, *[torch.zeros(2, 4)] * 2,
                                           torch.zeros(3, 4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), i,
                                           max_tok=1),
        lambda: kvcache.page_planes([x]),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def test_scratch_is_of_the_stream_of_the_call(monkeypatch):
    """Scratch that a page call allocates for another stream is allocated with that stream current: memory of
    the current one may still be in use by its work, and the plan in it is trusted."""
    inside, seen = [None], []

    class Within:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            inside.append(self.stream)

        def __exit__(self, *_):
            inside.pop()

    empty = torch.empty
    monkeypatch.setattr(torch.cuda, "stream", Within)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: (seen.append(inside[-1]), empty(*a, **k))[1])

    class Stream:
        pass

    s = Stream()
    assert kvcache._scratch(64, "cpu", s).numel() == 16 and seen == [s]
    assert kvcache._scratch(0, "cpu", None).numel() == 1 and seen == [s, None]


def test_lists_that_one_launch_does_not_hold(L, p):
    """Forks and releases of 2^24 entries and more, 2^32 threads, of which a launch would drop the last."""
    for n in (1 << 24, (1 << 24) + 5, 2**31 - 1):
        assert L.qkv_pages_fork(p, 2**31 - 1, 1, 16, p, 8, p, p, p, n, p, None) == -3
        assert L.qkv_pages_release(p, 2**31 - 1, 1, 16, p, 8, p, p, n, p, None) == -3


def test_workspace_of_calls_that_are_refused():
    """The wrapper refuses numbers that the call refuses, at the stated limits, instead of handing out nothing; a
    batch without rows needs none."""
    def w(nq=16, kv=4, slots=4, rows=64, tok=4, ctx=4096, hd=256):
        return kvcache.attn_f8_paged_workspace(nq, kv, slots, rows, tok, ctx, "cpu", head_dim=hd)
    assert w().numel() > 0
    assert w(slots=0).numel() == w(rows=0).numel() == w(tok=0).numel() == 0
    for bad in (dict(nq=18), dict(nq=36), dict(hd=64), dict(kv=0), dict(ctx=0), dict(ctx=(1 << 30) + 1), dict(nq=2048, kv=1024)):
        with pytest.raises(ValueError, match="no call of these numbers"):
            w(**bad)
    size = kvcache.lib().qkv_attn_f8_paged_workspace_bytes
    # n_slots * (max_tok * gqa / 256 + 1) * num_kv up to 2^22: 2^20 / (1 + 1/64) slots of one token
    for hd in (128, 256):
        last = int((1 << 20) / (1 + 4 / 256))
        assert size(16, 4, hd, last, 1 << 20, 1, 100) > 0 and size(16, 4, hd, last + 1, 1 << 20, 1, 100) == 0
        # tiles * max(num_kv, 2) * (max_ctx / 32 + 16): one prompt of 2^20 rows at GQA 4
        tiles = (1 << 20) * 4 / 256 + 1
        ctx = int((2147483000 / (tiles * 8) - 16) * 32)
        assert size(32, 8, hd, 1, 1 << 20, 1 << 20, ctx - 32) > 0 == size(32, 8, hd, 1, 1 << 20, 1 << 20, ctx + 32)
