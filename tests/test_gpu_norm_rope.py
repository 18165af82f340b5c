"""Norms of heads with the rotation, and their gradient, against the 64-bit formulas: layouts, part of the head,
strides, odd sizes, extreme rows, places, empty calls, differences, graphs and streams."""
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


def _np(t):
    return t.cpu().numpy().astype(np.float64)


def _case(tokens, heads, hd, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((tokens, heads, hd)) * np.exp(rng.standard_normal((tokens, heads, 1)))
    return (rng, x.astype(np.float16), (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32),
            rng.integers(0, 50000, tokens).astype(np.int32))


SIZES = [(1, 16, 256, 64), (3, 5, 128, 128), (257, 4, 256, 256), (2, 1, 64, 16), (33, 3, 64, 32), (700, 20, 128, 96),
         (7, 3, 80, 10), (5, 2, 66, 66), (9, 1, 33, 2), (4, 4, 256, 200), (3, 2, 512, 128), (2, 3, 1024, 1024), (6, 2, 1, 0),
         (11, 7, 128, 0), (5, 3, 1000, 400), (9, 5, 96, 32)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,hd,rot", SIZES)
def test_against_the_formula(layout, tokens, heads, hd, rot):
    rng, x, w, pos = _case(tokens, heads, hd, tokens * 1000 + hd + rot)
    t = kvcache.rope_table(rot, device=DEV) if rot else None
    out = torch.empty(x.shape, dtype=torch.float16, device=DEV)
    kvcache.norm_rope(_t(x), None, _t(w), None, _t(pos), t, layout=layout, q_out=out)
    ref, tol = L.norm_rope(x, w, pos, rot, layout)
    assert (np.abs(_np(out) - ref) <= tol).all()
    kvcache.norm_rope(None, _t(x), None, None, _t(pos), t, layout=layout, k_out=out, eps=0.25)   # k alone, no weight
    ref, tol = L.norm_rope(x, np.ones(hd), pos, rot, layout, eps=0.25)
    assert (np.abs(_np(out) - ref) <= tol).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,hd,rot", SIZES)
def test_gradient_against_the_formula(layout, tokens, heads, hd, rot):
    rng, x, w, pos = _case(tokens, heads, hd, tokens * 1000 + hd + rot + 1)
    dy = rng.standard_normal(x.shape).astype(np.float16)
    t = kvcache.rope_table(rot, scaling=("yarn", 4.0, 2048), device=DEV) if rot else None
    dx, dw = torch.empty(x.shape, dtype=torch.float16, device=DEV), torch.empty(hd, device=DEV)
    kvcache.norm_rope_grad(_t(x), None, _t(dy), None, _t(w), None, _t(pos), t, dw, layout=layout, q_grad=dx)
    ref, tol, rw, tw = L.norm_rope_grad(x, dy, w, pos, rot, layout, scaling=("yarn", 4.0, 2048) if rot else None)
    assert (np.abs(_np(dx) - ref) <= tol).all()
    assert (np.abs(_np(dw) - rw) <= tw).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_against_differences(layout):
    """d/dx and d/dw of sum(c * norm_rope(x)), the 64-bit formula's central differences (step 1e-5: truncation below
    1e-9, rounding below 1e-8)."""
    rng, x, w, pos = _case(5, 3, 64, 17)
    c = rng.standard_normal(x.shape).astype(np.float16)
    dx, dw = torch.empty(x.shape, dtype=torch.float16, device=DEV), torch.empty(64, device=DEV)
    kvcache.norm_rope_grad(_t(x), None, _t(c), None, _t(w), None, _t(pos), kvcache.rope_table(48, device=DEV), dw,
                           layout=layout, q_grad=dx)
    _, tol, _, tw = L.norm_rope_grad(x, c, w, pos, 48, layout)

    def f(a, b):
        return (c.astype(np.float64) * L.norm_rope(a, b, pos, 48, layout)[0]).sum()
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    for _ in range(60):
        i = tuple(rng.integers(0, n) for n in x.shape)
        d = np.zeros(x.shape)
        d[i] = 1e-5
        assert abs((f(x64 + d, w64) - f(x64 - d, w64)) / 2e-5 - _np(dx)[i]) <= tol[i] + 1e-7
    for i in range(64):
        d = np.zeros(64)
        d[i] = 1e-5
        assert abs((f(x64, w64 + d) - f(x64, w64 - d)) / 2e-5 - _np(dw)[i]) <= tw[i] + 1e-7


@pytest.mark.parametrize("hd,rot", [(256, 64), (128, 128), (48, 30)])
def test_strided_views_places_and_q_with_k(hd, rot):
    """q and k as views of one projection buffer, in place and apart: the same bits, and v untouched."""
    rng = np.random.default_rng(hd)
    buf = _t(rng.standard_normal((37, 6 + 2 + 2, hd)).astype(np.float16))
    pos = torch.arange(37, dtype=torch.int32, device=DEV) * 11
    wq, wk = torch.rand(hd, device=DEV) + 0.5, torch.rand(hd, device=DEV) + 0.5
    t = kvcache.rope_table(rot, device=DEV)
    before = buf.clone()
    q, k = buf[:, :6], buf[:, 6:8]
    qo = torch.empty(37, 6, hd, dtype=torch.float16, device=DEV)
    ko = torch.full((37, 3, hd), 7.0, dtype=torch.float16, device=DEV)
    kvcache.norm_rope(q, k, wq, wk, pos, t, q_out=qo, k_out=ko[:, :2])
    assert torch.equal(buf, before) and (ko[:, 2] == 7).all()
    only = torch.empty_like(qo)
    kvcache.norm_rope(q, None, wq, None, pos, t, q_out=only)
    assert torch.equal(only, qo)
    # gradients: apart, in place of the outputs' and in place of the rows
    dq, dk = torch.randn(37, 6, hd, device=DEV).half(), torch.randn(37, 2, hd, device=DEV).half()
    gq, gk, dwq, dwk = torch.empty_like(dq), torch.empty_like(dk), torch.empty(hd, device=DEV), torch.empty(hd, device=DEV)
    ws = kvcache.norm_rope_grad_workspace(37, 6, 2, hd, DEV)
    kvcache.norm_rope_grad(q, k, dq, dk, wq, wk, pos, t, dwq, dwk, q_grad=gq, k_grad=gk, workspace=ws)
    assert torch.equal(buf, before)
    in_q, in_k, w2 = dq.clone(), dk.clone(), torch.empty(hd, device=DEV)
    kvcache.norm_rope_grad(q, k, in_q, in_k, wq, wk, pos, t, w2, None)
    assert torch.equal(in_q, gq) and torch.equal(in_k, gk) and torch.equal(w2, dwq)
    own = buf.clone()
    kvcache.norm_rope_grad(own[:, :6], own[:, 6:8], dq, dk, wq, wk, pos, t, q_grad=own[:, :6], k_grad=own[:, 6:8])
    assert torch.equal(own[:, :6], gq) and torch.equal(own[:, 6:8], gk) and torch.equal(own[:, 8:], before[:, 8:])
    kvcache.norm_rope(q, k, wq, wk, pos, t)   # in place
    assert torch.equal(buf[:, :6], qo) and torch.equal(buf[:, 6:8], ko[:, :2]) and torch.equal(buf[:, 8:], before[:, 8:])


def test_far_and_negative_positions():
    """Far and negative positions turn as rope turns them: rows of +-2 are normed to +-1."""
    x = np.sign(np.random.default_rng(4).standard_normal((9, 2, 128))).astype(np.float16) * np.float16(2)
    pos = np.array([0, 1, -1, 1 << 20, 999_999_937, -999_999_937, 2**31 - 1, -2**31 + 1, -2**31], np.int32)
    t = kvcache.rope_table(128, base=500000.0, device=DEV)
    out, turned = torch.empty(x.shape, dtype=torch.float16, device=DEV), torch.empty(x.shape, dtype=torch.float16, device=DEV)
    kvcache.norm_rope(_t(x), None, None, None, _t(pos), t, q_out=out, eps=1e-30)
    kvcache.rope(_t(x / 2), None, _t(pos), t, q_out=turned)
    # the norm's scale is off by _scale_error(128), then both round once
    lim = 2 * 2.0 ** -11 * 1.5 + L._scale_error(128) * 2
    assert (out.float() - turned.float()).abs().max().item() <= lim


def test_extreme_rows():
    """Zeros, the largest and the smallest fp16 numbers; a row with an infinity or NaN is not finite and leaves the
    others alone."""
    x = np.zeros((6, 1, 256), np.float16)
    x[1] = 65504
    x[2] = 2.0 ** -24
    x[3, 0, 5] = np.inf
    x[4, 0, 9] = np.nan
    x[5] = 1
    pos = np.arange(6).astype(np.int32)
    for hd, rot in ((256, 64), (250, 64)):
        t = kvcache.rope_table(rot, device=DEV)
        a = np.ascontiguousarray(x[..., :hd])
        out = torch.empty(a.shape, dtype=torch.float16, device=DEV)
        kvcache.norm_rope(_t(a), None, None, None, _t(pos), t, q_out=out)
        ref, tol = L.norm_rope(a, np.ones(hd), pos, rot, "half")
        got = _np(out)
        for i in (0, 1, 2, 5):
            assert (np.abs(got[i] - ref[i]) <= tol[i]).all()
        assert np.isnan(got[3]).any() and np.isnan(got[4]).all()


def test_empty_calls():
    t = kvcache.rope_table(32, device=DEV)
    e = torch.empty(0, 4, 64, dtype=torch.float16, device=DEV)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    kvcache.norm_rope(e, None, None, None, none, t)
    dw = torch.full((64,), 3.0, device=DEV)
    kvcache.norm_rope_grad(e, None, e.clone(), None, None, None, none, t, dw)
    assert (dw == 0).all()   # (a sum of nothing)


def test_unaligned_rows_give_the_formula_too():
    rng, x, w, pos = _case(3, 2, 64, 5)
    flat = torch.zeros(3 * 2 * 64 + 1, dtype=torch.float16, device=DEV)
    flat[1:] = _t(x).flatten()
    t = kvcache.rope_table(32, device=DEV)
    out = torch.empty(x.shape, dtype=torch.float16, device=DEV)
    kvcache.norm_rope(flat[1:].view(3, 2, 64), None, _t(w), None, _t(pos), t, q_out=out)
    ref, tol = L.norm_rope(x, w, pos, 32, "half")
    assert (np.abs(_np(out) - ref) <= tol).all()


def test_the_gradients_sums_do_not_change():
    rng, x, w, pos = _case(900, 5, 128, 6)
    dy = _t(rng.standard_normal(x.shape).astype(np.float16))
    t = kvcache.rope_table(128, device=DEV)
    sums = []
    for _ in range(4):
        dw, dx = torch.empty(128, device=DEV), torch.empty_like(dy)
        kvcache.norm_rope_grad(_t(x), None, dy, None, _t(w), None, _t(pos), t, dw, q_grad=dx)
        sums.append(dw)
    assert all(torch.equal(s, sums[0]) for s in sums)


def test_captured_and_replayed_and_on_a_stream():
    rng, x, w, pos = _case(40, 6, 128, 7)
    q, wq, ps, dy = _t(x), _t(w), _t(pos), torch.randn(40, 6, 128, device=DEV).half()
    t = kvcache.rope_table(64, device=DEV)
    out, dx, dw = torch.empty_like(q), torch.empty_like(q), torch.empty(128, device=DEV)
    ws = kvcache.norm_rope_grad_workspace(40, 6, 0, 128, DEV)

    def both(stream=None):
        kvcache.norm_rope(q, None, wq, None, ps, t, q_out=out, stream=stream)
        kvcache.norm_rope_grad(q, None, dy, None, wq, None, ps, t, dw, q_grad=dx, workspace=ws, stream=stream)
    both()
    torch.cuda.synchronize()
    want = [a.clone() for a in (out, dx, dw)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        both()
    for i in range(4):
        for a in (out, dx, dw):
            a.fill_(9)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, dx, dw), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for a in (out, dx, dw):
        a.fill_(9)
    s.wait_stream(torch.cuda.current_stream())
    both(s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((out, dx, dw), want))


def test_more_than_four_billion_bytes_of_rows():
    """Tokens whose offsets pass 32 bits (2.4e9 elements): first, middle and last as in calls of their own."""
    n, heads, hd = 150000, 64, 256
    x = torch.randn(64, heads, hd, device=DEV).half().repeat(n // 64 + 1, 1, 1)[:n]
    w = torch.rand(hd, device=DEV) + 0.5
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    t = kvcache.rope_table(64, device=DEV)
    small = [(a, torch.empty(64, heads, hd, dtype=torch.float16, device=DEV)) for a in (0, n // 2, n - 64)]
    for a, o in small:
        kvcache.norm_rope(x[a:a + 64], None, w, None, pos[a:a + 64], t, q_out=o)
    kvcache.norm_rope(x, None, w, None, pos, t)
    for a, o in small:
        assert torch.equal(x[a:a + 64], o)
