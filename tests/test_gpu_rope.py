"""Rotary positions against the 64-bit formula: layouts, part of the head, strides, odd
sizes, far and negative positions, scaling, and the inverse as the gradient."""
import numpy as np
import pytest
import torch

from qengine_amd import kvcache
from tests import _paged8 as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _run(x, pos, table, **kw):
    out = torch.empty_like(x, memory_format=torch.contiguous_format)
    kvcache.rope(x, None, pos, table, q_out=out, **kw)
    return out


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,hd,rot", [
    (1, 16, 256, 64), (3, 5, 128, 128), (257, 4, 256, 256), (2, 1, 16, 16), (33, 3, 64, 32), (1000, 28, 128, 96),
    (7, 3, 80, 10), (5, 2, 66, 66), (9, 1, 33, 2), (4, 4, 256, 200)])
def test_against_the_formula(layout, tokens, heads, hd, rot):
    rng = np.random.default_rng(tokens * 1000 + hd + rot)
    x = rng.standard_normal((tokens, heads, hd)).astype(np.float16)
    pos = rng.integers(0, 5000, tokens).astype(np.int32)
    t = kvcache.rope_table(rot, device=DEV)
    for inverse in (False, True):
        got = _run(torch.from_numpy(x).to(DEV), torch.from_numpy(pos).to(DEV), t, layout=layout, inverse=inverse)
        ref = R.rotate(x, pos, rot, layout, inverse)
        err = np.abs(got.cpu().numpy().astype(np.float64) - ref)
        assert (err <= R.rope_tolerance(x, ref, rot, layout)).all(), err.max()
        assert np.array_equal(got.cpu().numpy()[..., rot:], x[..., rot:])


@pytest.mark.parametrize("scaling", [None, ("linear", 8.0), ("ntk", 4.0), ("yarn", 16.0, 8192),
                                     ("yarn", 4.0, 32768, 24.0, 2.0)])
def test_far_and_negative_positions(scaling):
    """Angles of positions up to 2^31: fp32 products would be off by radians."""
    rng = np.random.default_rng(3)
    pos = np.array([0, 1, -1, 1 << 20, (1 << 20) + 1, 999_999_937, -999_999_937, 2**31 - 1, -2**31 + 1], np.int32)
    x = rng.standard_normal((len(pos), 2, 128)).astype(np.float16)
    t = kvcache.rope_table(128, base=500000.0, scaling=scaling, device=DEV)
    _, amp = R.frequencies(128, 500000.0, scaling)
    got = _run(torch.from_numpy(x).to(DEV), torch.from_numpy(pos).to(DEV), t).cpu().numpy().astype(np.float64)
    ref = R.rotate(x, pos, 128, "half", base=500000.0, scaling=scaling)
    # the 64-bit reference's own angles are off by position * 2^-52 radians
    extra = np.abs(pos.astype(np.float64))[:, None, None] * 2.0 ** -51 * np.abs(x).max() * 2 * amp
    assert (np.abs(got - ref) <= R.rope_tolerance(x, ref, 128, "half", amp) + extra).all()


def test_the_lowest_position():
    """-2^31 has no int32 negative: its inverse turns as 2^31 does, one position past 2^31 - 1."""
    rng = np.random.default_rng(8)
    for hd in (128, 66):   # (each kernel)
        x = rng.standard_normal((1, 2, hd)).astype(np.float16)
        t = kvcache.rope_table(hd, base=500000.0, device=DEV)
        got = _run(torch.from_numpy(x).to(DEV), torch.tensor([-2**31], dtype=torch.int32, device=DEV), t, inverse=True)
        ref = R.rotate(x, np.array([2**31]), hd, "half", base=500000.0)
        extra = 2.0 ** 31 * 2.0 ** -51 * np.abs(x).max() * 2
        assert (np.abs(got.cpu().numpy().astype(np.float64) - ref) <= R.rope_tolerance(x, ref, hd, "half") + extra).all()


@pytest.mark.parametrize("hd,rot", [(256, 64), (128, 128), (48, 30)])
def test_strided_views_in_place_and_q_with_k(hd, rot):
    """q and k as views of one projection buffer, in place and apart: the same bits, and v untouched."""
    rng = np.random.default_rng(hd)
    buf = torch.from_numpy(rng.standard_normal((37, 6 + 2 + 2, hd)).astype(np.float16)).to(DEV)
    pos = torch.arange(37, dtype=torch.int32, device=DEV) * 11
    t = kvcache.rope_table(rot, device=DEV)
    q, k = buf[:, :6], buf[:, 6:8]
    qo = torch.empty(37, 6, hd, dtype=torch.float16, device=DEV)
    ko = torch.full((37, 3, hd), 7.0, dtype=torch.float16, device=DEV)
    kvcache.rope(q, k, pos, t, q_out=qo, k_out=ko[:, :2])
    before = buf.clone()
    assert torch.equal(buf, before) and (ko[:, 2] == 7).all()
    only = torch.empty_like(qo)
    kvcache.rope(q, None, pos, t, q_out=only)
    assert torch.equal(only, qo)
    kvcache.rope(q, k, pos, t, k_out=None, q_out=None)   # in place
    assert torch.equal(buf[:, :6], qo) and torch.equal(buf[:, 6:8], ko[:, :2])
    assert torch.equal(buf[:, 8:], before[:, 8:])
    kvcache.rope(None, before[:, 6:8], pos, t)   # k alone
    assert torch.equal(before[:, 6:8], buf[:, 6:8])


def test_empty_and_unaligned():
    t = kvcache.rope_table(32, device=DEV)
    kvcache.rope(torch.empty(0, 4, 64, dtype=torch.float16, device=DEV), None,
                 torch.empty(0, dtype=torch.int32, device=DEV), t)
    rng = np.random.default_rng(5)
    flat = torch.from_numpy(rng.standard_normal(3 * 2 * 64 + 1).astype(np.float16)).to(DEV)
    x = flat[1:].view(3, 2, 64)   # 2-byte aligned
    pos = torch.tensor([4, 5, 6], dtype=torch.int32, device=DEV)
    a, b = _run(x, pos, t), _run(x.clone(), pos, t)
    assert torch.equal(a, b)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_inverse_is_the_gradient(layout):
    """sum(w * rope(x)) differentiated by x: the inverse of w, against the formula's differences."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((6, 2, 64))
    w = rng.standard_normal((6, 2, 64)).astype(np.float16)
    pos = np.array([0, 3, 100, 77777, 5, 9], np.int32)
    scaling = ("yarn", 4.0, 2048)
    t = kvcache.rope_table(48, scaling=scaling, device=DEV)
    got = _run(torch.from_numpy(w).to(DEV), torch.from_numpy(pos).to(DEV), t, layout=layout,
               inverse=True).cpu().numpy().astype(np.float64)
    f = lambda y: (w.astype(np.float64) * R.rotate(y, pos, 48, layout, scaling=scaling)).sum()  # noqa: E731
    _, amp = R.frequencies(48, scaling=scaling)
    ref = R.rotate(w, pos, 48, layout, True, scaling=scaling)
    assert (np.abs(got - ref) <= R.rope_tolerance(w, ref, 48, layout, amp)).all()
    for _ in range(40):
        i = tuple(rng.integers(0, n) for n in x.shape)
        d = np.zeros_like(x)
        d[i] = 1.0   # (f is linear: the difference is the derivative, up to 64-bit rounding)
        assert abs((f(x + d) - f(x)) - ref[i]) < 1e-9


def test_undoes_itself_and_moves_cached_keys():
    """Turning by p then back gives the rows; turning rows at p on by d is turning by p + d."""
    rng = np.random.default_rng(9)
    x = torch.from_numpy(rng.standard_normal((50, 4, 128)).astype(np.float16)).to(DEV)
    pos = torch.randint(0, 10000, (50,), dtype=torch.int32, device=DEV)
    d = torch.full((50,), -321, dtype=torch.int32, device=DEV)
    t = kvcache.rope_table(128, device=DEV)
    y = _run(x, pos, t)
    back = _run(y, pos, t, inverse=True)
    # two roundings to fp16, each 2^-11 of a pair's length, which is at most sqrt(2) * |max|
    lim = 2 * 2.0 ** -11 * 1.5 * x.abs().max().item() + 1e-5
    assert (back.float() - x.float()).abs().max().item() <= lim
    assert (_run(y, d, t).float() - _run(x, pos + d, t).float()).abs().max().item() <= lim


def test_more_than_four_billion_threads():
    """A call of 2^32 elements and more (9 GB, rows that the wide kernel does not take): first, middle and last
    tokens as in calls of their own."""
    n, heads, hd = 70000, 64, 1001
    x = torch.randn(64, heads, hd, device=DEV).half().repeat(n // 64 + 1, 1, 1)[:n]
    out = torch.zeros_like(x)
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    t = kvcache.rope_table(2, device=DEV)
    kvcache.rope(x, None, pos, t, q_out=out)
    for a in (0, n // 2, n - 4000, n - 64):
        assert torch.equal(out[a:a + 64], _run(x[a:a + 64], pos[a:a + 64], t))


@pytest.mark.parametrize("hd,rot", [(256, 64), (128, 128), (48, 30)])
def test_a_rotation_apart_leaves_its_input(hd, rot):
    """q, k and v of one projection buffer are as they were after q and k are rotated into buffers of their own."""
    rng = np.random.default_rng(hd + rot)
    buf = torch.from_numpy(rng.standard_normal((37, 6 + 2 + 2, hd)).astype(np.float16)).to(DEV)
    before = buf.clone()
    qo, ko = torch.empty(37, 6, hd, dtype=torch.float16, device=DEV), torch.empty(37, 2, hd, dtype=torch.float16, device=DEV)
    kvcache.rope(buf[:, :6], buf[:, 6:8], torch.arange(37, dtype=torch.int32, device=DEV) * 11,
                 kvcache.rope_table(rot, device=DEV), q_out=qo, k_out=ko)
    assert torch.equal(buf, before)
    assert not torch.equal(qo, before[:, :6]) and torch.equal(ko[..., rot:], before[:, 6:8, rot:])
