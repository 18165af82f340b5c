"""Beam selection against 64-bit scores, and the reordering of slots that follows it."""
import numpy as np
import pytest
import torch

from qengine_amd import kvcache
from tests import _loop as L

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f16": torch.float16, "f32": torch.float32, "bf16": torch.bfloat16}


def _select(logits, scores, take, done=None, end_token=0, ws=None, stream=None):
    n, beams = scores.shape
    p, t = (torch.full((n, take), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    s = torch.full((n, take), 7.0, device=DEV)
    ws = kvcache.beam_select_workspace(n, beams, logits.shape[1], take, DEV) if ws is None else ws
    kvcache.beam_select(logits, scores, p, t, s, ws, done=done, end_token=end_token, stream=stream)
    return p, t, s


def _check(logits, scores, take, done=None, end_token=0, **kw):
    out = _select(logits, scores, take, done, end_token, **kw)
    torch.cuda.synchronize()
    return L.beam_check(logits.float().cpu().numpy(), scores.cpu().numpy(), take, *(o.cpu().numpy() for o in out),
                        None if done is None else done.cpu().numpy(), end_token)


def _inputs(n, beams, vocab, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = 3 * torch.randn(n * beams, vocab, device=DEV, generator=g)
    x[torch.rand(n * beams, vocab, device=DEV, generator=g) < 0.02] = -float("inf")
    return x.to(TYPES[dtype]), -20 * torch.rand(n, beams, device=DEV, generator=g)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,beams,vocab,take", [
    (1, 1, 1, 1), (1, 1, 7, 4), (1, 4, 32003, 8), (3, 2, 63, 64), (2, 5, 1000, 10), (1, 64, 257, 64), (7, 3, 2049, 6),
    (1, 1, 200000, 64), (40, 8, 5003, 16), (2, 12, 50257, 24), (300, 4, 151, 8), (1, 8, 8192, 5)])
def test_against_64_bits(dtype, n, beams, vocab, take):
    x, s = _inputs(n, beams, vocab, dtype, vocab + n)
    assert _check(x, s, take) > 0


@pytest.mark.parametrize("n,beams,vocab,take", [(2100, 1, 40000, 4), (64, 8, 131072, 16)])
def test_large_batches(n, beams, vocab, take):
    """Many rows, whose segments are the longest: checked in 64 bits on the device."""
    x, s = _inputs(n, beams, vocab, "f16", n)
    p, t, top = _select(x, s, take)
    ref = torch.cat([(x[i:i + 8 * beams].double().log_softmax(-1) + s.double().view(-1, 1)[i:i + 8 * beams]).view(-1, beams * vocab)
                     .topk(take, -1).values for i in range(0, n * beams, 8 * beams)])
    assert (top.double() - ref).abs().max().item() <= 40 * 2.0 ** -24 + 60 * 2.0 ** -24 + 5 * 4 * 2.0 ** -24
    got = x[p.long().view(-1), t.long().view(-1)].double().view(n, take)
    lse = x.float().double().logsumexp(-1) if n * beams * vocab < 2 ** 27 else torch.cat([r.double().logsumexp(-1) for r in x.split(64)])
    assert ((got - lse[p.long()] + s.double().view(-1)[p.long()]) - ref).abs().max().item() <= 1e-5
    assert (torch.sort(p.long() * vocab + t, -1).values.diff(dim=-1) > 0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [5, 3000, 70000])
def test_ties_go_to_the_lowest_beam_and_token(dtype, vocab):
    """Equal logits throughout (more ties than a workgroup keeps), and three values in turn."""
    s = torch.zeros(2, 4, device=DEV)
    for x in (torch.zeros(8, vocab, device=DEV), (torch.arange(8 * vocab, device=DEV) % 3).float().view(8, vocab)):
        p, t, top = _select(x.to(TYPES[dtype]), s, 6)
        S, _ = L.beam_scores(x.cpu().numpy(), s.cpu().numpy())
        for r in range(2):
            # rows of one value are the same sums; in the other case beams differ in their sums' last bits
            if (x == 0).all():
                want = np.lexsort((np.arange(S.shape[1]), -S[r]))[:6]
                assert (p[r].cpu().numpy() == r * 4 + want // vocab).all() and (t[r].cpu().numpy() == want % vocab).all()
            else:
                for b in range(4):   # of one beam's, the lowest tokens of its largest value in order
                    mine = t[r][p[r] == r * 4 + b].cpu().numpy()
                    best = np.nonzero((x[r * 4 + b] == 2).cpu().numpy())[0][:len(mine)]
                    assert (mine[:len(best)] == best).all()


def test_rising_and_falling_rows():
    """All of a thread's, a wave's or a segment's logits above the others'."""
    v = 60000
    up = torch.arange(v, device=DEV).float() / 4096
    x = torch.stack([up, up.flip(0), torch.where(torch.arange(v, device=DEV) < 40, up + 30, up),
                     torch.where(torch.arange(v, device=DEV) // 256 == 100, up + 30, up)])
    for take in (4, 64):
        assert _check(x, torch.zeros(1, 4, device=DEV), take) == take


@pytest.mark.parametrize("dtype", list(TYPES))
def test_masked_infinite_and_missing(dtype):
    inf, nan = float("inf"), float("nan")
    x, s = _inputs(6, 3, 900, dtype, 1)
    x[0] = -inf                      # a row that allows nothing
    x[3:6] = -inf                    # a request that allows nothing
    x[6, 1:] = -inf                  # one token
    x[7, 5] = nan
    x[7, 9] = inf
    x[8] = torch.finfo(x.dtype).min  # masks of the lowest value, all of a row
    x[9, :890] = torch.finfo(x.dtype).min
    x[10] = torch.finfo(x.dtype).max
    s[4] = torch.tensor([-inf, 0.0, nan], device=DEV)
    s[5] = -inf
    assert _check(x, s, 7) > 0
    p, t, top = _select(x, s, 7)
    assert (p[1] == -1).all() and (p[5] == -1).all() and (top[5] == -inf).all()


def test_the_first_step_and_ended_beams():
    x, s = _inputs(5, 4, 3001, "f16", 2)
    s[:, 1:] = -float("inf")
    assert _check(x, s, 8) == 40
    x, s = _inputs(5, 4, 3001, "f16", 3)
    done = torch.tensor([[0, 0, 0, 0], [1, 0, 0, 0], [1, 1, 1, 1], [0, 2, 0, -1], [0, 0, 0, 1]], dtype=torch.int32, device=DEV)
    x[4:8] = float("nan")            # (an ended beam's logits are not read)
    x[5:8] = 0
    _check(x, s, 8, done=done, end_token=3000)
    p, t, top = _select(x, s, 8, done=done, end_token=3000)
    assert (t[2, :4] == 3000).all() and (p[2, 4:] == -1).all() and torch.equal(top[2, :4], s[2].sort(descending=True).values)


def test_rows_apart_and_unaligned():
    """Rows of a wider buffer, from every offset of a 16-byte word."""
    for dtype in TYPES:
        buf, s = _inputs(2, 3, 1201, dtype, 4)
        for off in (1, 2, 3, 5, 8):
            _check(buf[:, off:off + 1000 + off], s, 9)


@pytest.mark.parametrize("dtype,vocab", [("f16", 50257), ("bf16", 50257), ("f32", 32003), ("f16", 1001), ("bf16", 999), ("f32", 133),
                                         ("f16", 200003), ("f32", 70001), ("f16", 5), ("f32", 3)])
def test_equal_beams_tie_at_every_alignment(dtype, vocab):
    """Rows of equal logits and scores that begin at other offsets of a 16-byte word: each token from the lowest beam on, and
    the same bits from any address."""
    beams, take = 5, 12
    row = _inputs(1, 1, vocab, dtype, vocab)[0][0]
    x, s = row.repeat(2 * beams, 1), torch.full((2, beams), -3.25, device=DEV)
    p, t, top = (o.cpu().numpy() for o in _select(x, s, take))
    r = row.float().cpu().numpy()
    want = np.lexsort((np.arange(beams * vocab), -np.tile(r, beams)))[:take]
    k = min(take, beams * int((r > -np.inf).sum()))
    for i in range(2):
        assert np.array_equal(t[i, :k], want[:k] % vocab) and np.array_equal(p[i, :k], i * beams + want[:k] // vocab)
    buf = torch.zeros(vocab + 16, dtype=row.dtype, device=DEV)
    first = None
    for off in range(9):
        buf[off:off + vocab] = row
        got = _select(buf[off:off + vocab].view(1, vocab), s[:1, :1].contiguous(), take)
        first = got if first is None else first
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_a_workspace_of_larger_numbers_and_a_stream_and_a_graph():
    ws = kvcache.beam_select_workspace(64, 8, 60000, 32, DEV)
    cases = [(_inputs(3, 4, 5000, "f16", i), 8) for i in range(3)] + [(_inputs(1, 8, 60000, "f32", 5), 16)]
    st = torch.cuda.Stream()
    for (x, s), take in cases:
        _check(x, s, take, ws=ws)
        st.wait_stream(torch.cuda.current_stream())
        _check(x, s, take, ws=ws, stream=st)
    (x, s), take = cases[0]
    n, beams = s.shape
    p, t = (torch.zeros(n, take, dtype=torch.int32, device=DEV) for _ in range(2))
    top = torch.zeros(n, take, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kvcache.beam_select(x, s, p, t, top, ws)
    for (x2, s2), _ in cases[:3]:
        x.copy_(x2)
        s.copy_(s2)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((p, t, top), _select(x, s, take)))


# ---- reorder -----------------------------------------------------------------

def _pool(rng, n_slots, mb, n_pages, fill):
    tables = np.full((n_slots, mb), -1, np.int32)
    for s in range(n_slots):
        k = rng.integers(0, int(mb * fill) + 1)
        tables[s, :k] = rng.integers(0, n_pages, k)
    refs = np.bincount(tables[tables >= 0], minlength=n_pages).astype(np.int32)
    return tables, refs


@pytest.mark.parametrize("n_slots,mb,bt,n", [(4, 3, 16, 4), (1, 1, 64, 1), (32, 40, 16, 20), (300, 700, 64, 300), (1024, 33, 16, 1024),
                                             (1500, 9, 16, 700)])
def test_reorder_against_the_list(n_slots, mb, bt, n):
    rng = np.random.default_rng(n_slots + mb)
    for trial in range(3):
        tables, refs = _pool(rng, n_slots, mb, 4 * n_slots + 5, 0.9)
        slots = rng.permutation(n_slots)[:n].astype(np.int32)
        parents = rng.integers(0, n_slots, n).astype(np.int32)
        tokens = rng.integers(0, mb * bt + 1, n).astype(np.int32)
        if trial == 1:                       # entries that are none
            slots[rng.integers(0, n)] = n_slots
            parents[rng.integers(0, n)] = -1
            tokens[rng.integers(0, n)] = mb * bt + 1
            slots[n - 1] = slots[0]
            if n > 1:
                tokens[n // 2] = -1
        if trial == 2:
            parents = slots.copy()           # themselves
            tokens[:] = mb * bt
        states = [rng.integers(0, 256, (n_slots, b)).astype(np.uint8) for b in (16, 48, 4, 20, 7, 4112)]
        t, r = torch.from_numpy(tables).to(DEV), torch.from_numpy(refs).to(DEV)
        dev = [torch.from_numpy(s).to(DEV) for s in states]
        st = torch.full((n,), 5, dtype=torch.int32, device=DEV)
        kvcache.pages_reorder(t, r, *(torch.from_numpy(a).to(DEV) for a in (slots, parents, tokens)), st,
                              kvcache.page_planes(dev), block_tokens=bt)
        want = L.reorder(tables, refs, slots.tolist(), parents.tolist(), tokens.tolist(), bt, states)
        assert st.cpu().tolist() == want
        assert np.array_equal(t.cpu().numpy(), tables) and np.array_equal(r.cpu().numpy(), refs)
        for a, b in zip(dev, states):
            assert np.array_equal(a.cpu().numpy(), b)


def test_reorder_entries_past_the_pool_and_without_status():
    tables = torch.tensor([[0, 99, -1], [1, 2, -7], [-1, -1, -1]], dtype=torch.int32, device=DEV)
    refs = torch.tensor([1, 1, 1], dtype=torch.int32, device=DEV)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    kvcache.pages_reorder(tables, refs, i(1, 0), i(0, 2), i(48, 48), block_tokens=16)
    assert tables.tolist() == [[-1, -1, -1], [0, 99, -1], [-1, -1, -1]] and refs.tolist() == [1, 0, 0]


def test_reorder_large_states_captured():
    """States of a megabyte a slot, a cycle of all slots replayed: after as many replays as slots all is as before."""
    n = 12
    state = torch.randn(n, 300000, device=DEV)
    odd = torch.randint(0, 255, (n, 100003), dtype=torch.uint8, device=DEV)
    tables = torch.arange(n * 50, dtype=torch.int32, device=DEV).view(n, 50)
    refs = torch.ones(n * 50, dtype=torch.int32, device=DEV)
    before = [a.clone() for a in (state, odd, tables, refs)]
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    parents, tokens = (slots + 5) % n, torch.full((n,), 800, dtype=torch.int32, device=DEV)
    planes = kvcache.page_planes([state, odd])
    args = (tables, refs, slots, parents, tokens, None, planes)
    g = torch.cuda.CUDAGraph()
    kvcache.pages_reorder(*args, block_tokens=16)
    torch.cuda.synchronize()
    assert torch.equal(state, before[0].roll(-5, 0)) and torch.equal(tables, before[2].roll(-5, 0))
    with torch.cuda.graph(g):
        kvcache.pages_reorder(*args, block_tokens=16)
    for _ in range(n - 1):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((state, odd, tables, refs), before))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_numbers_that_are_none_of_every_kind(dtype):
    """Quiet and signalling NaN and infinities beside the largest logits of their words, in rows of every length up to
    some words of a wave: none is selected, none is summed."""
    rng = np.random.default_rng(21)
    bits = {torch.float16: ([0x7e00, 0x7d01, 0xfe00, 0xfd55, 0x7c00, 0xfc00], torch.int16),
            torch.bfloat16: ([0x7fc0, 0x7f81, 0xffc0, 0xff95, 0x7f80, 0xff80], torch.int16),
            torch.float32: ([0x7fc00000, 0x7f800001, 0xffc00000, 0xff955555, 0x7f800000, 0xff800000], torch.int32)}[dtype]
    kinds = torch.tensor(np.array(bits[0], np.uint32).astype(np.int64)).to(torch.int64)
    kinds = (kinds - (kinds >= 2 ** (31 if dtype is torch.float32 else 15)) * 2 ** (32 if dtype is torch.float32 else 16)).to(bits[1])
    for vocab in (1, 7, 8, 9, 33, 500, 5000, 40000):
        for k in (1, 3, 8):
            x = torch.from_numpy(rng.standard_normal((6, vocab)) * 3).to(dtype)
            at = torch.from_numpy(rng.random((6, vocab)) < 0.2)
            pick = torch.from_numpy(rng.integers(0, 6, (6, vocab)))
            x.view(bits[1])[at] = kinds[pick][at]
            scores = torch.from_numpy(rng.standard_normal((3, 2)).astype(np.float32))
            _check(x.to(DEV), scores.to(DEV), k)


def test_the_most_rows_of_a_call():
    """2^24 requests of a beam, three tokens each, checked on the device.  A score is off by
    its sum's rounding (L.beam_scores: at most 3 / e * 5 + 42 of 2^-24) and its own."""
    n = 1 << 24
    g = torch.Generator(device=DEV).manual_seed(24)
    x = torch.randn(n, 3, device=DEV, generator=g).half()
    s = -torch.rand(n, 1, device=DEV, generator=g)
    p, t, top = _select(x, s, 2)
    assert torch.equal(p, torch.arange(n, dtype=torch.int32, device=DEV)[:, None].expand(n, 2))
    for i in range(0, n, n // 8):
        a = slice(i, i + n // 8)
        value, token = x[a].float().sort(stable=True, dim=-1, descending=True)
        ref = (value[:, :2].double() - x[a].double().logsumexp(-1, keepdim=True)) + s[a].double()
        assert torch.equal(t[a], token[:, :2].int())
        assert ((top[a].double() - ref).abs() <= (3 / np.e * 5 + 42 + ref.abs()) * 2.0 ** -24).all()


def test_rows_and_states_past_four_billion_bytes():
    g = torch.Generator(device=DEV).manual_seed(3)
    wide = torch.zeros(4, 1 << 30, dtype=torch.float16, device=DEV)
    x = wide[:, :33333]
    x.copy_(3 * torch.randn(4, 33333, device=DEV, generator=g))
    assert _check(x, torch.randn(2, 2, device=DEV, generator=g), 5) == 10
    del wide, x
    states = torch.zeros(260, 17 << 20, dtype=torch.uint8, device=DEV)
    rows = torch.randint(0, 256, (2, 17 << 20), dtype=torch.uint8, device=DEV, generator=g)
    states[0], states[259] = rows[0], rows[1]
    tables = torch.full((260, 2), -1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(4, dtype=torch.int32, device=DEV)
    slots = torch.tensor([0, 259, 130], dtype=torch.int32, device=DEV)
    parents = torch.tensor([259, 0, 259], dtype=torch.int32, device=DEV)
    kvcache.pages_reorder(tables, refs, slots, parents, torch.zeros_like(slots), None, kvcache.page_planes([states]), block_tokens=16)
    assert torch.equal(states[0], rows[1]) and torch.equal(states[259], rows[0]) and torch.equal(states[130], rows[1])
    assert not states[1:130].any() and not states[131:259].any()
