"""64-bit references of rotary positions, the paged 8-bit cache and the page calls,
and the layout helpers of their tests (numpy only)."""
import math

import numpy as np


def frequencies(rot, base=10000.0, scaling=None):
    f = base ** (-2.0 * np.arange(rot // 2) / rot)
    amp = 1.0
    if scaling is None:
        return f, amp
    if scaling[0] == "linear":
        f = f / scaling[1]
    elif scaling[0] == "ntk":
        f = (base * scaling[1] ** (rot / (rot - 2))) ** (-2.0 * np.arange(rot // 2) / rot)
    else:
        fast, slow = (list(scaling[3:]) + [32.0, 1.0][len(scaling) - 3:])[:2]
        turns = scaling[2] * f / (2 * math.pi)
        keep = np.clip((turns - slow) / (fast - slow), 0, 1)
        f, amp = keep * f + (1 - keep) * f / scaling[1], 1.0 + 0.1 * math.log(scaling[1])
    return f, amp


def rotate(x, positions, rot, layout, inverse=False, base=10000.0, scaling=None):
    """x [tokens][heads][hd] to 64-bit rows, and the bound of the kernel's fp32 steps before
    its rounding to fp16 (see rope_tolerance)."""
    f, amp = frequencies(rot, base, scaling)
    a = np.asarray(positions, np.float64)[:, None, None] * f * (-1 if inverse else 1)
    c, s = amp * np.cos(a), amp * np.sin(a)
    y = x.astype(np.float64).copy()
    ix, iy = (np.arange(rot // 2), np.arange(rot // 2) + rot // 2) if layout == "half" else \
        (np.arange(0, rot, 2), np.arange(1, rot, 2))
    p, q = x[..., ix].astype(np.float64), x[..., iy].astype(np.float64)
    y[..., ix], y[..., iy] = p * c - q * s, p * s + q * c
    return y


def rope_tolerance(x, ref, rot, layout, amp=1.0):
    """Half a step of fp16 (2^-11 relative, 2^-25 below the normal range) and the fp32 work: the
    cosine and sine are off by at most 2^-22 (polynomial 2^-29, its roundings and the
    angle's 2^-32 turns), the amplitude's product and the two products by 2^-24 each."""
    p = np.abs(x[..., :rot].astype(np.float64))
    mag = np.zeros_like(ref)
    if layout == "half":
        m = p[..., :rot // 2] + p[..., rot // 2:]
        mag[..., :rot] = np.concatenate([m, m], -1)
    else:
        m = p[..., 0::2] + p[..., 1::2]
        mag[..., :rot] = np.repeat(m, 2, -1)
    return np.abs(ref) * 2.0 ** -11 + 2.0 ** -25 + amp * mag * (2.0 ** -22 + 3 * 2.0 ** -24)


# ---- e4m3 ------------------------------------------------------------------

def e4m3_values():
    """The value of every code (NaN for 0x7f, 0xff)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0 ** -6)
    v[(b & 0x7f) == 0x7f] = np.nan
    return np.where(b & 0x80, -v, v)


CODES = e4m3_values()
_POS = CODES[:0x7f]


def e4m3_encode(x):
    """Nearest code of 64-bit |x| <= 448, ties to the even code."""
    a = np.abs(x)
    hi = np.clip(np.searchsorted(_POS, a), 1, 0x7e)
    lo = hi - 1
    dl, dh = a - _POS[lo], _POS[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def exponent(amax):
    """Smallest biased exponent >= 95 with amax <= 448 * 2^(e - 127)."""
    e = 95
    while amax > 448 * 2.0 ** (e - 127):
        e += 1
    return e


def limit(x):
    return np.clip(np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=61440, neginf=-61440), -61440, 61440)


def append(pool, exp, x, tables, starts, positions, max_tok=1 << 30):
    """In place: rows x [rows][kv][hd] into pool [pages][bt][kv][hd] / exp [pages][kv]."""
    n_pages, bt, kv, _ = pool.shape
    for s in range(len(positions)):
        n, p0 = min(starts[s + 1] - starts[s], max_tok), positions[s]
        t = 0
        while p0 >= 0 and t < n:
            p = p0 + t
            k = min(n - t, bt - p % bt)
            b, off = p // bt, p % bt
            page = tables[s][b] if b < tables.shape[1] else -1
            if 0 <= page < n_pages:
                rows = limit(x[starts[s] + t:starts[s] + t + k])
                for h in range(kv):
                    e = exponent(np.abs(rows[:, h]).max())
                    if off:
                        was = int(exp[page, h])
                        if e > was:
                            pool[page, :off, h] = e4m3_encode(CODES[pool[page, :off, h]] * 2.0 ** (was - e))
                        e = max(e, was)
                    exp[page, h] = e
                    pool[page, off:off + k, h] = e4m3_encode(rows[:, h] * 2.0 ** (127 - e))
            t += k


def random_pool(rng, n_pages, bt, kv, hd, scale=1.0):
    """Codes and exponents as the append writes them, pages of differing magnitudes."""
    x = rng.standard_normal((n_pages, bt, kv, hd)) * scale * 2.0 ** rng.integers(-3, 4, (n_pages, 1, kv, 1))
    exp = np.array([[exponent(np.abs(x[p, :, h]).max()) for h in range(kv)] for p in range(n_pages)], np.uint8)
    return e4m3_encode(x * 2.0 ** (127.0 - exp[:, None, :, None])), exp


def attention(q, kp, vp, ke, ve, tables, starts, positions, scale, window=0, sink=0, max_ctx=1 << 30):
    """64-bit outputs and tolerances of the rows that the slots own (others NaN).

    The tolerance counts, relative to A = sum p |v| / sum p and |o|: the rounding of each weight to fp16
    (2^-11; numerator and denominator hold the same rounded weights), weights below fp16's normal range
    (2^-25 of the reference weight each, which is at most the largest), the scores' fp32 sums (head_dim
    additions, 2^-24 of sum |q k| each, then the scaling, the difference and the exponential: 4 of 2^-23
    of the largest score), the fp32 sums over the keys (2^-24 each), and the output's rounding to fp16."""
    rows, nq, hd = q.shape
    n_pages, bt, kv, _ = kp.shape
    g = nq // kv
    out = np.full((rows, nq, hd), np.nan)
    tol = np.zeros((rows, nq, hd))
    for s in range(len(positions)):
        n, p0 = starts[s + 1] - starts[s], positions[s]
        if n <= 0 or p0 < 0:
            continue
        j = np.arange(min(p0 + n, max_ctx))
        b = j // bt
        page = np.where(b < tables.shape[1], tables[s][np.minimum(b, tables.shape[1] - 1)], -1)
        ok = (page >= 0) & (page < n_pages)
        page = np.where(ok, page, 0)
        for h in range(kv):
            k = CODES[kp[page, j % bt, h]] * 2.0 ** (ke[page, h].astype(np.float64) - 127)[:, None]
            v = CODES[vp[page, j % bt, h]] * 2.0 ** (ve[page, h].astype(np.float64) - 127)[:, None]
            for t in range(n):
                pos = p0 + t
                see = ok & (j <= pos)
                if window > 0:
                    see &= (j > pos - window) | (j < sink)
                kk, vv = k[see], v[see]
                for i in range(g):
                    r, qh = starts[s] + t, h * g + i
                    if not len(kk):
                        out[r, qh], tol[r, qh] = 0.0, 0.0
                        continue
                    x = q[r, qh].astype(np.float64)
                    sc = kk @ x * scale
                    mag = np.abs(kk) @ np.abs(x) * abs(scale)
                    w = np.exp(sc - sc.max())
                    l = w.sum()
                    o = w @ vv / l
                    a = w @ np.abs(vv) / l
                    d = 2 * ((hd + 2) * 2.0 ** -24 * mag.max() + 4 * np.abs(sc).max() * 2.0 ** -23)
                    # (the largest weight against the reference may be 1, all of l)
                    sub = len(kk) * 2.0 ** -25 * (np.abs(vv).max(0) + np.abs(o)) / l
                    out[r, qh] = o
                    tol[r, qh] = 2.0 ** -11 * np.abs(o) + 2.0 ** -25 + \
                        (2.0 ** -11 + np.expm1(d) + (len(kk) + 8) * 2.0 ** -23) * (a + np.abs(o)) + sub
    return out, tol


def layout(rng, lens, new, bt, kv, hd, spare=2, max_blocks=None):
    """Random pages for slots that hold lens[s] tokens and get new[s]: tables, starts, positions, n_pages."""
    need = [-(-(a + b) // bt) for a, b in zip(lens, new)]
    n_pages = sum(need) + spare
    order = rng.permutation(n_pages)
    tables = np.full((len(lens), max_blocks or max(max(need), 1)), -1, np.int32)
    at = 0
    for s, k in enumerate(need):
        tables[s, :k] = order[at:at + k]
        at += k
    return tables, np.cumsum([0] + list(new)).astype(np.int32), np.array(lens, np.int32), n_pages


# ---- page calls, one entry after the other ----------------------------------

OK, INVALID, PAGES = 0, -1, -9


def fork(tables, refs, parents, children, tokens, bt):
    st = []
    n_slots, mb = tables.shape
    before = tables.copy()
    for i, (p, c, k) in enumerate(zip(parents, children, tokens)):
        bad = not (0 <= p < n_slots and 0 <= c < n_slots and k >= 0) or -(-k // bt) > mb
        bad = bad or c in parents or c in children[:i]
        if not bad:
            nb = -(-k // bt)
            bad = (before[c] >= 0).any() or (before[p, :nb] >= len(refs)).any()
        st.append(INVALID if bad else OK)
        if not bad:
            tables[c, :nb] = before[p, :nb]
            for g in before[p, :nb]:
                if g >= 0:
                    refs[g] += 1
    return st


def release(tables, refs, slots, keep, bt):
    st = []
    for i, (s, k) in enumerate(zip(slots, keep)):
        bad = not 0 <= s < tables.shape[0] or k < 0 or s in slots[:i]
        st.append(INVALID if bad else OK)
        if not bad:
            for b in range(-(-k // bt), tables.shape[1]):
                if tables[s, b] >= 0:
                    refs[tables[s, b]] -= 1
                    tables[s, b] = -1
    return st


def reserve(tables, refs, slots, positions, n_new, max_new, bt):
    """Statuses and copied pairs."""
    start = refs.copy()
    free = [p for p in range(len(refs)) if start[p] == 0]
    st, pairs, taken = [], [], 0
    for i, (s, p0, k) in enumerate(zip(slots, positions, n_new)):
        pair = (-1, -1)
        bad = not 0 <= s < tables.shape[0] or p0 < 0 or not 0 <= k <= max_new or s in slots[:i]
        bad = bad or (k > 0 and (p0 + k - 1) // bt >= tables.shape[1])
        blocks = list(range(p0 // bt, (p0 + k - 1) // bt + 1)) if not bad and k else []
        bad = bad or any(tables[s, b] >= len(refs) for b in blocks)
        if bad:
            st.append(INVALID)
        else:
            want = [b for b in blocks if tables[s, b] < 0 or start[tables[s, b]] > 1]
            taken += len(want)
            if want and taken > len(free):
                st.append(PAGES)
            else:
                st.append(OK)
                fresh = free[taken - len(want):taken]
                for b, f in zip(want, fresh):
                    old = tables[s, b]
                    if old >= 0:
                        refs[old] -= 1
                        if b == p0 // bt and p0 % bt:
                            pair = (old, f)
                    tables[s, b] = f
                    refs[f] = 1
        pairs.append(pair)
    return st, pairs


def compact(tables, refs):
    """moved and the number of pages in use."""
    used = [p for p in range(len(refs)) if refs[p] > 0]
    n = len(used)
    holes = [p for p in range(n) if refs[p] <= 0]
    moved = np.full(len(refs), -1, np.int32)
    for p in used:
        moved[p] = p if p < n else holes.pop(0)
    for s in range(tables.shape[0]):
        for b in range(tables.shape[1]):
            if 0 <= tables[s, b] < len(refs) and moved[tables[s, b]] >= 0:
                tables[s, b] = moved[tables[s, b]]
    after = np.zeros_like(refs)
    for p in used:
        after[moved[p]] = refs[p]
    refs[:] = np.where((after > 0) | (refs > 0), after, refs)
    return moved, n
