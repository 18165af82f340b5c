"""64-bit references of the operators around the paged 8-bit cache in a decoding loop (numpy only): norms of
heads with the rotation and their gradient."""
import numpy as np

from tests import _paged8 as R


def _pair_sums(a, rot, layout):
    """|x| + |y| of each turned pair in both its places, |x| elsewhere (a >= 0)."""
    out = a.copy()
    if rot == 0:
        return out
    if layout == "half":
        m = a[..., :rot // 2] + a[..., rot // 2:rot]
        out[..., :rot] = np.concatenate([m, m], -1)
    else:
        out[..., :rot] = np.repeat(a[..., 0:rot:2] + a[..., 1:rot:2], 2, -1)
    return out


def _turn(x, positions, rot, layout, inverse, base, scaling):
    if rot == 0:
        return x, 1.0
    return R.rotate(x, positions, rot, layout, inverse, base, scaling), R.frequencies(rot, base, scaling)[1]


# Relative errors of the kernels' fp32 steps, each rounding 2^-24: a sum of hd squares (hd of them, halved by the
# root) with its mean, eps and v_rsq_f32 (one step); a cosine or sine 2^-22 (rope_tolerance) and the products
# and sum around it 3.
def _scale_error(hd):
    return hd * 2.0 ** -25 + 2.0 ** -22


_TURN = 2.0 ** -22 + 3 * 2.0 ** -24


def norm_rope(x, w, positions, rot, layout, eps=1e-6, base=10000.0, scaling=None):
    """x [tokens][heads][hd] to 64-bit rows and their tolerance: half a step of fp16 (2^-11, 2^-25 below the
    normal range) and the fp32 steps ahead of it."""
    x = x.astype(np.float64)
    hd = x.shape[-1]
    u = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    y, amp = _turn(u, positions, rot, layout, False, base, scaling)
    mag = amp * _pair_sums(np.abs(u), rot, layout)
    return y, np.abs(y) * 2.0 ** -11 + 2.0 ** -25 + mag * (_TURN + _scale_error(hd) + 3 * 2.0 ** -24)


def norm_rope_grad(x, dy, w, positions, rot, layout, eps=1e-6, base=10000.0, scaling=None):
    """(dx, its tolerance, dw, its tolerance) in 64 bits."""
    x, dy, w = x.astype(np.float64), dy.astype(np.float64), w.astype(np.float64)
    hd = x.shape[-1]
    rows = x.shape[0] * x.shape[1]
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    g, amp = _turn(dy, positions, rot, layout, True, base, scaling)
    xr, h = x * r, g * w
    m = (h * xr).mean(-1, keepdims=True)
    dx = r * (h - xr * m)
    er = _scale_error(hd) + 2.0 ** -24
    eg = amp * _pair_sums(np.abs(dy), rot, layout) * _TURN
    eh = np.abs(w) * eg + np.abs(h) * 2.0 ** -24
    # the mean's products and sum, and the scale in it
    em = (np.abs(xr) * eh).mean(-1, keepdims=True) + np.abs(h * xr).mean(-1, keepdims=True) * (hd + 4) * 2.0 ** -24 + np.abs(m) * er
    tol = r * (eh + np.abs(xr) * em + (np.abs(h) + 2 * np.abs(xr * m)) * (er + 3 * 2.0 ** -24))
    tol = tol + np.abs(dx) * 2.0 ** -11 + 2.0 ** -25
    dw = (g * xr).sum((0, 1))
    # sums of rows numbers in any order: rows additions
    tw = (np.abs(xr) * eg).sum((0, 1)) + np.abs(g * xr).sum((0, 1)) * (er + (rows + 4) * 2.0 ** -24)
    return dx, tol, dw, tw


# ---- beam search -------------------------------------------------------------

def beam_scores(logits, scores, done=None, end_token=0):
    """S [n][beams * vocab] in 64 bits (-inf: no candidate) and the tolerance of the searched beams' scores.

    Ahead of the rounding to fp32 (2^-24 of S): the distances t to a segment's maximum (rounded once), their product
    with log2(e) (two roundings) and the exponential (2^-23), weighted by their share of the sum; the sum's additions
    in a thread (32), a wave (6) and a workgroup (2)."""
    n, beams = scores.shape
    x = logits.astype(np.float64)
    x[~(x < np.inf)] = -np.inf
    x = x.reshape(n, beams, -1)
    out = np.full(x.shape, -np.inf)
    tol = np.zeros((n, beams))
    for r in range(n):
        for b in range(beams):
            s = float(scores[r, b])
            if not s > -np.inf:
                continue
            if done is not None and done[r, b]:
                out[r, b, end_token] = s
                continue
            m = x[r, b].max()
            if m == -np.inf:
                continue
            t = x[r, b] - m
            p = np.exp(t)
            out[r, b] = s + (t - np.log(p.sum()))
            far = np.where(p > 0, -t, 0)
            tol[r, b] = ((p * far).sum() / p.sum() * 5 + 2 + 40) * 2.0 ** -24
    return out.reshape(n, -1), tol


def beam_check(logits, scores, take, parents, tokens, top, done=None, end_token=0):
    """Asserts that parents, tokens and top (numpy) are the selection, and returns how many candidates there were."""
    n, beams = scores.shape
    S, tol = beam_scores(logits, scores, done, end_token)
    vocab = S.shape[1] // beams
    total = 0
    for r in range(n):
        order = np.lexsort((np.arange(S.shape[1]), -S[r]))[:take + 1]
        order = order[S[r][order] > -np.inf]
        want = order[:take]
        k = len(want)
        total += k
        assert (parents[r, k:] == -1).all() and (tokens[r, k:] == -1).all() and (top[r, k:] == -np.inf).all()
        got = (parents[r, :k] - r * beams) * vocab + tokens[r, :k]
        assert (parents[r, :k] // beams == r).all() and ((tokens[r, :k] >= 0) & (tokens[r, :k] < vocab)).all()
        s = S[r][want]
        lim = np.abs(s) * 2.0 ** -24 + tol[r].max()
        assert (np.abs(top[r, :k] - s) <= lim).all()
        assert len(set(got.tolist())) == k and (np.abs(S[r][got] - s) <= 2 * lim).all()
        # the same entries, but where two beams' candidates are nearer than the scores' errors
        for i in range(k):
            near = [j for j in (i - 1, i + 1) if 0 <= j < len(order) and order[j] // vocab != order[i] // vocab and
                    abs(S[r][order[j]] - s[i]) <= 4 * lim[i]]
            assert got[i] == want[i] or near, (r, i, got, want)
    return total


# ---- pages -------------------------------------------------------------------

def reorder(tables, refs, slots, parents, n_tokens, bt, states=()):
    """In place; the statuses."""
    n_slots, mb = tables.shape
    before, rows = tables.copy(), [s.copy() for s in states]
    st = []
    for i, (s, p, k) in enumerate(zip(slots, parents, n_tokens)):
        nb = -(-k // bt)
        bad = not (0 <= s < n_slots and 0 <= p < n_slots and k >= 0) or nb > mb or s in slots[:i]
        st.append(R.INVALID if bad else R.OK)
        if bad:
            continue
        new = np.full(mb, -1, np.int32)
        new[:nb] = before[p, :nb]
        new[new < 0] = -1
        for g in new:
            if 0 <= g < len(refs):
                refs[g] += 1
        for g in before[s]:
            if 0 <= g < len(refs):
                refs[g] -= 1
        # (an entry below zero that stays one is not written)
        tables[s] = np.where((new < 0) & (before[s] < 0) & (np.arange(mb) >= nb) & (before[s] == -1), before[s], new)
        for a, b in zip(states, rows):
            a[s] = b[p]
    return st


# ---- eviction ------------------------------------------------------------------

def evict(pools, exps, weights, tables, lens, keep, max_ctx, max_keep, sink=0, recent=0):
    """In place on [k, v] pools, exponents and weights [pages][kv][bt]; returns kept."""
    n_pages, bt, kv, _ = pools[0].shape
    n_slots, mb = tables.shape
    kept = np.full((n_slots, kv, max_keep), -1, np.int32)
    for s in range(n_slots):
        n, k = int(lens[s]), int(keep[s])
        if n < 0 or n > max_ctx or k < 0 or min(n, k) > max_keep or -(-n // bt) > mb:
            continue
        pages = tables[s, :-(-n // bt)]
        if ((pages < 0) | (pages >= n_pages)).any():
            continue
        j = np.arange(n)
        page, row = pages[j // bt], j % bt
        for h in range(kv):
            if k >= n:
                kept[s, h, :n] = j
                continue
            last = min(k, recent)
            first = min(k - last, sink)
            w = weights[page, h, row].astype(np.float64)
            mid = np.arange(first, n - last)
            v = np.where(np.isnan(w[mid]), -np.inf, w[mid])
            # (a NaN is below -infinity too)
            order = np.lexsort((mid, -v, np.isnan(w[mid])))
            rows = np.sort(np.concatenate([np.arange(first), mid[order[:k - first - last]], np.arange(n - last, n)]).astype(int))
            kept[s, h, :k] = rows
            if k == 0:
                continue
            weights[page[:k], h, row[:k]] = weights[page[rows], h, row[rows]]
            for pool, exp in zip(pools, exps):
                codes, e = pool[page[rows], row[rows], h], exp[page[rows], h].astype(int)
                for a in range(0, k, bt):
                    b = min(k, a + bt)
                    top = e[a:b].max()
                    x = R.e4m3_encode(R.CODES[codes[a:b]] * 2.0 ** (e[a:b] - top)[:, None])
                    pool[page[a], :b - a, h] = np.where((e[a:b] == top)[:, None], codes[a:b], x)
                    exp[page[a], h] = top
    return kept


# ---- accumulated weights ---------------------------------------------------------

def weigh(q, kp, ke, weights, tables, starts, positions, scale, weighed=None, decay=1.0, window=0, sink=0,
          max_ctx=1 << 30, max_tok=1 << 30):
    """64-bit weights [pages][kv][bt] after a call, and tolerances (0 where nothing is written).

    Each softmax weight is off, relatively, by: its score's fp32 sum (head_dim additions, 2^-24 of sum |q k| each),
    the scaling, the difference and the exponential (4 of 2^-23 of the largest score), the same in its row's sum,
    that sum's additions (half the keys in a lane, 40 joining lanes, waves and chunks) and reciprocal, and the sum over
    rows (half of them in a lane, 40 joining); then the decay's product and sum."""
    rows, nq, hd = q.shape
    n_pages, bt, kv, _ = kp.shape
    g = nq // kv
    out = weights.astype(np.float64)
    tol = np.zeros(weights.shape)
    for s in range(len(positions)):
        n, p0 = min(int(starts[s + 1] - starts[s]), max_tok), int(positions[s])
        if n <= 0 or p0 < 0:
            continue
        j = np.arange(min(p0 + n, max_ctx))
        b = j // bt
        page = np.where(b < tables.shape[1], tables[s][np.minimum(b, tables.shape[1] - 1)], -1)
        ok = (page >= 0) & (page < n_pages)
        page = np.where(ok, page, 0)
        pos = p0 + np.arange(n)[:, None]
        see = ok & (j <= pos)
        if window > 0:
            see &= (j > pos - window) | (j < sink)
        for h in range(kv):
            k = R.CODES[kp[page, j % bt, h]] * 2.0 ** (ke[page, h].astype(np.float64) - 127)[:, None]
            k = np.where(ok[:, None], k, 0.0)
            a, e = np.zeros(len(j)), np.zeros(len(j))
            for i in range(g):
                x = q[starts[s]:starts[s] + n, h * g + i].astype(np.float64)
                sc = np.where(see, x @ k.T * scale, -np.inf)
                mag = np.where(see, np.abs(x) @ np.abs(k).T * abs(scale), 0).max(1)
                top = np.where(see, np.abs(sc), 0).max(1)
                with np.errstate(invalid="ignore"):
                    w = np.exp(sc - np.where(see.any(1), sc.max(1), 0)[:, None])
                w = w / np.maximum(w.sum(1, keepdims=True), 1e-300)
                d = 2 * ((hd + 2) * 2.0 ** -24 * mag + 4 * (top + 1) * 2.0 ** -23) + (len(j) / 2 + 44) * 2.0 ** -24
                a += w.sum(0)
                e += (w * np.expm1(d)[:, None]).sum(0)
            e += a * (n * g / 2 + 40) * 2.0 ** -24
            old = np.zeros(len(j))
            stands = j < (p0 if weighed is None else weighed[s])
            if decay != 0:
                old = np.where(stands, decay * weights[page, h, j % bt].astype(np.float64), 0.0)
            at = page[ok], h, (j % bt)[ok]
            out[at] = (old + a)[ok]
            tol[at] = (e + (np.abs(old) * 2 + a) * 2.0 ** -24 + 2.0 ** -120)[ok]
    return out, tol
