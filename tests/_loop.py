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
