"""Plain numpy forms, in 64 bits, of rotated rows and of attention over a window and sinks."""
import numpy as np

from tests import serve_util as S


def turned(x, pos, freqs, interleaved=False, magnitude=1.0, norm=None, eps=1e-6):
    """x [T, heads, D] f64: (rows normed and turned, how far f32 arithmetic may be off them).

    A turned dimension is w c + p s. What f32 leaves in units of 2^-24 of |w| + |p|: the mean square, a sum of
    at most 13 roundings, halved by the root (7); root, quotient, and two products (4); c and s, whose argument,
    sum and factor are rounded (5); product and last addition (2). 24 of them cover that. The angle is a
    product of f64 numbers and is reduced there: 2^-51 of its size."""
    x = np.asarray(x, np.float64)
    rot = 2 * len(freqs)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(norm, np.float64)
    angle = (np.asarray(pos, np.longdouble)[:, None] * np.asarray(freqs, np.longdouble))[:, None]
    c, s = (f(angle).astype(np.float64) * magnitude for f in (np.cos, np.sin))
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    y, off = x.copy(), np.abs(x) * 24 * 2.0 ** -24
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size = (np.abs(x[..., a]) + np.abs(x[..., b])) * abs(magnitude)
    off[..., a] = off[..., b] = size * (24 * 2.0 ** -24 + np.abs(angle).astype(np.float64) * 2.0 ** -51)
    return y, off


def seen(last, n, window, sinks):
    """Whether rows at positions last [m] see positions 0 .. n - 1."""
    j, p = np.arange(n)[None], np.asarray(last)[:, None]
    ok = j <= p
    return ok & ((j > p - window) | (j < sinks)) if window else ok


def attend(q, k, v, ok, scale):
    """q [m, D], k and v [n, D], ok [m, n]: f64 (out, sum p |v|, worst |q| . |k| scale) as serve_util.attend's."""
    z = np.where(ok, (np.where(np.isfinite(k), k, 0) @ q.T).T * scale, -np.inf)
    top = z.max(1, initial=-np.inf)
    e = np.exp(z - np.where(np.isfinite(top), top, 0)[:, None])
    total = e.sum(1, keepdims=True)
    p = e / np.where(total == 0, 1, total)
    size = np.where(ok, np.abs(q) @ np.abs(np.where(np.isfinite(k), k, 0)).T, 0).max(1, initial=0) * abs(scale)
    fine = np.where(np.isfinite(v), v, 0)
    return p @ fine, p @ np.abs(fine), size


def far(got, out, mass, size, bound):
    """By how much the worst element passes its bound."""
    d = np.abs(got - out) - bound(out, mass, size)
    return float(d.max(initial=-1.0)) if np.isfinite(got).all() else np.inf


KV4, PROMPT = S.kv4_bound, S.prompt_bound
