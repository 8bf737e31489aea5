"""Plain numpy forms of the serving operators' definitions (64 bits unless a rule is in 32), and
the cache's layout written element by element."""
import math

import numpy as np

from glint_amd import codebook

PAGE = 64
PARENT = np.array(codebook.PARENT, np.float64).astype(np.float32)


def hole_codes(w):
    """[..., D] f32 -> (codes u8 [..., D], absmax f32 [..., D / 64]) by the codec's rule in f32."""
    w = np.asarray(w, np.float32)
    blocks = w.reshape(*w.shape[:-1], -1, 64)
    a = np.abs(blocks)
    s = np.where(np.isnan(a), np.float32(0), a).max(-1).astype(np.float32)
    with np.errstate(all="ignore"):
        v = np.where(s[..., None] == 0, np.float32(0), blocks / s[..., None]).astype(np.float32)
        d = np.abs(v[..., None] - PARENT)
    code = np.where(np.isnan(v), 0, np.argmin(np.where(np.isnan(d), np.float32(np.inf), d), -1)).astype(np.uint8)
    return code.reshape(w.shape), s


def empty_planes(pages, H, D, fill=0):
    nb = D // 64
    return [np.full((pages, H, PAGE, D // 2), fill, np.uint8), np.zeros((pages, H, nb, PAGE), np.float32),
            np.full((pages, H, D // 2, PAGE), fill, np.uint8), np.zeros((pages, H, nb, PAGE), np.float32)]


def _k_at(d, nb):
    return ((d % 64) // 16 * nb + d // 64) * 8 + d % 16 // 2, 4 * (d % 2)


def _v_at(d):
    return d // 32 * 16 + d % 16, 4 * (d % 32 // 16)


def put(planes, slot, k, v):
    """Token (k, v [H, D]) into slot, one nibble at a time."""
    kh, ka, vh, va = planes
    page, t = divmod(int(slot), PAGE)
    D = k.shape[-1]
    (ck, sk), (cv, sv) = hole_codes(k), hole_codes(v)
    ka[page, :, :, t], va[page, :, :, t] = sk, sv
    for d in range(D):
        b, sh = _k_at(d, D // 64)
        kh[page, :, t, b] = (kh[page, :, t, b] & (0xF0 >> sh)) | (ck[:, d] << sh)
        r, sh = _v_at(d)
        vh[page, :, r, t] = (vh[page, :, r, t] & (0xF0 >> sh)) | (cv[:, d] << sh)


def put_all(planes, slots, k, v):
    """put() for tokens [T, H, D] in different slots, all at once."""
    kh, ka, vh, va = planes
    page, t = np.divmod(np.asarray(slots, np.int64), PAGE)
    D = k.shape[-1]
    (ck, sk), (cv, sv) = hole_codes(k), hole_codes(v)
    ka[page, :, :, t], va[page, :, :, t] = sk, sv
    for d in range(D):
        b, sh = _k_at(d, D // 64)
        kh[page, :, t, b] = (kh[page, :, t, b] & (0xF0 >> sh)) | (ck[..., d] << sh)
        r, sh = _v_at(d)
        vh[page, :, r, t] = (vh[page, :, r, t] & (0xF0 >> sh)) | (cv[..., d] << sh)


def held(planes, slots):
    """f64 (k, v) [tokens, H, D] of the slots."""
    kh, ka, vh, va = planes
    slots = np.asarray(slots, np.int64)
    page, t = slots // PAGE, slots % PAGE
    H, D = kh.shape[1], kh.shape[3] * 2
    k, v = np.zeros((2, len(slots), H, D))
    for d in range(D):
        b, sh = _k_at(d, D // 64)
        k[:, :, d] = PARENT[kh[page, :, t, b] >> sh & 15].astype(np.float64) * ka[page, :, d // 64, t]
        r, sh = _v_at(d)
        v[:, :, d] = PARENT[vh[page, :, r, t] >> sh & 15].astype(np.float64) * va[page, :, d // 64, t]
    return k, v


def attend(q, k, v, last, scale):
    """q [n, D], k and v [m, D]; row i sees keys 0 .. last[i]. f64 (out, sum p |v|, worst |q| . |k| scale)."""
    out, mass, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros(len(q))
    for i, n in enumerate(last):
        n = min(int(n) + 1, len(k))
        if n <= 0:
            continue
        with np.errstate(invalid="ignore"):
            z = k[:n] @ q[i] * scale
            p = np.exp(z - z.max())
            p /= p.sum()
            out[i], mass[i] = p @ v[:n], p @ np.abs(v[:n])
        size[i] = (np.abs(k[:n]) @ np.abs(q[i])).max() * abs(scale)
    return out, mass, size


def bf16_values(bits):
    return (np.asarray(bits).view(np.uint16).astype(np.uint32) << 16).view(np.float32)


def kv4_bound(out, mass, size):
    """What f16 products may be off: the output's bf16 rounding; 2^-12 of each value, each weight and each
    key element (a score is off by at most 2^-12 |q| . |k|, a weight by e to twice that); f32 sums and
    a hardware 2^x of 1 ulp."""
    return 2.0 ** -8 * np.abs(out) + mass * (2 * 2.0 ** -12 + np.expm1(2 * (2.0 ** -12 + 2.0 ** -18) * size)[:, None] + 2.0 ** -16)


def prompt_bound(out, mass, size):
    """The output's bf16 rounding (2^-8); 2^-9 for the weights, half of what they would be off if bf16 rounded
    all of them the same way: many average out, and where few count their rest is added back; f32 scores."""
    return 2.0 ** -8 * np.abs(out) + mass * (2.0 ** -9 + np.expm1(2.0 ** -16 * size)[:, None] + 2.0 ** -16)


def logprobs(x, tok, top):
    """One row: (lse, logprob, entropy, rank, top indices), and how far f32 may be off the lse: the
    sums of a thread's elements and of the threads, the rounded exponents (weighted by their size), and
    the last additions."""
    x = np.asarray(x, np.float64)
    m = x.max()
    e = np.exp(x - m)
    s = e.sum()
    lse = m + math.log(s)
    fin = e > 0
    mean = (e[fin] * (m - x[fin])).sum() / s
    ent = math.log(s) + mean
    rank = int(((x > x[tok]) | ((x == x[tok]) & (np.arange(len(x)) < tok))).sum())
    order = np.lexsort((np.arange(len(x)), -x))[:top]
    off = (len(x) / 1024 + 40) * 2.0 ** -24 + mean * 2.0 ** -22 + (abs(lse) + abs(m)) * 2.0 ** -23
    return lse, x[tok] - lse, ent, rank, order, off
