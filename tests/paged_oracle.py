"""TEST INFRASTRUCTURE ONLY: the paged cache and its attention in numpy, from
their definitions, nibble by nibble and sequence by sequence, in float64 (the
rotation of a key that is stored in 4 bits also in the float32 steps that
define its code)."""
from __future__ import annotations

import numpy as np

F16, F32, F64 = np.float16, np.float32, np.float64
GROUP = 32
HALF_ULP16 = 2.0**-11  # half a step of fp16, relative


def rotate(x, w, eps, cos, sin, f=F64):
    """Norm (w not None) and rotate-half of x [T, H, hd], cos / sin [T, hd/2]; f = float32: each step rounded, the norm's
    factor computed in float64 and rounded once."""
    x = x.astype(f)
    if w is not None:
        inv = (1 / np.sqrt((x.astype(F64) ** 2).mean(-1, keepdims=True) + F64(F32(eps)))).astype(f)
        x = x * inv * w.astype(f)
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cos[:, None].astype(f), sin[:, None].astype(f)
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def quantize(x, group):
    """(codes, fp16 scales) of x [..., n] float32 in groups of `group`."""
    g = x.astype(F32).reshape(*x.shape[:-1], -1, group)
    with np.errstate(all="ignore"):
        amax = np.abs(g).max(-1)
        s = np.where(amax / F32(7) < F32(2.0**-14), F32(2.0**-14), amax / F32(7)).astype(F16)
        q = np.rint(g / s.astype(F32)[..., None])
        q = np.where(np.isnan(q), 0, np.clip(q, -7, 7)).astype(np.int64)
    return q.reshape(x.shape), s


def put(pools, bits, page, pid, slot, k, v):
    """One position's rows k (float32), v (float16) [H, hd] into page pid."""
    kp, vp = pools
    H, hd = k.shape
    if bits == 16:
        kp[pid, :, slot], vp[pid, :, slot] = k.astype(F16), v
        return
    kq, ks = quantize(k, GROUP)
    vq, vs = quantize(v.astype(F32), hd)
    for h in range(H):
        kb, vb = kp[pid, h].reshape(-1), vp[pid, h].reshape(-1)
        for d in range(hd):
            j, t, e = d // 32, d % 32 // 8, d % 8
            n = e // 2 + 4 * (e % 2)
            at, sh = slot * (hd // 2) + 4 * (t * (hd // 32) + j) + n // 2, 4 * (n % 2)
            kb[at] = int(kb[at]) & ~(15 << sh) & 255 | (int(kq[h, d]) & 15) << sh
            at, sh = slot // 2 * hd + d // 4 * 4 + 2 * (slot % 2) + d % 4 // 2, 4 * (d % 2)
            vb[at] = int(vb[at]) & ~(15 << sh) & 255 | (int(vq[h, d]) & 15) << sh
        code = page * hd // 2
        kb[code:].view(F16)[slot * (hd // GROUP) : (slot + 1) * (hd // GROUP)] = ks[h]
        vb[code:].view(F16)[slot] = vs[h, 0]


def get(pools, bits, page, hd, pid, slot):
    """(k, v) float64 [H, hd] that position slot of page pid stands for."""
    kp, vp = pools
    if bits == 16:
        return kp[pid, :, slot].astype(F64), vp[pid, :, slot].astype(F64)
    H, code = kp.shape[1], page * hd // 2
    d = np.arange(hd)
    j, t, e = d // 32, d % 32 // 8, d % 8
    n = e // 2 + 4 * (e % 2)

    def nib(b, at, sh):
        x = (b[:, at] >> sh & 15).astype(np.int64)
        return np.where(x > 7, x - 16, x).astype(F64)

    kb, vb = kp[pid].reshape(H, -1), vp[pid].reshape(H, -1)
    k = nib(kb, slot * (hd // 2) + 4 * (t * (hd // 32) + j) + n // 2, 4 * (n % 2))
    v = nib(vb, slot // 2 * hd + d // 4 * 4 + 2 * (slot % 2) + d % 4 // 2, 4 * (d % 2))
    ks = np.ascontiguousarray(kb[:, code:]).view(F16).astype(F64)[:, slot * (hd // GROUP) + d // GROUP]
    vs = np.ascontiguousarray(vb[:, code:]).view(F16).astype(F64)[:, slot : slot + 1]
    with np.errstate(invalid="ignore"):
        return k * ks, v * vs


def context(pools, bits, page, hd, table_row, n, pages):
    """Rows of a sequence's first n positions and which of them have a page: k, v [n, H, hd], on [n]."""
    H = pools[0].shape[1]
    k, v, on = np.zeros((n, H, hd)), np.zeros((n, H, hd)), np.zeros(n, bool)
    for p in range(n):
        pid = int(table_row[p // page]) if p // page < len(table_row) else -1
        if 0 <= pid < pages:
            k[p], v[p] = get(pools, bits, page, hd, pid, p % page)
            on[p] = True
    return k, v, on


def attention(q, k, v, seen):
    """q [R, NQ, hd] over k, v [n, NKV, hd]; seen [R, n].  Returns (out, mean of |v| under the weights, largest
    sum |q k| / sqrt hd of a row and head), all float64; a row that sees nothing gives zeros."""
    R, nq, hd = q.shape
    rep = nq // k.shape[1]
    out, mag, dot = np.zeros((R, nq, hd)), np.zeros((R, nq, hd)), np.zeros((R, nq, 1))
    for h in range(nq):
        kk, vv, qq = k[:, h // rep], v[:, h // rep], q[:, h].astype(F64)
        x = qq @ kk.T / np.sqrt(hd)
        a = np.abs(qq) @ np.abs(kk).T / np.sqrt(hd)
        for r in range(R):
            on = seen[r]
            if on.any():
                w = np.exp(x[r, on] - x[r, on].max())
                w /= w.sum()
                out[r, h], mag[r, h], dot[r, h] = w @ vv[on], w @ np.abs(vv[on]), a[r, on].max()
    return out, mag, dot


def attention_bound(out, mag, dot, q=None, kscale=0.0):
    """How far a kernel's output may be off: probabilities rounded once to 11 bits (half a step, 2^-11, of each term);
    scores off by d = 2^-19 of the sum of their products' magnitudes (fp32 sums of up to 128 products, in any order, and
    the exponential's argument), which moves a weight by 2 d and the weights' sum by as much; the output's own rounding.
    4-bit keys enter as 72 + code: their products' magnitudes are up to 80 scale |q|."""
    d = dot
    if q is not None:
        d = d + 80 * kscale * np.abs(q.astype(F64)).sum(-1, keepdims=True) / np.sqrt(q.shape[-1])
    return mag * (HALF_ULP16 + 4 * 2.0**-19 * d + 2.0**-16) + HALF_ULP16 * np.abs(out) + 2.0**-24
