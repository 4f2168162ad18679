"""The 4-bit cache and its operators restated in numpy, 64 bits, from the
description in include/midgecuda.h and the tile layout of the cache: what the
kernel tests compare with.  Nothing here calls the library."""
from __future__ import annotations

import numpy as np

MAG = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
MID = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
SCALE_BYTES = np.arange(4, 114)  # 2^-14 .. 10240


def e5m2(b):
    return (np.asarray(b, np.uint16) << 8).view(np.float16).astype(np.float64)


def quantise(x):
    """[..., D] -> (codes [..., D], scale bytes [..., D / 32])"""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    g = np.where(np.isnan(g), 0.0, g)
    top = np.abs(g).max(-1)
    i = np.minimum(np.searchsorted(e5m2(SCALE_BYTES) * 6, top), len(SCALE_BYTES) - 1)
    sb = np.where(top > 0, SCALE_BYTES[i], 0).astype(np.uint8)
    s = e5m2(sb)[..., None]
    a = np.abs(g)
    code = np.zeros(g.shape, np.uint8)
    for k, m in enumerate(MID):
        code += ((a > m * s) if k % 2 == 0 else (a >= m * s)).astype(np.uint8)
    code = np.where(s > 0, code, 0).astype(np.uint8) | ((g < 0).astype(np.uint8) << 3)
    return code.reshape(x.shape), sb


def values(code, sb):
    v = np.where(code & 8, -1.0, 1.0) * MAG[code & 7]
    return (v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32) * e5m2(sb)[..., None]).reshape(v.shape)


def k_place(p, d, D):
    u, g, j = p >> 4, (p >> 1) & 7, p & 1
    lane = g * 4 + d // (D // 4)
    if D == 64:
        return u * 512 + lane * 16 + j * 8 + d % 16 // 2
    return (2 * u + j) * 512 + lane * 16 + d % 32 // 2


def v_place(p, d, D):
    u, t, i = p >> 4, (p >> 2) & 3, p & 3
    lane = d // (D // 8) * 4 + t
    if D == 64:
        return 16 * D + u * 512 + lane * 16 + i * 4 + d % 8 // 2
    return 16 * D + (2 * u + (i & 1)) * 512 + lane * 16 + (i >> 1) * 8 + d % 16 // 2


def k_scale_place(p, grp, D):
    return 32 * D + (((p >> 1) & 7) * (D // 32) + grp) * 4 + (p >> 4) * 2 + (p & 1)


def v_scale_place(p, grp, D):
    return 33 * D + ((((p >> 2) & 3) * (D // 32) + grp) * 2 + (p >> 4)) * 4 + (p & 3)


class Cache:
    """A pool of pages on the host."""

    def __init__(self, n_kv, D, page, tables, n_pages, fill=0):
        self.n_kv, self.D, self.page = n_kv, D, page
        self.pool = np.full((n_pages, n_kv, page // 32, 34 * D), fill, np.uint8)
        self.table = np.asarray(tables, np.int32)

    def store(self, seq, pos, head, x, keys):
        c, sb = quantise(x)
        tile = self.pool[self.table[seq, pos // self.page], head, pos % self.page // 32]
        d = np.arange(self.D)
        at, sc = (k_place, k_scale_place) if keys else (v_place, v_scale_place)
        p = pos % 32
        by = at(p, d, self.D)
        tile[by[0::2]] = c[0::2] | c[1::2] << 4
        tile[sc(p, np.arange(self.D // 32), self.D)] = sb

    def load(self, seq, length, head, keys):
        """Positions 0 .. length - 1 as [length, D]"""
        pos = np.arange(length)[:, None]
        d = np.arange(self.D)[None]
        at, sc = (k_place, k_scale_place) if keys else (v_place, v_scale_place)
        page = self.table[seq, pos // self.page]
        tile = pos % self.page // 32
        code = self.pool[page, head, tile, at(pos % 32, d, self.D)] >> (d % 2 * 4) & 15
        sb = self.pool[page, head, tile, sc(pos % 32, np.arange(self.D // 32)[None], self.D)]
        return values(code, sb)


def attention(cache, q, q_start, kv_len, n_heads, scale, window=0, sinks=None):
    """q [rows, n_heads * D] -> (out, bound) in 64 bits: bound [rows, n_heads] is
    max_t scale sum_d |q_d k_td| and max |v| over the seen positions."""
    D, n_kv = cache.D, cache.n_kv
    gq = n_heads // n_kv
    out = np.zeros((q.shape[0], n_heads, D))
    bs = np.zeros((q.shape[0], n_heads))
    bv = np.zeros((q.shape[0], n_heads))
    for s in range(len(kv_len)):
        a, b = int(q_start[s]), int(q_start[s + 1])
        n, length = b - a, int(kv_len[s])
        for h in range(n_kv):
            k, v = cache.load(s, length, h, True), cache.load(s, length, h, False)
            for j in range(n):
                p = length - n + j
                lo = max(0, p - window + 1) if window else 0
                if p < 0:
                    continue
                kk, vv = k[lo:p + 1], v[lo:p + 1]
                for i in range(h * gq, (h + 1) * gq):
                    x = q[a + j, i * D:(i + 1) * D].astype(np.float64)
                    sc = kk @ x * scale
                    m = sc.max()
                    extra = 0.0
                    if sinks is not None:
                        m = max(m, float(sinks[i]))
                        extra = np.exp(float(sinks[i]) - m)
                    e = np.exp(sc - m)
                    out[a + j, i] = e @ vv / (e.sum() + extra)
                    bs[a + j, i] = (np.abs(kk) @ np.abs(x)).max() * abs(scale)
                    bv[a + j, i] = np.abs(vv).max()
    return out, bs, bv


def logprobs(x, ids, top):
    """One row in 64 bits: (lp, entropy, order)"""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.lexsort((np.arange(len(x)), -x))[:top]
    m = x.max()
    if m == -np.inf:
        return np.full(len(ids), -np.inf), 0.0, order, np.full(len(order), -np.inf)
    d = x - m
    e = np.exp(d)
    z = np.log(e.sum())
    ent = z - np.sum(e[e > 0] * d[e > 0]) / e.sum()
    lp = np.array([d[i] - z if 0 <= i < len(x) else 0.0 for i in ids])
    return lp, ent, order, d[order] - z
