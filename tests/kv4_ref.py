"""The paged cache of 4-bit keys and values in plain numpy: its codes, its
layout, and causal attention over it in 64 bits (see citlali_hip_kv4_cache)."""
from __future__ import annotations

import numpy as np

GROUP, LIMIT = 32, 61440.0


def quantise(y):
    """(codes, d, m) of y [..., hd]; the definition's fp32 steps."""
    y = np.clip(np.asarray(y, np.float32), np.float32(-LIMIT), np.float32(LIMIT))
    y = y.reshape(*y.shape[:-1], -1, GROUP)
    m = y.min(-1, keepdims=True).astype(np.float16)
    with np.errstate(invalid="ignore", divide="ignore"):
        d = ((y.max(-1, keepdims=True) - m.astype(np.float32)) * np.float32(1 / 15)).astype(np.float16)
        c = np.rint((y - m.astype(np.float32)) / d.astype(np.float32))
        code = np.where(d > 0, np.clip(np.nan_to_num(c), 0, 15), 0).astype(np.uint8)
    bad = np.isnan(m)
    return code, np.where(bad, np.float16(0), d), m


def values(code, d, m):
    """What codes stand for: d code + m rounded to fp16 once."""
    v = (d.astype(np.float64) * code + m.astype(np.float64)).astype(np.float16)
    return v.reshape(*v.shape[:-2], -1)


def head_layout(page, hd):
    """Byte offsets of a head's K codes, K params, V codes, V params and its size."""
    codes, params = page * hd // 2, page * hd // 8
    return 0, codes, codes + params, 2 * codes + params, 2 * (codes + params)


class Cache:
    """num_pages pages as raw bytes, with writes and reads of single slots."""

    def __init__(self, num_pages, page, kv, hd, fill=0):
        self.num_pages, self.page, self.kv, self.hd = num_pages, page, kv, hd
        self.size = head_layout(page, hd)[4]
        self.raw = np.full((num_pages, kv, self.size), fill, np.uint8)

    def _places(self, page, o):
        hd, (kc, kp, vc, vp, _) = self.hd, head_layout(self.page, self.hd)
        dim = np.arange(hd)
        g = np.arange(hd // GROUP)
        k_byte = kc + o * (hd // 2) + dim // 8 * 4 + dim % 2 * 2 + dim % 8 // 4
        k_bit = dim % 4 // 2 * 4
        v_byte = vc + (o // 4 * (hd // 4) + dim // 4) * 8 + o % 4 * 2 + dim % 4 // 2
        v_bit = dim % 2 * 4
        k_par = kp + o * (hd // 8) + g * 4                       # d, then m two bytes on
        v_par = vp + (o // 4 * (hd // GROUP) + g) * 16 + o % 4 * 2   # d, then m eight bytes on
        return k_byte, k_bit, v_byte, v_bit, k_par, v_par

    def write(self, slot, k, v):
        """k, v [kv][hd]"""
        page, o = divmod(int(slot), self.page)
        k_byte, k_bit, v_byte, v_bit, k_par, v_par = self._places(page, o)
        for x, byte, bit, par, gap in ((k, k_byte, k_bit, k_par, 2), (v, v_byte, v_bit, v_par, 8)):
            code, d, m = quantise(x)
            code, d, m = code.reshape(self.kv, -1), d[..., 0], m[..., 0]
            for j in range(self.kv):
                row = self.raw[page, j]
                for i in range(self.hd):
                    row[byte[i]] = (row[byte[i]] & (0xF0 >> bit[i])) | (code[j, i] << bit[i])
                for g, p in enumerate(par):
                    row[p:p + 2] = np.frombuffer(d[j, g].tobytes(), np.uint8)
                    row[p + gap:p + gap + 2] = np.frombuffer(m[j, g].tobytes(), np.uint8)

    def read(self, slot):
        """(k, v) [kv][hd] fp16"""
        page, o = divmod(int(slot), self.page)
        k_byte, k_bit, v_byte, v_bit, k_par, v_par = self._places(page, o)
        out = []
        for byte, bit, par, gap in ((k_byte, k_bit, k_par, 2), (v_byte, v_bit, v_par, 8)):
            code = (self.raw[page][:, byte] >> bit) & 15
            half = lambda at: (self.raw[page][:, at].astype(np.uint16)                     # noqa: E731
                               | (self.raw[page][:, at + 1].astype(np.uint16) << 8)).view(np.float16)[..., None]
            out.append(values(code.reshape(self.kv, -1, GROUP), half(par), half(par + gap)))
        return tuple(out)

    def fill_random(self, rng, big=1.0):
        """Every slot a random token, all at once (fast path of write)."""
        n, kv, page, hd = self.num_pages, self.kv, self.page, self.hd
        k = (rng.standard_normal((n, kv, page, hd)) * big).astype(np.float16)
        v = rng.standard_normal((n, kv, page, hd)).astype(np.float16)
        (ck, dk, mk), (cv, dv, mv) = quantise(k), quantise(v)
        u = ck.reshape(n, kv, page, hd // 8, 4, 2).swapaxes(-1, -2).reshape(n, kv, page, hd // 8, 4, 2)
        kc = (u[..., 0] | (u[..., 1] << 4)).reshape(n, kv, -1)
        kp = np.concatenate((dk, mk), -1).reshape(n, kv, -1).view(np.uint8)
        u = cv.reshape(n, kv, page // 4, 4, hd // 4, 2, 2).swapaxes(3, 4)
        vc = (u[..., 0] | (u[..., 1] << 4)).reshape(n, kv, -1)
        vp = np.ascontiguousarray(np.concatenate((dv, mv), -1).reshape(n, kv, page // 4, 4, hd // GROUP, 2)
                                  .transpose(0, 1, 2, 4, 5, 3)).reshape(n, kv, -1).view(np.uint8)
        self.raw = np.ascontiguousarray(np.concatenate((kc, kp, vc, vp), -1))
        shape = (n, kv, page, hd)
        self.k = values(ck, dk, mk).reshape(shape)
        self.v = values(cv, dv, mv).reshape(shape)
        return self


def attention(cache, q, query_start, lens, table, max_context=None, max_query=None):
    """(out, spread, reach) in 64 bits.  q [tokens][heads][hd]; rows nobody asks
    for are NaN.  spread = sum_t p_t |v_t| and reach = the largest sum_d |q_d
    k_d| / sqrt(hd) a row meets: what an error bound needs."""
    tokens, heads, hd = q.shape
    kv, page = cache.kv, cache.page
    g = heads // kv
    out = np.full(q.shape, np.nan)
    spread, reach = np.zeros(q.shape), np.zeros((tokens, heads, 1))
    for s, length in enumerate(lens):
        r0, r1 = int(query_start[s]), int(query_start[s + 1])
        n = r1 - r0
        length = max(0, int(length))
        cap = length if max_context is None else min(length, max_context)
        p = np.arange(max(0, cap))
        pages = np.asarray(table[s])[p // page] if len(p) else np.zeros(0, int)
        here = (pages >= 0) & (pages < cache.num_pages)
        at = np.where(here, pages, 0)
        k = cache.k[at, :, p % page].astype(np.float64)      # [pos][kv][hd]
        v = cache.v[at, :, p % page].astype(np.float64)
        for i in range(n if max_query is None else min(n, max_query)):
            seen = here & (p < length - n + i + 1)
            for h in range(heads):
                kk, vv = k[seen, h // g], v[seen, h // g]
                if not len(kk):
                    out[r0 + i, h] = 0
                    continue
                qq = q[r0 + i, h].astype(np.float64)
                x = kk @ qq / np.sqrt(hd)
                w = np.exp(x - x.max())
                w /= w.sum()
                out[r0 + i, h] = w @ vv
                spread[r0 + i, h] = w @ np.abs(vv)
                reach[r0 + i, h] = (np.abs(kk) @ np.abs(qq)).max() / np.sqrt(hd)
    return out, spread, reach


def tolerance(out, spread, reach):
    """How far fp16 outputs may be off: their own rounding (2^-11), weights
    rounded to fp16 against weights summed before it (2^-11 of sum p |v|, 2^-10
    with the sum's), and scores of at most 128 fp32 additions and a few
    multiplications (2^-17 of their terms, 2^-21 on the exponential), which
    change a weight by twice their size against the others."""
    score = reach * 2.0 ** -16 + 2.0 ** -20
    return np.abs(out) * 2.0 ** -11 + spread * (2.0 ** -10 + 2 * score) + 2.0 ** -24
