"""The paged cache of 4-bit keys and values: appending tokens (head norms,
rotation, codes) and reading slots, against numpy in 64 bits.

Bar: stored values equal the definition's exactly (keys are normed and rotated
in 64 bits, so a code is the one next to the real number); queries, computed in
fp32 and rounded once, are off by half a step of fp16 (2^-11) plus 2^-19 of the
two normed values a rotation adds (a sum of 128 squares in seven levels and a
handful of roundings of 2^-24 each), or half the smallest step, 2^-25."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref

pytestmark = pytest.mark.gpu
THETA, EPS = 1e6, 1e-6


def _half(rng, *shape, big=False):
    x = rng.standard_normal(shape)
    if big:
        x = x * np.where(rng.random(shape[-1]) < 0.05, 20, 1)
    return x.astype(np.float16)


def _table(positions, hd):
    angle = np.arange(positions)[:, None] * THETA ** (-np.arange(0, hd, 2) / hd)
    return np.stack((np.cos(angle), np.sin(angle)), -1).astype(np.float32)


def _rotated(x, w, table, at):
    """(rotated, |n_i| + |n_partner|) of x [tokens][heads][hd] in 64 bits."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w.astype(np.float64)
    a, b = np.split(x, 2, -1)
    cos, sin = (table[at][:, None, :, i].astype(np.float64) for i in (0, 1))
    size = np.abs(a) + np.abs(b)
    return np.concatenate((a * cos - b * sin, a * sin + b * cos), -1), np.concatenate((size, size), -1)


class Step:
    """One append: host data, device copies, expected results."""

    def __init__(self, hip, rng, tokens, heads, kv, hd, page, norm=True, positions=300, gap=0, num_pages=None):
        self.hip, self.dims = hip, (tokens, heads, kv, hd)
        self.width = (heads + 2 * kv) * hd + gap
        self.qkv = _half(rng, tokens, self.width, big=True)
        self.q_norm, self.k_norm = ((1 + 0.3 * rng.standard_normal(hd)).astype(np.float16) if norm else None
                                    for _ in range(2))
        self.table = _table(positions, hd)
        self.at = rng.integers(0, positions, tokens).astype(np.int32)
        self.cache = kv4_ref.Cache(num_pages or tokens // page + 2, page, kv, hd, fill=0x5A)
        self.slots = rng.permutation(self.cache.num_pages * page)[:tokens].astype(np.int32)

    def run(self, q_stride=None, in_place=False):
        hip, (tokens, heads, kv, hd) = self.hip, self.dims
        up = lambda x: hip.DeviceArray.from_numpy(x) if x is not None else None    # noqa: E731
        self.d_qkv, self.d_pages = up(self.qkv), up(self.cache.raw)
        d_qn, d_kn, d_t, d_at, d_s = (up(x) for x in (self.q_norm, self.k_norm, self.table, self.at, self.slots))
        stride = self.width if in_place else heads * hd + 16
        d_out = self.d_qkv if in_place else up(np.full((max(1, tokens), stride), 7, np.float16))
        view = hip.device.kv4_cache(self.d_pages, self.cache.num_pages, self.cache.page, kv, hd)
        base = self.d_qkv.ptr
        hip.device.kv4_append(view, base if heads else None, base + 2 * heads * hd, base + 2 * (heads + kv) * hd,
                              self.width, self.width, d_qn, d_kn, EPS, d_t, len(self.table), d_at, d_s, tokens, heads,
                              d_out if heads else None, stride)
        self.q_out = d_out.download(np.float16, tokens * stride).reshape(tokens, stride)
        self.raw = self.d_pages.download(np.uint8).reshape(self.cache.raw.shape)
        d_k, d_v = (hip.DeviceArray(max(16, tokens * kv * hd * 2)) for _ in range(2))
        hip.device.kv4_read(view, d_s, tokens, d_k, d_v)
        self.k, self.v = (d.download(np.float16, tokens * kv * hd).reshape(tokens, kv, hd) for d in (d_k, d_v))
        return self

    def check(self):
        tokens, heads, kv, hd = self.dims
        known = (self.at >= 0) & (self.at < len(self.table))
        kept = known & (self.slots >= 0) & (self.slots < self.cache.num_pages * self.cache.page)
        at = np.where(known, self.at, 0)
        x = self.qkv[:, :(heads + 2 * kv) * hd].reshape(tokens, -1, hd)
        want, size = _rotated(x[:, :heads], self.q_norm, self.table, at)
        got = self.q_out[:, :heads * hd].reshape(tokens, heads, hd).astype(np.float64)
        off = np.abs(got - want) - (np.abs(want) * 2.0 ** -11 + size * 2.0 ** -19 + 2.0 ** -25)
        assert (off[known] <= 0).all(), off[known].max()
        k = _rotated(x[:, heads:heads + kv], self.k_norm, self.table, at)[0].astype(np.float32)
        for t in np.flatnonzero(kept):
            self.cache.write(self.slots[t], k[t], x[t, heads + kv:])
        # every byte of the cache: what was stored, and nothing else touched
        wrong = np.argwhere(self.raw != self.cache.raw)
        assert not len(wrong), wrong[:5]
        for t in np.flatnonzero(kept):
            want_k, want_v = self.cache.read(self.slots[t])
            assert np.array_equal(self.k[t], want_k, equal_nan=True)
            assert np.array_equal(self.v[t], want_v, equal_nan=True)
        return known, kept


@pytest.mark.parametrize("tokens,heads,kv,hd,page,norm", [
    (1, 16, 8, 128, 16, True), (1, 32, 8, 128, 256, True), (3, 4, 4, 64, 16, True), (5, 40, 8, 128, 32, False),
    (9, 14, 2, 64, 64, True), (17, 3, 1, 128, 128, True), (64, 8, 8, 64, 16, False), (130, 8, 2, 128, 16, True)])
def test_append_and_read(hip, tokens, heads, kv, hd, page, norm):
    rng = np.random.default_rng(tokens * 100 + heads)
    known, kept = Step(hip, rng, tokens, heads, kv, hd, page, norm, gap=24).run().check()
    assert kept.all()


@pytest.mark.parametrize("hd", [64, 128])
def test_consecutive_slots_of_a_prompt(hip, hd):
    """A prompt's slots follow each other from an odd row on, over page ends."""
    step = Step(hip, np.random.default_rng(hd), 75, 4, 2, hd, 16, num_pages=7)
    step.slots = (np.arange(75) + 5).astype(np.int32)
    step.run().check()


def test_padded_rows_are_left_alone(hip):
    step = Step(hip, np.random.default_rng(2), 12, 4, 2, 128, 16)
    step.slots[[1, 5]] = [-1, step.cache.num_pages * 16]     # rotated, not stored
    step.at[[3, 4, 7]] = [-1, len(step.table), -2 ** 31]     # nothing at all
    step.run()
    known, kept = step.check()
    assert known.sum() == 9 and kept.sum() == 7
    assert (step.q_out[~known] == 7).all()
    assert (step.q_out[:, 4 * 128:] == 7).all()              # nothing behind the heads
    outside = (step.slots < 0) | (step.slots >= step.cache.num_pages * 16)
    assert not step.k[outside].any() and not step.v[outside].any()


def test_queries_in_place_in_a_fused_buffer(hip):
    step = Step(hip, np.random.default_rng(3), 21, 8, 2, 128, 32, gap=8).run(in_place=True)
    step.check()
    assert np.array_equal(step.q_out[:, 8 * 128:], step.qkv[:, 8 * 128:])


def test_keys_and_values_alone(hip):
    step = Step(hip, np.random.default_rng(4), 6, 0, 3, 64, 16).run()
    step.check()


def test_values_at_the_edges(hip):
    """Constant groups, ranges below fp16's steps, saturation, infinities, NaN."""
    step = Step(hip, np.random.default_rng(5), 8, 1, 1, 128, 16, norm=False)
    step.at[:] = 0                                            # no rotation
    rows = step.qkv[:, 128:].reshape(8, 2, 128)
    rows[0] = 0
    rows[1] = 1.25
    rows[2, :, ::2], rows[2, :, 1::2] = 1.0, 1.0 + 2.0 ** -10
    rows[3, :, :5] = 65504
    rows[3, :, 40:45] = -65504
    rows[4, :, 3], rows[4, :, 70] = np.inf, -np.inf
    rows[5, :, 33] = np.nan
    rows[6] = (np.arange(128) % 7) * 2.0 ** -24               # subnormal
    rows[7, :, 1:] = np.float16(-0.0)
    step.qkv[:, 128:] = rows.reshape(8, -1)
    step.run().check()
    assert np.isnan(step.k[5, 0, 32:64]).all() and np.isfinite(step.k[5, 0, :32]).all()
    assert np.isfinite(step.v[[0, 1, 2, 3, 4, 6, 7]]).all()


def test_slots_past_four_gigabytes(hip):
    """Byte offsets of late pages pass 32 bits."""
    page, kv, hd = 256, 8, 128
    size = hip.device.kv4_page_bytes(page, kv, hd)
    num = (1 << 32) // size + 40
    pages = hip.DeviceArray(num * size)
    view = hip.device.kv4_cache(pages, num, page, kv, hd)
    step = Step(hip, np.random.default_rng(6), 4, 1, kv, hd, page)
    slots = np.array([num * page - 1, num * page - 256, (num - 30) * page + 77, 3], np.int32)
    up = hip.DeviceArray.from_numpy
    d_qkv, d_t, d_at, d_s = up(step.qkv), up(step.table), up(step.at), up(slots)
    hip.device.kv4_append(view, None, d_qkv.ptr + 2 * hd, d_qkv.ptr + 2 * hd * (1 + kv), 0, step.width, None,
                          None, EPS, d_t, len(step.table), d_at, d_s, 4, 0, None, 0)
    d_k, d_v = (hip.DeviceArray(4 * kv * hd * 2) for _ in range(2))
    hip.device.kv4_read(view, d_s, 4, d_k, d_v)
    x = step.qkv.reshape(4, -1, hd)
    k = _rotated(x[:, 1:1 + kv], None, step.table, step.at)[0].astype(np.float32)
    assert np.array_equal(d_k.download(np.float16).reshape(4, kv, hd), kv4_ref.values(*kv4_ref.quantise(k)))
    assert np.array_equal(d_v.download(np.float16).reshape(4, kv, hd),
                          kv4_ref.values(*kv4_ref.quantise(x[:, 1 + kv:])))


@pytest.mark.parametrize("positions,hd,theta", [(1, 64, 1e4), (513, 128, 1e6), (40000, 64, 1e6)])
def test_rope_table(hip, positions, hd, theta):
    """Each number within half a step of fp32 (2^-25 at 1) and 64-bit noise."""
    d = hip.DeviceArray(positions * hd * 4)
    hip.device.rope_table(d, positions, hd, theta)
    got = d.download(np.float32).reshape(positions, hd // 2, 2)
    angle = np.arange(positions)[:, None] * float(np.float32(theta)) ** (-np.arange(0, hd, 2) / hd)
    want = np.stack((np.cos(angle), np.sin(angle)), -1)
    # the angle itself, at most 40000 and some roundings of 2^-53 off
    assert np.abs(got - want).max() <= 2.0 ** -25 + 40000 * 2.0 ** -50


@pytest.mark.parametrize("tokens,heads,kv,hd", [(2500, 32, 8, 128), (5003, 7, 3, 64), (9001, 4, 2, 128), (4099, 0, 5, 64)])
def test_many_tokens_equal_few_at_a_time(hip, tokens, heads, kv, hd):
    """Queries and every byte of the cache do not depend on the call's size."""
    rng = np.random.default_rng(tokens)
    s = Step(hip, rng, tokens, heads, kv, hd, 16)
    s.at[rng.integers(0, tokens, 30)] = -1
    row = heads * hd
    up = hip.DeviceArray.from_numpy
    d_qkv, d_qn, d_kn, d_t, d_at, d_s = (up(x) for x in (s.qkv, s.q_norm, s.k_norm, s.table, s.at, s.slots))
    got = []
    for step in (tokens, 97):
        d_pages, d_out = up(s.cache.raw), up(np.full((tokens, row + 8), 7, np.float16))
        view = hip.device.kv4_cache(d_pages, s.cache.num_pages, 16, kv, hd)
        for t in range(0, tokens, step):
            base = d_qkv.ptr + t * s.width * 2
            hip.device.kv4_append(view, base if heads else None, base + 2 * row, base + 2 * (row + kv * hd), s.width,
                                  s.width, d_qn, d_kn, EPS, d_t, len(s.table), d_at.ptr + 4 * t, d_s.ptr + 4 * t,
                                  min(step, tokens - t), heads, d_out.ptr + t * (row + 8) * 2 if heads else None,
                                  row + 8)
        got.append((d_pages.download(np.uint8), d_out.download(np.uint16)))
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])
    assert (got[0][0] != 0x5A).mean() > 0.5


@pytest.mark.parametrize("hd", [64, 128])
def test_infinities_under_a_norm(hip, hd):
    """A head with an infinity has an infinite root mean square: its finite dims
    become 0, the infinite one and its rotation partner NaN, in queries and (a
    group of 32 at a time) in keys."""
    step = Step(hip, np.random.default_rng(7), 9, 2, 2, hd, 16)
    x = step.qkv.reshape(9, 6, hd)
    x[2, :4, 3] = np.inf
    x[5, :4, hd // 2 + 1] = -np.inf
    x[7, :4, 0], x[7, :4, hd - 1] = np.inf, np.inf
    step.run()
    rows = [2, 5, 7]
    with np.errstate(invalid="ignore"):
        q, k = (_rotated(x[rows, lo:lo + 2], w, step.table, step.at[rows])[0]
                for lo, w in ((0, step.q_norm), (2, step.k_norm)))
    got = step.q_out[rows, :2 * hd].reshape(3, 2, hd)
    assert np.array_equal(np.isnan(got), np.isnan(q)) and np.isnan(q).sum() == 2 * (2 + 2 + 4)
    assert not got[~np.isnan(q)].any()
    want = kv4_ref.values(*kv4_ref.quantise(k.astype(np.float32)))
    assert np.array_equal(step.k[rows], want, equal_nan=True)
    finite = ~np.isnan(want)
    assert finite.any() == (hd == 128) and not step.k[rows][finite].any()
