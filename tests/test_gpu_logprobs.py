"""Log probabilities, ranks, entropies and alternatives per row of logits,
against numpy in 64 bits.

Bar: ids and ranks equal.  A log probability is x - m - log s with at most two
roundings of its size and log s (2^-23 of |x - m| + log s), and s, a sum of n
exponentials that are 2^-21 off each (an argument of size y is 2^-24 y off, which
counts y exp(-y) <= 1/e), in chains of at most n / 1024 additions and 24 levels;
the entropy adds the same error to sum e^y y / s, at most log n."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _want(x, tokens, k):
    x = x.astype(np.float64)
    n = x.shape[1]
    order = np.lexsort((np.broadcast_to(np.arange(n), x.shape), -np.where(np.isnan(x), -np.inf, x)), -1)
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(-1, keepdims=True)
        y = x - m
        e = np.exp(y)
        s = e.sum(-1, keepdims=True)
        lp = y - np.log(s)
        ent = np.log(s[:, 0]) - np.where(e > 0, e * y, 0).sum(-1) / s[:, 0]
    none = ~(m[:, 0] < np.inf) | (m[:, 0] == -np.inf)
    lp[none], ent[none] = np.nan, np.nan
    return lp, ent, order[:, :k]


def _run(hip, x, tokens, k, stride=None, shift=0, parts=("logprob", "rank", "entropy")):
    rows, vocab = x.shape
    stride = stride or vocab
    flat = np.full(shift + rows * stride + 8, 1e4, x.dtype)          # a neighbour would win
    for r in range(rows):
        flat[shift + r * stride:shift + r * stride + vocab] = x[r]
    up = hip.DeviceArray.from_numpy
    d_x, d_t = up(flat), up(np.asarray(tokens, np.int32))
    out = {n: up(np.full(rows, 99, np.int32 if n == "rank" else np.float32)) for n in parts}
    d_ids, d_top = up(np.full(max(1, rows * k), 99, np.int32)), up(np.full(max(1, rows * k), 99, np.float32))
    size = hip.device.token_logprobs_workspace_bytes(rows, vocab, k)
    ws = up(np.full(max(16, size), 0xFF, np.uint8))
    hip.device.token_logprobs(d_x.ptr + shift * x.itemsize, "fp16" if x.dtype == np.float16 else "fp32", stride, rows,
                              vocab, d_t if out.keys() & {"logprob", "rank"} else None, out.get("logprob"),
                              out.get("rank"), out.get("entropy"), k, d_ids if k else None, d_top if k else None, ws,
                              size)
    get = {n: d.download(np.int32 if n == "rank" else np.float32) for n, d in out.items()}
    return get, d_ids.download(np.int32)[:rows * k].reshape(rows, k), d_top.download(np.float32)[:rows * k].reshape(rows, k)


def _check(hip, x, tokens, k, **kw):
    rows, vocab = x.shape
    got, ids, top = _run(hip, x, tokens, k, **kw)
    lp, ent, order = _want(x, tokens, k)
    err = (vocab / 1024 + 32) * 2.0 ** -24                           # of s, relative
    bound = lambda v: 2.0 ** -22 * (np.abs(v) + np.log(vocab) + 1) + err   # noqa: E731
    r = np.arange(rows)
    tokens = np.asarray(tokens)
    given = (tokens >= 0) & (tokens < vocab)
    at = np.where(given, tokens, 0)

    def near(a, b):
        same = (a == b) | (np.isnan(a) & np.isnan(b))
        with np.errstate(invalid="ignore"):
            assert (same | (np.abs(a - b) <= bound(b))).all(), np.nanmax(np.abs(a - b) - bound(b))

    if "logprob" in got:
        near(got["logprob"], np.where(given, lp[r, at], 0))
    if "rank" in got:
        xf = x.astype(np.float64)
        mine = xf[r, at][:, None]
        ahead = np.where(np.isnan(mine), ~np.isnan(xf), (xf > mine) | ((xf == mine) & (np.arange(vocab) < at[:, None])))
        assert np.array_equal(got["rank"], np.where(given, ahead.sum(-1), -1))
    if "entropy" in got:
        with np.errstate(invalid="ignore"):
            close = np.abs(got["entropy"] - ent) <= bound(ent) + err * (np.log(vocab) + 1)
        assert (close | (np.isnan(got["entropy"]) & np.isnan(ent))).all()
    listed = np.minimum((~np.isnan(x)).sum(-1), k)
    for i in range(rows):
        assert np.array_equal(ids[i, :listed[i]], order[i, :listed[i]]), (i, ids[i], order[i])
        assert (ids[i, listed[i]:] == -1).all() and (top[i, listed[i]:] == -np.inf).all()
        near(top[i, :listed[i]], lp[i, order[i, :listed[i]]])
    return got, ids, top


def _logits(rng, rows, vocab, half=False):
    x = rng.standard_normal((rows, vocab)) * 3
    return x.astype(np.float16 if half else np.float32)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (1, 5, 20), (3, 63, 64), (2, 64, 1), (5, 1000, 7), (1, 4097, 64),
                                         (7, 32003, 20), (1, 151936, 20), (40, 9999, 5)])
def test_rows(hip, rows, vocab, k, half):
    rng = np.random.default_rng(rows * 1000 + vocab)
    x = _logits(rng, rows, vocab, half)
    _check(hip, x, rng.integers(0, vocab, rows), k)


def test_many_rows(hip):
    rng = np.random.default_rng(1)
    _check(hip, _logits(rng, 700, 3001), rng.integers(0, 3001, 700), 3)


@pytest.mark.parametrize("half,shift,stride", [(False, 1, 1003), (False, 3, 1005), (True, 1, 1001), (True, 5, 1015),
                                              (True, 0, 1007), (False, 0, 1008)])
def test_rows_at_any_element(hip, half, shift, stride):
    rng = np.random.default_rng(shift + stride)
    _check(hip, _logits(rng, 6, 1001, half), rng.integers(0, 1001, 6), 9, shift=shift, stride=stride)


@pytest.mark.parametrize("half", [False, True])
def test_equal_logits_go_by_id(hip, half):
    kind = np.float16 if half else np.float32
    x = np.zeros((4, 5003), kind)
    x[1] = np.random.default_rng(2).integers(0, 4, 5003)
    x[2, 1::2] = -0.0
    x[3, 4000:4100] = 2
    _, ids, _ = _check(hip, x, [5002, 17, 4, 4050], 64)
    assert ids[0].tolist() == list(range(64)) and ids[2].tolist() == list(range(64))
    assert ids[3].tolist() == list(range(4000, 4064))


def test_ascending_and_descending_rows(hip):
    """Every next logit enters the list, or none after the first ones."""
    up = np.linspace(-20, 20, 40001, dtype=np.float32)
    _check(hip, np.stack((up, up[::-1])), [0, 0], 64)


def test_masked_tokens(hip):
    rng = np.random.default_rng(3)
    x = _logits(rng, 5, 20011)
    x[0, rng.random(20011) < 0.99] = -np.inf
    x[1, :] = -np.inf
    x[1, [7, 12000]] = 1.0, 2.0
    x[2, :] = -np.inf                                           # nothing can come
    x[3, 5000:] = np.finfo(np.float32).min
    x[4, 11] = 300.0                                            # one token takes it all
    got, ids, top = _check(hip, x, [3, 7, 5, 19999, 11], 12)
    assert np.isnan(got["logprob"][2]) and np.isnan(got["entropy"][2])
    assert got["logprob"][4] == 0 and got["rank"][4] == 0 and abs(got["entropy"][4]) < 1e-30
    assert (top[1, 2:] == -np.inf).all() and ids[1, :2].tolist() == [12000, 7]


def test_rows_that_are_no_distribution(hip):
    rng = np.random.default_rng(4)
    x = _logits(rng, 5, 3000)
    x[0, 1234] = np.nan
    x[1, 77] = np.inf
    x[2, :] = np.nan
    x[3, 5:] = np.nan
    x[4, 2999], x[4, 0] = np.inf, -np.inf
    got, ids, _ = _check(hip, x, [1234, 5, 0, 2, 2999], 8)
    assert np.isnan(got["logprob"]).all() and np.isnan(got["entropy"]).all()
    assert ids[1, 0] == 77 and ids[4, 0] == 2999 and (ids[2] == -1).all()


@pytest.mark.parametrize("half", [False, True])
def test_signalling_nans_hide_no_logit(hip, half):
    """NaN logits of any kind beside the largest ones: the ids stay ordered."""
    rng = np.random.default_rng(8)
    x = _logits(rng, 6, 9001, half)
    bits = x.view(np.uint16 if half else np.uint32)
    for r, nan in enumerate((0x7c01, 0xfdff, 0x7e00) if half else (0x7f800001, 0xffbfffff, 0x7fc00000)):
        bits[r, rng.random(9001) < 0.5] = nan
        bits[r + 3, 1::2] = nan
    _check(hip, x, [5, 6, 7, 8, 9, 10], 40)
    many = np.tile(x.view(bits.dtype), (171, 1)).view(x.dtype)        # a wave has several steps of a row
    _check(hip, many, rng.integers(0, 9001, len(many)), 40)


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (9, 32000), (1100, 5000)])
def test_equal_logits_over_a_row_in_pieces(hip, rows, vocab):
    """A handful of values, so that waves and pieces end on equal logits; most
    of the row at -inf or at the type's lowest value in others."""
    rng = np.random.default_rng(vocab)
    x = rng.integers(0, 3, (rows, vocab)).astype(np.float32)
    x[0, rng.random(vocab) < 0.5] = 0
    if rows > 1:
        x[1] = np.finfo(np.float32).min
        x[2] = -np.inf
        x[2, rng.integers(0, vocab, 30)] = 1.5
        x[3, :] = -np.inf
        x[3, -70:] = 4
        x[4, rng.random(vocab) < 0.999] = -np.inf
        x[5, : vocab // 2] = 5
        x[6, vocab // 2:] = 5
    _check(hip, x, rng.integers(0, vocab, rows), 64)
    _check(hip, x.astype(np.float16) if rows == 1 else x, rng.integers(0, vocab, rows), 3)


def test_rows_without_a_token(hip):
    rng = np.random.default_rng(5)
    got, _, _ = _check(hip, _logits(rng, 4, 500), [-1, 499, 500, -2 ** 31], 2)
    assert got["logprob"][[0, 2, 3]].tolist() == [0, 0, 0] and got["rank"][[0, 2, 3]].tolist() == [-1, -1, -1]


@pytest.mark.parametrize("parts,k", [(("logprob",), 0), (("rank",), 0), (("entropy",), 0), ((), 4),
                                    (("logprob", "rank", "entropy"), 0)])
def test_outputs_that_are_not_asked_for(hip, parts, k):
    rng = np.random.default_rng(6)
    _check(hip, _logits(rng, 3, 6001), [5, 6, 7], k, parts=parts)


def test_captured(hip):
    """A captured call, replayed on new logits with eager calls between."""
    rng = np.random.default_rng(7)
    rows, vocab, k = 3, 30011, 10
    up = hip.DeviceArray.from_numpy
    stream = hip.device.Stream()
    hip.device.set_stream(stream)
    try:
        d_x, d_t = hip.DeviceArray(rows * vocab * 4), up(np.array([4, 5, 6], np.int32))
        lp, en, rk = (hip.DeviceArray(rows * 4) for _ in range(3))
        ids, top = (hip.DeviceArray(rows * k * 4) for _ in range(2))
        size = hip.device.token_logprobs_workspace_bytes(rows, vocab, k)
        ws = hip.DeviceArray(max(16, size))
        call = lambda: hip.device.token_logprobs(d_x, "fp32", vocab, rows, vocab, d_t, lp, rk, en, k, ids, top,   # noqa: E731
                                                 ws, size)
        d_x.upload(_logits(rng, rows, vocab))
        graph = hip.device.Graph.capture(call)
        for _ in range(3):
            d_x.upload(_logits(rng, rows, vocab))
            call()
            want = [d.download(np.int32).copy() for d in (lp, en, rk, ids, top)]
            for d in (lp, en, rk, ids, top):
                d.zero()
            graph.launch()
            assert all(np.array_equal(d.download(np.int32), w) for d, w in zip((lp, en, rk, ids, top), want))
        graph.close()
        hip.synchronize()
    finally:
        hip.device.set_stream(None)
        stream.close()
