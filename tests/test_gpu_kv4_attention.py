"""Causal attention over the paged cache of 4-bit keys and values, against
numpy in 64 bits over the values the codes stand for.  Bar: kv4_ref.tolerance."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref

pytestmark = pytest.mark.gpu


class Batch:
    def __init__(self, hip, seed, heads, kv, hd, page, lens, asked=None, spare=2, big=1.0, behind=0):
        rng = np.random.default_rng(seed)
        self.hip, self.heads, self.kv, self.hd, self.page = hip, heads, kv, hd, page
        self.lens = np.array(lens, np.int32)
        need = [max(0, -(-int(n) // page)) for n in lens]
        self.cache = kv4_ref.Cache(sum(need) + spare, page, kv, hd).fill_random(rng, big)
        order = rng.permutation(self.cache.num_pages)
        self.wide = max(need + [1]) + 1
        self.table = np.full((len(lens), self.wide), -7, np.int32)      # entries no position uses
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.single = asked is None
        self.start = np.concatenate(([0], np.cumsum(asked if asked is not None else [1] * len(lens)))).astype(np.int32)
        self.tokens = int(self.start[-1]) + behind
        self.max_query = max([1] + list(asked or []))
        self.max_context = max(1, int(self.lens.max()))
        self.q = rng.standard_normal((self.tokens, heads, hd)).astype(np.float16)

    def upload(self):
        up = self.hip.DeviceArray.from_numpy
        self.d_raw, self.d_lens, self.d_table, self.d_start = (up(x) for x in (self.cache.raw, self.lens, self.table,
                                                                              self.start))
        row = self.heads * self.hd
        self.q_stride, self.o_stride = row + 8, row + 24
        q = np.zeros((max(1, self.tokens), self.q_stride), np.float16)
        q[:self.tokens, :row] = self.q.reshape(self.tokens, row)
        self.d_q = up(q)
        self.d_out = up(np.full((max(1, self.tokens), self.o_stride), 7, np.float16))
        self.view = self.hip.device.kv4_cache(self.d_raw, self.cache.num_pages, self.page, self.kv, self.hd)
        self.bytes = self.hip.device.kv4_attention_workspace_bytes(self.max_context, self.max_query, len(self.lens),
                                                                   self.tokens, self.heads, self.kv, self.hd)
        self.d_ws = up(np.full(max(16, self.bytes), 0xFF, np.uint8))     # NaN where it is read before it is written
        return self

    def launch(self, workspace=None):
        self.hip.device.kv4_attention(self.view, self.d_q, self.q_stride, None if self.single else self.d_start,
                                      self.d_lens, self.d_table, self.wide, len(self.lens), self.tokens,
                                      self.max_query, self.max_context, self.heads,
                                      self.d_ws if workspace is None else workspace, self.bytes, self.d_out,
                                      self.o_stride)
        return self

    def result(self):
        row = self.heads * self.hd
        out = self.d_out.download(np.float16, self.tokens * self.o_stride).reshape(self.tokens, self.o_stride)
        assert (out[:, row:] == 7).all()
        return out[:, :row].reshape(self.tokens, self.heads, self.hd)

    def expected(self):
        return kv4_ref.attention(self.cache, self.q, self.start, self.lens, self.table, self.max_context,
                                 self.max_query)

    def check(self):
        got = self.result()
        want, spread, reach = self.expected()
        asked = ~np.isnan(want[:, 0, 0])
        assert (got[~asked] == 7).all()                                   # rows nobody asks for
        got, want = got[asked].astype(np.float64), want[asked]
        off = np.abs(got - want) - kv4_ref.tolerance(want, spread[asked], reach[asked])
        assert np.isfinite(got).all() and (off <= 0).all(), (np.isfinite(got).all(), off.max())
        return got


@pytest.mark.parametrize("page", [16, 32, 256])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 2), (16, 2)])
def test_decode(hip, heads, kv, hd, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 511, 700]
    Batch(hip, 1, heads, kv, hd, page, lens).upload().launch().check()


@pytest.mark.parametrize("group", range(1, 17))
def test_every_group(hip, group):
    Batch(hip, group, group * 2, 2, 128 if group % 2 else 64, 16, [77, 5]).upload().launch().check()


@pytest.mark.parametrize("lens", [[5000], [9000, 40, 1], [2049] * 3, [768, 513], [769, 256, 512], [20000]])
def test_long_contexts(hip, lens):
    Batch(hip, len(lens), 8, 2, 128, 64, lens).upload().launch().check()


def test_a_large_weight_beside_small_ones(hip):
    """Scores far apart: weights over the whole range of the exponential."""
    Batch(hip, 9, 8, 2, 128, 16, [300, 1500], big=12.0).upload().launch().check()


@pytest.mark.parametrize("heads,kv,hd,page,lens,asked", [
    (8, 2, 128, 16, [40, 17, 300], [3, 2, 4]),                # a few queries each
    (10, 2, 128, 16, [40, 700], [4, 1]),
    (8, 8, 64, 32, [130, 64, 90], [16, 9, 1]),
    (8, 2, 128, 16, [100], [100]),                            # whole prompts
    (4, 1, 64, 16, [257, 33, 1], [257, 33, 1]),
    (16, 2, 128, 64, [300, 129], [129, 65]),                  # chunks behind a prefix
    (6, 2, 128, 128, [513], [200]),
    (32, 2, 64, 16, [90, 20], [31, 20]),
    (5, 5, 128, 16, [70, 300], [70, 40]),
    (64, 32, 128, 16, [131, 66, 5, 90, 300], [130, 66, 5, 65, 33]),   # more workgroups than fit the CUs at once
    (64, 32, 64, 32, [131, 66, 5, 90, 300], [130, 66, 5, 65, 33]),
    (16, 2, 64, 32, [900, 500], [20, 9]),                     # chunks of a prompt's positions
    (32, 2, 128, 16, [900, 33, 5], [3, 3, 1]),                # 33 to 48 rows of a kv head
    (10, 2, 128, 64, [1300, 40], [8, 3]),
    (14, 2, 128, 16, [40, 7, 1300], [6, 7, 5]),               # 49 to 64
    (16, 2, 64, 32, [100, 2100, 5], [5, 4, 5]),
    (8, 2, 128, 128, [640, 64, 15], [16, 12, 15]),
    (3, 3, 64, 16, [900, 61], [64, 61])])
def test_several_queries(hip, heads, kv, hd, page, lens, asked):
    Batch(hip, sum(lens), heads, kv, hd, page, lens, asked, behind=3).upload().launch().check()


def test_sequences_without_positions_or_queries(hip):
    b = Batch(hip, 3, 8, 2, 128, 16, [0, 5, 33], asked=None).upload().launch()
    got = b.check()
    assert not got[0].any()
    Batch(hip, 4, 8, 2, 128, 16, [40, 40, 0, 40], asked=[0, 7, 0, 20]).upload().launch().check()


def test_lengths_below_zero_count_as_zero(hip):
    b = Batch(hip, 16, 8, 2, 128, 16, [0, 40, 0], asked=[2, 3, 40])
    b.lens[[0, 2]] = -1, -2 ** 31
    got = b.upload().launch().check()
    assert not got[:2].any() and got[2:5].any() and not got[5:].any()
    b = Batch(hip, 17, 8, 2, 64, 16, [0, 9000])
    b.lens[0] = -2 ** 31
    assert not b.upload().launch().check()[0].any()


def test_queries_before_the_first_position(hip):
    """More queries than positions: the first ones see nothing."""
    got = Batch(hip, 5, 4, 2, 64, 16, [3, 30], asked=[9, 30]).upload().launch().check()
    assert not got[:6].any() and got[6:].any()
    got = Batch(hip, 6, 4, 2, 128, 16, [2, 0], asked=[3, 2]).upload().launch().check()
    assert not got[0].any() and got[1:3].any() and not got[3:].any()


@pytest.mark.parametrize("asked", [None, [1, 6, 40]])
def test_slots_past_the_end_may_hold_anything(hip, asked):
    """NaN scales and codes behind every sequence's last position."""
    b = Batch(hip, 7, 8, 2, 128, 32, [1, 37, 95], asked)
    clean = b.upload().launch().check()
    live = np.zeros((b.cache.num_pages, b.page), bool)
    for s, n in enumerate(b.lens):
        for p in range(n):
            live[b.table[s, p // b.page], p % b.page] = True
    _, kp, _, vp, _ = kv4_ref.head_layout(b.page, b.hd)
    for page, o in np.argwhere(~live):
        g = b.hd // 32
        b.cache.raw[page, :, kp + o * g * 4:kp + (o + 1) * g * 4] = 0xFF
        for j in range(g):
            at = vp + (o // 4 * g + j) * 16 + o % 4 * 2
            b.cache.raw[page, :, at:at + 2] = 0xFF
            b.cache.raw[page, :, at + 8:at + 10] = 0xFF
    assert np.array_equal(b.upload().launch().check(), clean)


def _nan_tokens(b, where):
    """Makes K and V NaN in one group of dims at (sequence, position, group)."""
    _, kp, _, vp, _ = kv4_ref.head_layout(b.page, b.hd)
    g, nan = b.hd // 32, np.frombuffer(np.float16(np.nan).tobytes(), np.uint8)
    for s, p, j in where:
        page, o = b.table[s, p // b.page], p % b.page
        raw = b.cache.raw[page]
        k, v = kp + (o * g + j) * 4, vp + (o // 4 * g + j) * 16 + o % 4 * 2
        raw[:, k:k + 2], raw[:, k + 2:k + 4], raw[:, v:v + 2], raw[:, v + 8:v + 10] = 0, nan, 0, nan
        raw[:, o * b.hd // 2 + j * 16:o * b.hd // 2 + j * 16 + 16] = 0
        for w in range(8):
            at = kp + g * 4 * b.page + (o // 4 * (b.hd // 4) + j * 8 + w) * 8 + o % 4 * 2
            raw[:, at:at + 2] = 0
    return b


@pytest.mark.parametrize("hd,page", [(128, 16), (64, 64)])
@pytest.mark.parametrize("heads,kv,asked", [(8, 2, [4, 2, 3]), (8, 2, [8, 1, 5]), (8, 2, [10, 9, 12]),
                                            (8, 2, [12, 9, 16]),
                                            (8, 2, [70, 9, 200])])
def test_a_nan_is_kept_from_the_queries_before_it(hip, heads, kv, asked, hd, page):
    """NaN keys and values at positions that the last queries see and the first
    ones do not: the first ones' results are those of a cache without them."""
    lens = [80, 33, 700]
    b = Batch(hip, 18, heads, kv, hd, page, lens, asked)
    want, spread, reach = b.expected()         # of the cache without them
    near = kv4_ref.tolerance(want, spread, reach)
    first = [lens[s] - max(1, n // 2) for s, n in enumerate(asked)]    # the first NaN position
    _nan_tokens(b, [(s, p, (s + p) % (hd // 32)) for s in range(3) for p in range(first[s], lens[s], 3)])
    got = b.upload().launch().result()[:b.start[-1]].astype(np.float64)
    for s, n in enumerate(asked):
        sees = lens[s] - n + np.arange(n) + 1 > first[s]
        rows = slice(b.start[s], b.start[s + 1])
        assert sees.any() and np.isnan(got[rows][sees]).all()
        assert (np.abs(got[rows] - want[rows])[~sees] <= near[rows][~sees]).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("asked", [[4, 2], [70, 9]])
def test_nan_values_reach_their_dims_alone(hip, hd, asked):
    """Values (not keys) that are NaN in one group of dims."""
    lens = [80, 33]
    b = Batch(hip, 19, 8, 2, hd, 16, lens, asked)
    want, spread, reach = b.expected()
    near = kv4_ref.tolerance(want, spread, reach)
    keys = b.cache.raw.copy()
    where = [(0, 78, 1), (0, 79, 0), (1, 32, 1)]
    _nan_tokens(b, where)
    behind = kv4_ref.head_layout(16, hd)[2]
    b.cache.raw[:, :, :behind] = keys[:, :, :behind]
    got = b.upload().launch().result()[:b.start[-1]].astype(np.float64)
    nan = np.zeros((len(got), hd // 32), bool)
    for s, p, j in where:
        nan[b.start[s]:b.start[s + 1], j] |= lens[s] - asked[s] + np.arange(asked[s]) + 1 > p
    nan = np.repeat(nan, 32, axis=1)[:, None, :] & np.ones((1, 8, 1), bool)
    assert np.isnan(got[nan]).all() and (np.abs(got - want)[~nan] <= near[~nan]).all()


@pytest.mark.parametrize("asked", [None, [1, 6, 70]])
def test_pages_that_are_not_there(hip, asked):
    b = Batch(hip, 8, 8, 2, 128, 16, [20, 50, 90], asked)
    b.table[0, 0] = -1
    b.table[1, 1] = b.cache.num_pages
    b.table[2, :] = 1 << 30
    got = b.upload().launch().check()
    assert not got[-1].any() and got[0].any()


def test_bounds_of_the_plan(hip):
    """Positions past max_context and queries past max_query are not touched."""
    b = Batch(hip, 9, 8, 2, 128, 16, [300, 40])
    b.max_context = 100
    b.upload().launch().check()
    b = Batch(hip, 10, 8, 2, 64, 16, [60, 40], asked=[30, 4])
    b.max_query = 21
    b.upload().launch().check()
    b = Batch(hip, 11, 8, 2, 64, 16, [60, 40], asked=[3, 2])
    b.max_query = 2
    b.upload().launch().check()


def test_prefixes_share_pages(hip):
    b = Batch(hip, 12, 8, 2, 128, 16, [64, 64, 80])
    b.table[1, :3] = b.table[0, :3]
    b.table[2, :4] = b.table[0, :4]
    b.upload().launch().check()


def test_two_graphs_and_eager_calls(hip):
    """Two captured calls with a workspace each, replayed in turn with eager
    calls between, give the eager results every time."""
    stream = hip.device.Stream()
    hip.device.set_stream(stream)
    try:
        batches = [Batch(hip, 13, 8, 2, 128, 16, [900, 20, 333]).upload(),
                   Batch(hip, 14, 8, 2, 64, 32, [600, 100], asked=[40, 3]).upload()]
        want = [b.launch().check() for b in batches]
        graphs = [hip.device.Graph.capture(b.launch) for b in batches]
        for _ in range(3):
            for b in batches:
                b.d_out.zero()
                b.d_out.upload(np.full((b.tokens, b.o_stride), 7, np.float16))
            for g in graphs:
                g.launch()
            for b, w in zip(batches, want):
                assert np.array_equal(b.check(), w)
            batches[0].launch()
            assert np.array_equal(batches[0].check(), want[0])
        for g in graphs:
            g.close()
        hip.synchronize()
    finally:
        hip.device.set_stream(None)
        stream.close()


def test_pages_past_four_gigabytes(hip):
    page, kv, hd = 256, 8, 128
    b = Batch(hip, 15, 16, kv, hd, page, [300], spare=0).upload()
    size = hip.device.kv4_page_bytes(page, kv, hd)
    num = (1 << 32) // size + 9
    pages = hip.DeviceArray(num * size)
    for i in range(b.cache.num_pages):
        pages.upload(b.cache.raw[i], (num - 1 - i) * size)
    want = b.launch().check()
    b.view = hip.device.kv4_cache(pages, num, page, kv, hd)
    b.d_table = hip.DeviceArray.from_numpy(np.where(b.table >= 0, num - 1 - b.table, -1).astype(np.int32))
    assert np.array_equal(b.launch().check(), want)


@pytest.mark.parametrize("hd,asked", [(64, None), (128, None), (128, [40, 30]), (64, [40, 33])])
def test_infinite_queries(hip, hd, asked):
    """Scores that are all -inf give zeros, +inf among them NaN; other rows keep theirs."""
    b = Batch(hip, 20, 4, 2, hd, 16, [40, 33], asked)
    want, spread, reach = b.expected()
    sign = np.sign(b.cache.k[..., 5].astype(np.float64))
    b.q[0, 1] = 0
    b.q[0, 1, 5] = -np.inf
    b.q[-1, 2] = 0
    pages = b.table[0, :3]
    raw = kv4_ref.Cache(b.cache.num_pages, 16, 2, hd)
    raw.raw, raw.k, raw.v = b.cache.raw, b.cache.k, b.cache.v
    for p in range(40):                                        # sequence 0, kv head 0: dim 5 of every key above 0
        k, v = raw.read(pages[p // 16] * 16 + p % 16)
        k = np.abs(k.astype(np.float32)) + np.float32(0.5) if p or asked is None else k.astype(np.float32)
        raw.write(pages[p // 16] * 16 + p % 16, k, v.astype(np.float32))
    got = b.upload().launch().result()[:b.start[-1]].astype(np.float64)
    if asked is None:
        assert not got[0, 1].any()                             # every score -inf
    else:
        first = sign[pages[0], 0, 0]                           # the first row sees position 0 alone
        assert not got[0, 1].any() if first > 0 else np.isnan(got[0, 1]).all()
    seen = b.cache.v[b.table[1, np.arange(33) // 16], 1, np.arange(33) % 16].astype(np.float64)
    near = np.abs(seen).mean(0) * 2.0 ** -9 + 2.0 ** -20
    assert (np.abs(got[-1, 2] - seen.mean(0)) <= near).all()   # equal scores
    off = np.abs(got - want) - kv4_ref.tolerance(want, spread, reach)
    other = np.ones(got.shape[:2], bool)
    other[0], other[-1, 2] = False, False
    if asked is None:
        assert (off[other] <= 0).all()
    else:                                                      # sequence 1, whose keys are as they were
        assert (off[40:][other[40:]] <= 0).all()


@pytest.mark.parametrize("hd,big", [(64, 3000.0), (128, 3000.0), (128, 40000.0)])
@pytest.mark.parametrize("heads,kv,lens,asked", [
    (8, 2, [300, 37], None), (8, 2, [5000], None),           # one query: in one chunk, in several
    (8, 2, [700, 60], [8, 3]), (32, 2, [900, 33], [3, 2]),   # 17 to 48 rows
    (16, 2, [900, 500], [20, 9]),                            # a prompt's positions in chunks
    (8, 8, [300], [200])])                                   # and in two parts
def test_scores_of_large_queries_and_keys(hip, heads, kv, lens, asked, hd, big):
    """Finite queries and keys whose scores lie far beyond 2^20: a row whose
    largest score leads the next by more than the scores' own rounding (2^-16
    of their terms, both ways, and 30 for the exponential) is the value of that
    position: half a step for the weight, half for the output."""
    with np.errstate(over="ignore"):                         # infinities saturate
        b = Batch(hip, 21, heads, kv, hd, 16, lens, asked, big=big)
        b.q = np.clip(b.q.astype(np.float32) * big, -65504, 65504).astype(np.float16)
    got = b.upload().launch().result().astype(np.float64)
    assert np.isfinite(got).all()
    tested = 0
    for s, length in enumerate(lens):
        n = b.start[s + 1] - b.start[s]
        p = np.arange(length)
        k, v = (x[b.table[s, p // 16], :, p % 16].astype(np.float64) for x in (b.cache.k, b.cache.v))
        for i in range(n):
            seen = length - n + i + 1
            for h in range(heads):
                q = b.q[b.start[s] + i, h].astype(np.float64)
                x = k[:seen, h // (heads // kv)] @ q / np.sqrt(hd)
                reach = (np.abs(k[:seen, h // (heads // kv)]) @ np.abs(q)).max() / np.sqrt(hd)
                best = x.argmax()
                if seen > 1 and np.delete(x, best).max() > x[best] - 2 * reach * 2.0 ** -16 - 30:
                    continue
                tested += 1
                want = v[best, h // (heads // kv)]
                assert (np.abs(got[b.start[s] + i, h] - want) <= np.abs(want) * 2.0 ** -10 + 2.0 ** -24).all()
    assert tested >= 0.9 * heads * b.start[-1]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv,lens,asked", [
    (16, 2, [200, 40], None), (16, 2, [1500], None),         # one query: in one chunk, in several
    (16, 2, [200], [4]), (16, 1, [200, 90], [3, 3]),         # 17 to 48 rows
    (16, 2, [200], [20]), (8, 8, [300], [200])])             # prompts: in chunks, in two parts
def test_equal_values_come_out_as_they_are(hip, heads, kv, lens, asked, hd):
    """Every position has the same value and the weights are of two kinds: what
    rounding does to them is in the numerator and in their sum alike, so the
    value comes out to the bit (fp32 sums of at most 1500 terms are off by less
    than 2^-13, half a step is at least 2^-12 of the value)."""
    b = Batch(hip, 22, heads, kv, hd, 16, lens, asked)
    rng = np.random.default_rng(22)
    b.cache.raw[:] = 0
    value = np.repeat(1.999 - np.arange(kv * hd // 32) / (kv * hd // 32), 32).reshape(kv, hd).astype(np.float16)
    key = np.zeros((kv, hd), np.float32)
    for s, length in enumerate(lens):
        for p in range(length):
            key[:, :32] = 0 if p % 97 else 1                 # a group of one value is kept as it is
            b.cache.write(b.table[s, p // 16] * 16 + p % 16, key, value)
    b.q[:] = 0
    b.q[..., 0] = rng.uniform(2, 40, b.q.shape[:2])          # weights 1 and e^(-q / sqrt(hd)), e^-0.2 to e^-5
    got = b.upload().launch().result()
    want = np.repeat(value, heads // kv, axis=0)
    assert np.array_equal(got, np.broadcast_to(want, got.shape))


@pytest.mark.parametrize("nseq", [33, 49])                   # two parts of the positions, one
@pytest.mark.parametrize("hd,page,lens", [(64, 16, [3300, 1030, 2049]), (128, 16, [2500, 1100]),
                                          (64, 32, [2300, 4200]), (128, 64, [4500])])
def test_long_prompts_in_one_chunk(hip, nseq, hd, page, lens):
    """A prompt kernel's chunk of more pages than the lanes hold at once (64), of
    shuffled pages, more than twice as many too; sequences enough for no split."""
    asked = [60, 49, 60][:len(lens)]
    short = nseq - len(lens)
    b = Batch(hip, 23, 8, 8, hd, page, lens + [40] * short, asked + [2] * short).upload()
    assert b.bytes == 0 and max(lens) > 64 * page
    b.launch().check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("keys", [False, True])
def test_nan_in_two_parts_of_the_positions(hip, hd, keys):
    """As the two tests above, where two groups of waves share the positions."""
    lens, asked = [300, 290], [200, 65]
    b = Batch(hip, 24, 8, 8, hd, 16, lens, asked)
    want, spread, reach = b.expected()
    near = kv4_ref.tolerance(want, spread, reach)
    clean = b.cache.raw.copy()
    where = [(0, 150, 0), (0, 200, 1), (0, 259, 0), (0, 299, 1), (1, 255, 1), (1, 288, 0)]
    _nan_tokens(b, where)
    if not keys:
        behind = kv4_ref.head_layout(16, hd)[2]
        b.cache.raw[:, :, :behind] = clean[:, :, :behind]
    got = b.upload().launch().result().astype(np.float64)
    assert b.bytes == 0
    nan = np.zeros((len(got), hd // 32), bool)
    for s, p, j in where:
        nan[b.start[s]:b.start[s + 1], slice(None) if keys else j] |= (
            lens[s] - asked[s] + np.arange(asked[s]) + 1 > p)[(slice(None),) + (None,) * keys]
    nan = np.repeat(nan, 32, axis=1)[:, None, :] & np.ones((1, 8, 1), bool)
    assert nan.any() and not nan.all()
    assert np.isnan(got[nan]).all() and (np.abs(got - want)[~nan] <= near[~nan]).all()


def test_a_bound_of_very_many_queries(hip):
    """A plan whose row tiles pass one dimension of a grid."""
    b = Batch(hip, 25, 16, 1, 64, 16, [130, 9], asked=[120, 2])
    b.max_query = 270000
    b.upload().launch().check()
