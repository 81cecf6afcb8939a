"""Attention of trees of drafted tokens over the paged cache of 4-bit keys and
values, against numpy in 64 bits over the values the codes stand for.  Bar:
kv4_ref.tolerance, as for the causal attention whose products and sums it has."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref
import tree_ref
from test_gpu_kv4_attention import Batch, _nan_tokens

pytestmark = pytest.mark.gpu


class Trees(Batch):
    """A batch whose queries are the rows of a tree each; sees[s] as in tree_ref."""

    def __init__(self, hip, seed, heads, kv, hd, page, lens, asked, sees=None, max_query=None, **kw):
        super().__init__(hip, seed, heads, kv, hd, page, lens, asked, **kw)
        rng = np.random.default_rng(seed + 1000)
        self.sees = sees or [tree_ref.masks_of(tree_ref.tree(rng, n))[0] if n else np.zeros((0, 0), bool)
                             for n in asked]
        if max_query:
            self.max_query = max_query

    def upload(self):
        super().upload()
        self.bytes = self.hip.device.kv4_tree_attention_workspace_bytes(
            self.max_context, self.max_query, len(self.lens), self.tokens, self.heads, self.kv, self.hd)
        self.d_ws = self.hip.DeviceArray.from_numpy(np.full(max(16, self.bytes), 0xFF, np.uint8))
        words = -(-self.max_query // 64)
        masks = np.full((max(1, self.tokens), words), ~np.uint64(0))
        for s, see in enumerate(self.sees):
            n = min(len(see), self.max_query)
            # bits of rows that the sequence does not have are set: they name no position
            full = np.ones((n, words * 64), bool)
            full[:, :min(len(see), words * 64)] = see[:n, :words * 64]
            masks[self.start[s]:self.start[s] + n] = tree_ref.pack(full, words)
        self.d_masks = self.hip.DeviceArray.from_numpy(masks)
        return self

    def launch(self, workspace=None):
        self.hip.device.kv4_tree_attention(self.view, self.d_q, self.q_stride, None if self.single else self.d_start,
                                           self.d_lens, self.d_masks, self.d_table, self.wide, len(self.lens),
                                           self.tokens, self.max_query, self.max_context, self.heads,
                                           self.d_ws if workspace is None else workspace, self.bytes, self.d_out,
                                           self.o_stride)
        return self

    def expected(self):
        return tree_ref.attention(self.cache, self.q, self.start, self.lens, self.table, self.sees, self.max_context,
                                  self.max_query)


@pytest.mark.parametrize("hd,page", [(128, 16), (64, 32), (128, 256)])
@pytest.mark.parametrize("heads,kv,lens,asked", [
    (2, 2, [40, 9, 300], [1, 2, 16]),                 # up to 16 rows of a kv head
    (8, 2, [31, 64, 65], [3, 4, 1]),
    (8, 2, [100, 33, 700], [8, 7, 5]),                # up to 32
    (10, 2, [100, 9, 2000], [9, 9, 7]),               # up to 48
    (8, 2, [100, 90, 700], [30, 13, 20]),             # the prompt kernel, one tile of rows
    (10, 2, [300, 70, 1500], [60, 63, 64]),           # several
    (4, 2, [300, 70, 1500], [65, 70, 129]),           # masks of several words
    (6, 2, [256, 300, 999], [256, 255, 200]),
])
def test_trees(hip, heads, kv, lens, asked, hd, page):
    Trees(hip, 40, heads, kv, hd, page, lens, asked).upload().launch().check()


@pytest.mark.parametrize("asked,group", [([25, 3, 17], 2), ([32, 9, 1], 2), ([33, 24, 25], 2), ([40, 16, 8], 2),
                                         ([41, 40, 2], 2), ([16, 1, 4], 4), ([5, 2, 3], 16), ([80, 65, 17], 1),
                                         ([10, 2, 8], 8)])
def test_heads_of_64_have_up_to_80_rows_with_the_few(hip, asked, group):
    """Sequences with some of the column tiles beside the widest; short, with the tree
    across two chunks, and with slots whose values are NaN where a row is hidden."""
    for page, lens in ((16, [300, 40, 18]), (32, [1040, 1025, 2300]), (128, [5000, 790, 64])):
        Trees(hip, 60, 3 * group, 3, 64, page, lens, asked).upload().launch().check()
    b = Trees(hip, 61, 2 * group, 2, 64, 16, [90, 70, 800], asked)
    b.table[0, 1] = b.table[2, 3] = -1
    b.table[1, 0] = b.cache.num_pages
    b.upload().launch().check()
    b = Trees(hip, 62, 2 * group, 2, 64, 32, [90, 70, 800], asked)
    for s, see in enumerate(b.sees):
        see[::3] = False                      # rows that see the prefix alone
        b.lens[s] = max(len(see), b.lens[s])
    b.upload().launch().check()


@pytest.mark.parametrize("asked,group", [([16, 3, 9], 4), ([13, 12, 1], 4), ([33, 16, 17], 1), ([64, 32, 31], 1),
                                         ([32, 25, 8], 2), ([10, 9, 5], 5), ([8, 7, 1], 7)])
def test_heads_of_128_have_up_to_64_rows_in_half_a_tile(hip, asked, group):
    """One and two parts of the positions, chunks of them, sequences without pages in
    places and rows that see the prefix alone; some waves without a row."""
    for page, lens in ((16, [300, 80, 66]), (32, [100, 65, 190]), (64, [1040, 1025, 2300]), (256, [5000, 790, 64])):
        Trees(hip, 64, 3 * group, 3, 128, page, lens, asked).upload().launch().check()
    b = Trees(hip, 65, 2 * group, 2, 128, 16, [90, 70, 800], asked)
    b.table[0, 1] = b.table[2, 3] = -1
    b.table[1, 0] = b.cache.num_pages
    b.upload().launch().check()
    b = Trees(hip, 66, 2 * group, 2, 128, 32, [90, 70, 800], asked)
    for see in b.sees:
        see[::3] = False
    b.upload().launch().check()
    Trees(hip, 67, 2 * group, 2, 128, 16, [1, 0, 5], asked).upload().launch().check()   # more rows than positions
    rng = np.random.default_rng(2)
    many = [asked[0]] + [int(x) for x in rng.integers(0, asked[0] + 1, 69)]
    Trees(hip, 68, 2 * group, 2, 128, 16, [n + int(rng.integers(0, 90)) for n in many], many).upload().launch().check()


@pytest.mark.parametrize("hd,group,most", [(128, 2, 8), (128, 3, 10), (128, 4, 12), (128, 5, 16), (64, 2, 8),
                                           (64, 5, 6), (64, 2, 24), (64, 2, 32), (64, 5, 16)])
def test_more_workgroups_than_a_round(hip, hd, group, most):
    """Many short sequences, and some beside one of many chunks, at each number of
    column tiles and on the prompt kernel."""
    rng = np.random.default_rng(most)
    for seqs, kv, page, longest in ((90, 3, 16, 90), (20, 2, 32, 7000)):
        asked = [most] + [int(x) for x in rng.integers(0, most + 1, seqs - 1)]
        lens = [longest] + [n + int(rng.integers(0, 60)) for n in asked[1:]]
        Trees(hip, 63, kv * group, kv, hd, page, lens, asked).upload().launch().check()


@pytest.mark.parametrize("before", [0, 1, 15, 16, 31, 32, 33, 63, 64, 100, 127])
@pytest.mark.parametrize("asked", [[9], [40], [100]])
def test_trees_start_anywhere_in_a_tile(hip, before, asked):
    Trees(hip, 41, 4, 2, 128, 16, [before + n for n in asked], asked).upload().launch().check()


@pytest.mark.parametrize("group", range(1, 17))
def test_every_group(hip, group):
    Trees(hip, 42, 2 * group, 2, 64, 16, [70, 33], [7, 5]).upload().launch().check()


@pytest.mark.parametrize("asked", [[5, 3], [12, 9], [60, 20], [200, 100]])
def test_long_contexts(hip, asked):
    """Chunks of positions, the tree across the border of two of them in some."""
    for lens in ([5000, 1030], [2049, 2052], [9000, 9000 - 8]):
        Trees(hip, 43, 8, 2, 128, 64, lens, asked).upload().launch().check()


def test_chains_are_causal_attention(hip):
    """A chain's masks are the causal attention's: both are near the same numbers."""
    for asked in ([4, 4, 1], [11, 3, 8], [70, 64, 9]):
        lens = [80, 900, 9]
        chain = [np.tril(np.ones((n, n), bool)) for n in asked]
        trees = Trees(hip, 44, 8, 2, 128, 16, lens, asked, sees=chain)
        causal = Batch(hip, 44, 8, 2, 128, 16, lens, asked)
        assert np.array_equal(trees.expected()[0], causal.expected()[0])
        trees.upload().launch().check()
        causal.upload().launch().check()


def test_any_masks(hip):
    """Rows that see any of the others, later ones and not themselves too."""
    rng = np.random.default_rng(1)
    for asked, lens in (([9, 30], [20, 90]), ([100, 77], [100, 300])):
        sees = [rng.random((n, n)) < 0.3 for n in asked]
        Trees(hip, 45, 8, 2, 64, 16, lens, asked, sees=sees).upload().launch().check()


def test_rows_that_see_nothing(hip):
    """No position before the tree, and masks that are empty: zeros."""
    for n in (6, 40, 130):
        sees = np.eye(n, dtype=bool)
        sees[1::2] = False
        b = Trees(hip, 46, 8, 2, 128, 16, [n, n + 1], [n, n], sees=[sees, sees]).upload().launch()
        got = b.check()
        assert not got[1:n:2].any() and got[0:n:2].any() and got[n:].any()


def test_more_rows_than_positions(hip):
    """Rows whose own position is before the first: their bits name nothing."""
    for asked in ([9, 5], [40, 20]):
        b = Trees(hip, 47, 4, 2, 64, 16, [3, 0], asked).upload().launch()
        got = b.check()
        assert not got[asked[0]:].any()


def test_sequences_without_rows_or_positions(hip):
    Trees(hip, 48, 8, 2, 128, 16, [40, 40, 0, 40], [0, 7, 0, 20]).upload().launch().check()
    b = Trees(hip, 49, 8, 2, 128, 16, [0, 40, 0], [2, 3, 40])
    b.lens[[0, 2]] = -1, -2 ** 31
    got = b.upload().launch().check()
    assert not got[:2].any() and got[2:5].any() and not got[5:].any()


@pytest.mark.parametrize("asked", [[1, 6, 9], [1, 6, 40]])
def test_slots_past_the_end_may_hold_anything(hip, asked):
    b = Trees(hip, 50, 8, 2, 128, 32, [1, 37, 95], asked)
    clean = b.upload().launch().check()
    used = {(int(b.table[s, p // b.page]), p % b.page) for s, n in enumerate(b.lens) for p in range(n)}
    _, kp, _, vp, _ = kv4_ref.head_layout(b.page, b.hd)
    for page in range(b.cache.num_pages):
        for o in range(b.page):
            if (page, o) not in used:
                b.cache.raw[page, :, kp + o * 16:kp + (o + 1) * 16] = 0xFF
                for j in range(4):
                    at = vp + (o // 4 * 4 + j) * 16 + o % 4 * 2
                    b.cache.raw[page, :, at:at + 2] = b.cache.raw[page, :, at + 8:at + 10] = 0xFF
    assert np.array_equal(b.upload().launch().check(), clean)


@pytest.mark.parametrize("hd,page", [(128, 16), (64, 64)])
@pytest.mark.parametrize("heads,asked", [(8, [4, 2, 3]), (8, [8, 1, 5]), (8, [12, 9, 10]), (8, [30, 9, 16]),
                                         (4, [70, 9, 150]), (4, [40, 9, 26]), (8, [16, 9, 13]),
                                         (4, [32, 9, 17])])
@pytest.mark.parametrize("keys", [False, True])
def test_a_nan_is_kept_from_the_rows_that_do_not_see_it(hip, heads, asked, keys, hd, page):
    """Every third row of the tree has NaN values (and keys): the rows they are
    hidden from get the results of a cache without them, the others NaN."""
    lens = [80, 33, 700]
    b = Trees(hip, 51, heads, 2, hd, page, lens, asked)
    want, spread, reach = b.expected()
    near = kv4_ref.tolerance(want, spread, reach)
    nodes = [np.arange(1 if n > 1 else 0, n, 3) for n in asked]
    as_it_was = b.cache.raw.copy()
    _nan_tokens(b, [(s, lens[s] - asked[s] + j, j % (hd // 32)) for s in range(3) for j in nodes[s]])
    if not keys:
        behind = kv4_ref.head_layout(page, hd)[2]
        b.cache.raw[:, :, :behind] = as_it_was[:, :, :behind]
    got = b.upload().launch().result()[:b.start[-1]].astype(np.float64)
    for s, n in enumerate(asked):
        for i in range(n):
            r = b.start[s] + i
            dims = np.zeros(hd // 32, bool)
            for j in nodes[s]:
                dims[j % (hd // 32)] |= b.sees[s][i, j]
            nan = np.repeat(np.full(hd // 32, dims.any()) if keys else dims, 32)
            assert np.isnan(got[r][:, nan]).all()
            assert (np.abs(got[r] - want[r])[:, ~nan] <= near[r][:, ~nan]).all()


def test_infinities_in_hidden_rows(hip):
    """Codes of an infinite scale at tree rows that only themselves see."""
    for n in (8, 40):
        lens, asked = [60, 200], [n, n]
        b = Trees(hip, 52, 8, 2, 128, 16, lens, asked)
        for see in b.sees:                       # row 2 hidden from all but itself
            see[3:, 2] = False
        clean = b.upload().launch().check()
        _, kp, _, vp, _ = kv4_ref.head_layout(16, 128)
        inf = np.frombuffer(np.float16(np.inf).tobytes(), np.uint8)
        for s in range(2):
            p = lens[s] - n + 2
            page, o = b.table[s, p // 16], p % 16
            b.cache.raw[page, :, kp + o * 16 + 2:kp + o * 16 + 4] = inf
        got = b.upload().launch().result()
        for s in range(2):
            rows = np.delete(np.arange(n), 2) + b.start[s]
            assert np.array_equal(got[rows], clean.astype(np.float16)[rows])


def test_pages_that_are_not_there(hip):
    for asked in ([1, 6, 9], [20, 40, 70]):
        b = Trees(hip, 53, 8, 2, 128, 16, [20, 50, 90], asked)
        b.table[0, 0] = -1
        b.table[1, 1] = b.cache.num_pages
        b.table[2, :] = 1 << 30
        got = b.upload().launch().check()
        assert not got[-1].any()


def test_bounds_of_the_plan(hip):
    """Positions past max_context, rows past max_query, rows behind the last sequence."""
    for asked, most in (([30, 4], 21), ([3, 2], 2), ([100, 90], 64), ([100, 90], 65)):
        Trees(hip, 54, 8, 2, 64, 16, [160, 140], asked, max_query=most, behind=3).upload().launch().check()
    b = Trees(hip, 55, 8, 2, 128, 16, [300, 40], [9, 9])
    b.max_context = 100
    b.upload().launch().check()
    b = Trees(hip, 55, 8, 2, 128, 16, [300, 40], [40, 40])
    b.max_context = 295                          # within the tree
    b.upload().launch().check()


@pytest.mark.parametrize("asked", [[3], [16], [40]])
def test_pages_past_four_gigabytes(hip, asked):
    page, kv, hd = 256, 8, 128
    b = Trees(hip, 69, 32, kv, hd, page, [400], asked, spare=0).upload()
    size = hip.device.kv4_page_bytes(page, kv, hd)
    num = (1 << 32) // size + 9
    pages = hip.DeviceArray(num * size)
    for i in range(b.cache.num_pages):
        pages.upload(b.cache.raw[i], (num - 1 - i) * size)
    want = b.launch().check()
    b.view = hip.device.kv4_cache(pages, num, page, kv, hd)
    b.d_table = hip.DeviceArray.from_numpy(np.where(b.table >= 0, num - 1 - b.table, -1).astype(np.int32))
    assert np.array_equal(b.launch().check(), want)


def test_one_row_each(hip):
    """No query_start: one row a sequence, and a mask that hides its own position."""
    b = Trees(hip, 56, 8, 2, 128, 16, [40, 1, 9], [1, 1, 1])
    b.single = True
    b.sees[0] = b.sees[1] = np.zeros((1, 1), bool)
    got = b.upload().launch().check()
    assert got[0].any() and not got[1].any()


def test_two_graphs_and_eager_calls(hip):
    """Two captured calls with a workspace each, on a stream of their own, replayed
    in turn with eager calls between and with other masks and lengths."""
    stream = hip.device.Stream()
    hip.device.set_stream(stream)
    try:
        batches = [Trees(hip, 57, 8, 2, 128, 16, [900, 20, 333], [9, 4, 12]).upload(),
                   Trees(hip, 58, 8, 2, 64, 32, [1600, 100], [60, 31]).upload()]
        want = [b.launch().check() for b in batches]
        graphs = [hip.device.Graph.capture(b.launch) for b in batches]
        for turn in range(3):
            for b in batches:
                b.d_out.upload(np.full((b.tokens, b.o_stride), 7, np.float16))
            for g in graphs:
                g.launch()
            for b, w in zip(batches, want):
                assert np.array_equal(b.check(), w)
            batches[0].launch()
            assert np.array_equal(batches[0].check(), want[0])
        b = batches[0]
        b.lens = np.array([850, 19, 12], np.int32)
        b.sees = [np.tril(np.ones((n, n), bool)) for n in (9, 4, 12)]
        b.d_lens.upload(b.lens)
        b.d_masks.upload(np.concatenate([tree_ref.pack(s, 1) for s in b.sees]))
        graphs[0].launch()
        b.check()
        for g in graphs:
            g.close()
        hip.synchronize()
    finally:
        hip.device.set_stream(None)
        stream.close()


# column tiles of the few rows' kernel, by eight waves and by four, and the prompt kernel
KERNELS = [(8, 2, [300, 37, 5000], [3, 4, 2]), (8, 2, [700, 60], [8, 3]), (10, 2, [900, 33], [9, 7]),
           (8, 2, [1500, 300], [14, 9]), (8, 2, [90, 300], [20, 9]), (16, 2, [900, 500], [20, 9]), (8, 8, [300], [200]),
           (16, 8, [300] + [40] * 39, [5] * 40), (32, 8, [70] * 36, [8] * 36), (40, 8, [300] + [40] * 34, [9] * 35)]


def _seen(b, s, i):
    """Positions that row i of sequence s sees."""
    before = int(b.lens[s]) - len(b.sees[s])
    return np.concatenate((np.arange(before), before + np.flatnonzero(b.sees[s][i])))


@pytest.mark.parametrize("hd,big", [(64, 3000.0), (128, 3000.0), (128, 40000.0)])
@pytest.mark.parametrize("heads,kv,lens,asked", KERNELS)
def test_scores_of_large_queries_and_keys(hip, heads, kv, lens, asked, hd, big):
    """Finite queries and keys whose scores lie far beyond 2^20: a row whose
    largest score leads the next by more than the scores' own rounding (2^-16
    of their terms, both ways, and 30 for the exponential) is the value of that
    position: half a step for the weight, half for the output."""
    with np.errstate(over="ignore"):                         # infinities saturate
        b = Trees(hip, 70, heads, kv, hd, 16, lens, asked, big=big)
        b.q = np.clip(b.q.astype(np.float32) * big, -65504, 65504).astype(np.float16)
    got = b.upload().launch().result().astype(np.float64)
    assert np.isfinite(got).all()
    tested = 0
    for s in range(len(lens)):
        for i in range(asked[s]):
            p = _seen(b, s, i)
            k, v = (x[b.table[s, p // 16], :, p % 16].astype(np.float64) for x in (b.cache.k, b.cache.v))
            for h in range(heads):
                q = b.q[b.start[s] + i, h].astype(np.float64)
                kk = k[:, h // (heads // kv)]
                x = kk @ q / np.sqrt(hd)
                reach = (np.abs(kk) @ np.abs(q)).max() / np.sqrt(hd)
                best = x.argmax()
                if len(p) > 1 and np.delete(x, best).max() > x[best] - 2 * reach * 2.0 ** -16 - 30:
                    continue
                tested += 1
                want = v[best, h // (heads // kv)]
                assert (np.abs(got[b.start[s] + i, h] - want) <= np.abs(want) * 2.0 ** -10 + 2.0 ** -24).all()
    assert tested >= 0.9 * heads * b.start[-1]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv,lens,asked", KERNELS)
def test_scores_far_apart(hip, heads, kv, lens, asked, hd):
    """Weights over the whole range of the exponential, and references that move
    with the positions: keys that grow to their end, and that shrink."""
    for turn in (1, -1):
        b = Trees(hip, 71, heads, kv, hd, 16, lens, asked, big=12.0)
        for s, n in enumerate(lens):                         # the row's largest keys last, or first
            pages = b.table[s, :-(-n // 16)]
            pages = pages[np.argsort(np.abs(b.cache.k[pages]).max((1, 2, 3)))][::turn]
            b.table[s, :len(pages)] = pages
        b.upload().launch().check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv,lens,asked", KERNELS)
def test_infinite_queries(hip, hd, heads, kv, lens, asked):
    """A query with infinities gives zeros where all its scores are -inf and NaN where
    some are not; the other rows keep the bar of any row (to the bit they need not be
    the same: a wave's rows share the choice of when their references move)."""
    b = Trees(hip, 72, heads, kv, hd, 16, lens, asked)
    want, spread, reach = b.expected()
    other = np.ones(want.shape[:2], bool)
    rows = [(0, 0, 1), (len(lens) - 1, asked[-1] - 1, heads - 1)]       # sequence, its row, head
    for s, i, h in rows:
        b.q[b.start[s] + i, h] = 0
        b.q[b.start[s] + i, h, 5] = -np.inf
        other[b.start[s] + i, h] = False
    got = b.upload().launch().result().astype(np.float64)
    for s, i, h in rows:
        p = _seen(b, s, i)
        k = b.cache.k[b.table[s, p // 16], h // (heads // kv), p % 16, 5].astype(np.float64)
        out = got[b.start[s] + i, h]
        # -inf times 0 is NaN too
        assert np.isnan(out).all() if (k <= 0).any() else not out.any()
    off = np.abs(got - want) - kv4_ref.tolerance(want, spread, reach)
    assert (off[other] <= 0).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv,lens,asked", KERNELS)
def test_results_repeat(hip, hd, heads, kv, lens, asked):
    """The same bits every time."""
    b = Trees(hip, 73, heads, kv, hd, 16, lens, asked).upload()
    first = b.launch().result().copy()
    for _ in range(3):
        assert np.array_equal(b.launch().result().view(np.uint16), first.view(np.uint16))


@pytest.mark.parametrize("hd", [64, 128])
def test_as_many_sequences_as_there_can_be(hip, hd):
    Trees(hip, 74, 1, 1, hd, 16, [1 + s % 3 for s in range(65535)], [1] * 65535).upload().launch().check()
