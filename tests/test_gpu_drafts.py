"""Masks and positions of trees of drafted tokens, and which drafts stay, against
numpy in 64 bits.  Bars: masks, positions, paths, counts and tokens are equal;
probabilities are one fp32 rounding (2^-24) of 64-bit values that are off by
less than 1e-12 (an exponential by 1e-13, as are then their sums; 2^18 additions by
2^-53 each of what they have reached add less than 3e-11 in the worst case, and the
sums run over 32, 64 and 149 terms: 3e-14)."""
from __future__ import annotations

import numpy as np
import pytest

import tree_ref

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- masks
def _tree_call(hip, parents, lens, max_query, behind=2, positions=True, single=False):
    up = hip.DeviceArray.from_numpy
    sizes = [len(p) for p in parents]
    start = np.concatenate(([0], np.cumsum(sizes))).astype(np.int32)
    rows, words = int(start[-1]), -(-max_query // 64)
    flat = np.array([x for p in parents for x in p] + [0] * behind, np.int32)
    masks = up(np.full((rows + behind, words), 77, np.uint64))
    at = up(np.full(rows + behind, 77, np.int32))
    d = [up(x) for x in (flat, start, np.array(lens, np.int32))]
    hip.device.draft_tree(d[0], None if single else d[1], d[2], len(parents), rows + (0 if single else behind),
                          max_query, masks, at if positions else None)
    return masks.download(np.uint64, (rows + behind) * words).reshape(-1, words), at.download(np.int32, rows + behind)


def _check_tree(hip, parents, lens, max_query, **kw):
    masks, at = _tree_call(hip, parents, lens, max_query, **kw)
    row, words = 0, -(-max_query // 64)
    for ps, length in zip(parents, lens):
        see, depth = tree_ref.masks_of(ps)
        for i in range(len(ps)):
            if i >= max_query:
                assert (masks[row + i] == 77).all() and at[row + i] == 77
                continue
            assert np.array_equal(masks[row + i], tree_ref.pack(see[i:i + 1], words)[0]), (i, ps)
            assert at[row + i] == (max(length, 0) - len(ps) + depth[i] if depth[i] >= 0 else -1)
        row += len(ps)
    assert (masks[row:] == 77).all() and (at[row:] == 77).all()


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 127, 128, 129, 200, 255, 256])
def test_trees_of_every_size(hip, n):
    rng = np.random.default_rng(n)
    parents = [tree_ref.tree(rng, n), list(range(-1, n - 1)), [-1] + [0] * (n - 1), [-1] * n,
               [-1] + [int(rng.integers(-1, i)) for i in range(1, n)], tree_ref.tree(rng, max(1, n // 2)), []]
    _check_tree(hip, parents, [n + 5, n, 1000, 3, n + 64, 2 ** 30, 9], n)


def test_parents_that_are_no_earlier_row(hip):
    """Such a row and the rows below it see nothing."""
    parents = [[-1, 0, 2, 2, 1], [0, 0, -1, 2], [-2, 0, -1], [5, -1, 1, 0], [-1, 0, 2 ** 31 - 1, -2 ** 31, 3]]
    _check_tree(hip, parents, [9, 9, 3, 50, 0], 5)


def test_rows_past_the_bound_and_short_contexts(hip):
    rng = np.random.default_rng(3)
    parents = [tree_ref.tree(rng, n) for n in (100, 64, 30, 1)]
    for most in (1, 30, 64, 65, 99):
        _check_tree(hip, parents, [10, -5, 30, 0], most)


def test_one_row_each_and_no_positions(hip):
    _check_tree(hip, [[-1], [-1], [0]], [7, 1, 9], 1, behind=0, single=True)
    masks, at = _tree_call(hip, [[-1, 0], [-1]], [7, 1], 2, positions=False)
    assert (at == 77).all() and masks[:3, 0].tolist() == [1, 3, 1]


def test_many_sequences(hip):
    rng = np.random.default_rng(4)
    parents = [tree_ref.tree(rng, int(rng.integers(0, 40))) for _ in range(700)]
    _check_tree(hip, parents, list(rng.integers(40, 5000, 700)), 40)


# ---------------------------------------------------------------- verification
class Step:
    """The rows of a step: logits with a few likely tokens, drafts among them."""

    def __init__(self, hip, seed, sizes, vocab, tree=False, drafted=False, half=False, heat=1.0, pad=0, max_query=None,
                 behind=0, offset=0):
        rng = np.random.default_rng(seed)
        self.hip, self.vocab, self.half, self.sizes = hip, vocab, half, sizes
        self.start = np.concatenate(([0], np.cumsum(sizes))).astype(np.int32)
        self.rows = int(self.start[-1]) + behind
        self.max_query = max_query or max(1, max(sizes))
        self.type = np.float16 if half else np.float32
        self.stride, self.offset = vocab + pad, offset
        n = self.rows
        self.logits = rng.standard_normal((n, vocab)) * 2
        likely = rng.integers(0, vocab, (n, 5))
        np.put_along_axis(self.logits, likely, rng.random((n, 5)) * 5 + np.log(vocab), 1)
        self.logits = self.logits.astype(self.type)
        self.draft = (self.logits + rng.standard_normal((n, vocab)) * 0.7).astype(self.type) if drafted else None
        self.parents = [tree_ref.tree(rng, k) for k in sizes] if tree else None
        self.heat = np.broadcast_to(np.float32(heat), (len(sizes),)).copy()
        self.uniforms = rng.random(n).astype(np.float32)
        self.tokens = rng.integers(0, vocab, n).astype(np.int32)
        for s, k in enumerate(sizes):
            for i in range(1, k):
                up = self.parents[s][i] if tree else i - 1
                if up < 0:
                    continue
                row = int(self.start[s]) + up
                if drafted:
                    p = tree_ref.distribution(self.draft[row], self.heat[s])
                    self.tokens[self.start[s] + i] = rng.choice(vocab, p=p)
                else:
                    self.tokens[self.start[s] + i] = likely[row, i % 5]

    def _rows(self, x):
        """Rows `stride` apart, `offset` elements into their buffer; NaN between them."""
        flat = np.full(self.offset + max(1, len(x)) * self.stride, np.nan, self.type)
        flat[self.offset:].reshape(-1, self.stride)[:len(x), :self.vocab] = x
        return self.hip.DeviceArray.from_numpy(flat)

    def upload(self):
        up = self.hip.DeviceArray.from_numpy
        self.d_logits = self._rows(self.logits)
        self.d_draft = self._rows(self.draft) if self.draft is not None else None
        self.d_tokens, self.d_start, self.d_heat, self.d_uniforms = (
            up(x) for x in (self.tokens, self.start, self.heat, self.uniforms))
        flat = [p for ps in self.parents or [] for p in ps] + [0] * (self.rows - int(self.start[-1]))
        self.d_parents = up(np.array(flat, np.int32)) if self.parents is not None else None
        n = len(self.sizes)
        self.d_paths = up(np.full((n, self.max_query), 77, np.int32))
        self.d_counts, self.d_next = (up(np.full(n, 77, np.int32)) for _ in range(2))
        self.d_probs = up(np.full(max(1, self.rows), 77, np.float32))
        self.bytes = self.hip.device.verify_drafts_workspace_bytes(n, self.rows, self.max_query, self.vocab,
                                                                   self.draft is not None)
        self.d_ws = up(np.full(max(16, self.bytes), 0xFF, np.uint8))
        return self

    def launch(self, temperatures=True, outputs=True, single=False):
        size, at = self.type().itemsize, self.offset
        place = lambda d: None if d is None else d.ptr + at * size                      # noqa: E731
        wanted = (self.d_paths, self.d_counts) if outputs else (None, None)
        self.hip.device.verify_drafts(place(self.d_logits), "fp16" if self.half else "fp32", self.stride, self.vocab,
                                      place(self.d_draft), self.stride, self.d_tokens, self.d_parents,
                                      None if single else self.d_start, len(self.sizes), self.rows, self.max_query,
                                      self.d_heat if temperatures else None, self.d_uniforms, *wanted, self.d_next,
                                      self.d_probs if outputs else None, self.d_ws, self.bytes)
        return self

    def expected(self):
        out = []
        for s, n in enumerate(self.sizes):
            r = slice(self.start[s], self.start[s] + n)
            out.append(tree_ref.verify(self.logits[r], self.draft[r] if self.draft is not None else None,
                                       self.tokens[r], self.parents[s] if self.parents is not None else None,
                                       self.heat[s], self.uniforms[r], self.max_query))
        return out

    def check(self):
        n = len(self.sizes)
        paths = self.d_paths.download(np.int32, n * self.max_query).reshape(n, -1)
        counts, after = self.d_counts.download(np.int32, n), self.d_next.download(np.int32, n)
        probs = self.d_probs.download(np.float32, max(1, self.rows))
        seen = np.zeros(max(1, self.rows), bool)
        got = []
        for s, (path, token, p) in enumerate(self.expected()):
            assert counts[s] == len(path), (s, counts[s], path)
            assert paths[s].tolist() == path + [-1] * (self.max_query - len(path)), s
            assert after[s] == token, (s, after[s], token)
            r = slice(self.start[s], self.start[s] + len(p))
            assert (np.abs(probs[r] - p) <= p * (2.0 ** -24 + 1e-12) + 2.0 ** -149).all(), s
            seen[r] = True
            got.append((path, token))
        assert (probs[~seen] == 77).all()                # rows behind the last sequence, or past max_query
        return got


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 2047, 2048, 2049, 8192, 8193, 32003, 151936])
@pytest.mark.parametrize("drafted", [False, True])
def test_chains(hip, vocab, half, drafted):
    got = Step(hip, vocab, [5, 1, 4, 8, 2], vocab, drafted=drafted, half=half,
               heat=[1, 0.7, 0, 2, 0.5]).upload().launch().check()
    assert all(path == list(range(len(path))) for path, _ in got)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("sizes,vocab", [([40, 1, 17, 64], 2000), ([256, 100], 515), ([12] * 30, 4097),
                                         ([7, 0, 9], 151936)])
def test_trees(hip, sizes, vocab, half):
    heat = np.resize([1.0, 0.6, 0.0], len(sizes))
    Step(hip, vocab + 1, sizes, vocab, tree=True, half=half, heat=heat).upload().launch().check()


@pytest.mark.parametrize("seed", range(6))
def test_many_chains(hip, seed):
    """Enough of them that every way to end is met: accepted and rejected at
    any row, and the token drawn from what the draft leaves."""
    step = Step(hip, 100 + seed, [4] * 150, 700 + seed, drafted=seed % 2 == 0, heat=0.9).upload().launch()
    lengths = {len(path) for path, _ in step.check()}
    assert lengths >= {1, 2, 3}


@pytest.mark.parametrize("half,pad,offset", [(True, 1, 0), (True, 0, 1), (True, 3, 5), (False, 1, 0), (False, 2, 3),
                                             (False, 0, 1)])
def test_rows_of_any_alignment(hip, half, pad, offset):
    for drafted in (False, True):
        Step(hip, 7, [3, 5], 5001, drafted=drafted, half=half, pad=pad, offset=offset).upload().launch().check()


def test_draws_alone(hip):
    """One row each: the next token of a batch; no tokens, parents or temperatures."""
    step = Step(hip, 8, [1] * 60, 3001).upload()
    step.d_tokens = None
    step.launch(temperatures=False, single=True)
    got = step.check()
    assert len({t for _, t in got}) > 20
    step.upload()
    step.launch(temperatures=False, outputs=False, single=True)
    assert step.d_next.download(np.int32, 60).tolist() == [t for _, t in got]
    assert (step.d_paths.download(np.int32, 60) == 77).all()


def test_draws_follow_the_distribution(hip):
    """4096 draws over the unit interval come out in the proportions of p: each id
    as often as its share of the evenly spaced numbers, give or take one."""
    n, vocab = 4096, 50
    step = Step(hip, 9, [1] * n, vocab)
    step.logits[:] = step.logits[0]
    step.uniforms = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = step.upload().launch().check()
    p = tree_ref.distribution(step.logits[0], 1.0)
    counts = np.bincount([t for _, t in got], minlength=vocab)
    assert (np.abs(counts - p * n) <= 1.001).all()


def test_borders(hip):
    """Weights that 64 bits hold exactly: a running sum equal to u times the total
    does not exceed it, and u q equal to p does not accept."""
    vocab = 4096
    u = np.float32([0, 0.25, 0.5, 1 - 2 ** -24, np.nextafter(np.float32(0.5), np.float32(0))])
    step = Step(hip, 10, [1] * len(u), vocab)
    step.logits[:] = 3
    step.uniforms = u
    got = [t for _, t in step.upload().launch().check()]
    assert got == [0, 1024, 2048, 4095, 2047]
    # two tokens of p = 1/2: u = 1/2 rejects, the number below it accepts
    step = Step(hip, 11, [2, 2, 3], 3000)
    step.logits[:] = -np.inf
    step.logits[:, [5, 2500]] = 1
    step.tokens[:] = 5
    step.uniforms[:] = 0
    step.uniforms[[1, 3]] = 0.5, np.nextafter(np.float32(0.5), np.float32(0))
    step.uniforms[[5, 6]] = np.nextafter(np.float32(0.5), np.float32(0)), 0.5
    got = step.upload().launch().check()
    assert got == [([0], 2500), ([0, 1], 5), ([0, 1], 2500)]


def test_numbers_outside_the_unit_interval(hip):
    for drafted in (False, True):
        step = Step(hip, 12, [3] * 8, 500, drafted=drafted)
        step.uniforms = np.resize(np.float32([-1, np.nan, 1, 2, np.inf, -np.inf, 0, 0.999]), len(step.uniforms))
        step.upload().launch().check()


def test_a_token_drafted_twice(hip):
    """Siblings with one token: rejected once, it cannot come again, nor be drawn."""
    step = Step(hip, 13, [6] * 40, 300, tree=True)
    step.parents = [[-1, 0, 0, 0, 0, 0]] * 40
    for s in range(40):
        r = step.start[s]
        step.tokens[r + 1:r + 6] = step.tokens[r + 1], step.tokens[r + 2], step.tokens[r + 1], step.tokens[r + 2], 7
    got = step.upload().launch().check()
    for s, (path, token) in enumerate(got):
        r = step.start[s]
        tried = step.tokens[r + 1:r + (path[1] if len(path) > 1 else 6)]
        assert len(path) > 1 or token not in tried
        assert path[-1] not in (3, 4)


def test_all_that_could_come_is_rejected(hip):
    """Nothing is left of p: the token comes from p as it was."""
    step = Step(hip, 14, [3, 3], 5000, tree=True)
    step.parents = [[-1, 0, 0]] * 2
    step.logits[:] = -np.inf
    step.logits[:, 4100] = 2
    step.logits[3, 4200] = 2
    step.tokens[:] = 4100
    step.tokens[[2, 5]] = 4200
    step.uniforms[:] = 1 - 2 ** -24
    step.uniforms[0] = step.uniforms[3] = 0.3
    step.upload().launch().check()
    step = Step(hip, 15, [2], 5000, drafted=True)        # p = q, and the draft a token that cannot come
    step.draft[:] = step.logits
    step.logits[0, 17] = step.draft[0, 17] = -np.inf
    step.tokens[1] = 17
    got = step.upload().launch().check()
    assert got[0][0] == [0]


def test_tokens_and_parents_outside(hip):
    for drafted in (False, True):
        step = Step(hip, 16, [4, 4, 4, 4], 900, drafted=drafted)
        step.tokens[[1, 6, 11]] = -1, 900, 2 ** 31 - 1
        step.upload().launch().check()
    step = Step(hip, 17, [5, 4, 3], 900, tree=True)
    step.parents = [[-1, -1, 0, 7, 2], [3, 0, 1, 2], [-1, 2 ** 31 - 1, -2 ** 31]]
    step.uniforms[:] = 0
    got = step.upload().launch().check()
    assert [path for path, _ in got][1:] == [[0, 1, 2, 3], [0]]


def test_tokens_that_cannot_come(hip):
    """Nearly all logits -inf: only the others are drawn, at u = 0 and close to 1."""
    for vocab, keep in ((5000, [4999]), (5000, [0]), (9000, [2047, 2048, 8999]), (151936, [70000, 151935])):
        for drafted in (False, True):
            step = Step(hip, 18, [1, 1, 2], vocab, drafted=drafted)
            allowed = np.zeros(vocab, bool)
            allowed[keep] = True
            for x in (step.logits, step.draft) if drafted else (step.logits,):
                x[:, ~allowed] = -np.inf
                x[:, keep] = 1.5
            step.uniforms[:2] = 0, 1 - 2 ** -24
            got = step.upload().launch().check()
            assert [t for _, t in got][:2] == [keep[0], keep[-1]] and got[2][1] in keep


def test_rows_without_a_distribution(hip):
    """NaN, +inf, or nothing above -inf: no child is accepted, no token comes."""
    for heat in (1.0, 0.0):
        for at in (0, 700, 4999):
            for value in (np.nan, np.inf):
                step = Step(hip, 19, [3, 3, 3], 5000, heat=heat)
                step.uniforms[:] = 0
                step.logits[0, at] = step.logits[4, at] = value
                step.logits[8] = -np.inf
                got = step.upload().launch().check()
                assert got[0] == ([0], -1)
                if heat:               # (greedily the drafts are not the rows' largest)
                    assert got[1] == ([0, 1], -1) and got[2] == ([0, 1, 2], -1)
                step = Step(hip, 20, [3, 3], 5000, heat=heat, drafted=True)
                step.uniforms[:] = 0.2
                step.draft[0, at] = value
                step.draft[3] = -np.inf
                step.draft[5, at] = step.draft[2, at] = np.nan      # a last row's draft is not read
                got = step.upload().launch().check()
                assert [path for path, _ in got] == [[0], [0]]


def test_greedy_takes_the_lowest_of_equal_logits(hip):
    for half in (False, True):
        step = Step(hip, 21, [2, 2, 2], 9000, heat=[0, -1, np.nan], half=half)
        step.logits[:] = np.minimum(step.logits, 4)
        for r, ids in enumerate(([8999, 2100, 2500], [5, 6], [0, 8999], [4096, 2048], [2047, 63, 64], [8000, 8001])):
            step.logits[r, ids] = 9
        step.tokens[[1, 3, 5]] = 2100, 8999, 63
        got = step.upload().launch().check()
        assert got == [([0, 1], 5), ([0], 0), ([0, 1], 8000)]
        step.logits[0, 2099] = -0.0
        step.logits[0] = np.where(step.logits[0] == 9, 0.0, np.minimum(step.logits[0], -0.0))
        step.upload().launch().check()


@pytest.mark.parametrize("heat", [1e-30, 1e-3, 1e-45, 50.0, 3e38])
def test_temperatures_of_any_size(hip, heat):
    for drafted in (False, True):
        Step(hip, 22, [3, 3, 2], 2500, heat=heat, drafted=drafted).upload().launch().check()


def test_an_infinite_temperature(hip):
    """Every token that can come is as likely as the others, as at the largest
    finite one (where a difference of logits of 20 is 2^-123 of a weight)."""
    for drafted in (False, True):
        for half in (False, True):
            step = Step(hip, 30, [3, 3, 2], 2500, drafted=drafted, half=half)
            for x in (step.logits, step.draft) if drafted else (step.logits,):
                x[:, ::3] = -np.inf
            step.heat[:] = np.inf
            step.upload().launch()
            step.heat[:] = np.finfo(np.float32).max
            step.check()


def test_running_sums_that_rounding_does_not_order(hip):
    """Weights of e^-36.9 twice, 1, 0 and 1: the sum of the first three is 1 or its
    successor, as they are added, and half of the total 1.  A segment without a
    weight never has the token."""
    step = Step(hip, 31, [1, 1], 5 * 2048)
    step.logits[:] = -np.inf
    step.logits[:, [5, 2048]] = -36.9
    step.logits[:, [2 * 2048 + 7, 4 * 2048 + 9]] = 0
    step.uniforms[:] = 0.5, 0
    step.upload().launch()
    after = step.d_next.download(np.int32, 2)
    assert after[0] in (2 * 2048 + 7, 4 * 2048 + 9) and after[1] == 5


def test_millions_of_tokens(hip):
    """More than 64 * 64 segments; equal logits, whose sums are exact."""
    vocab = 2 ** 23 + 70001
    for drafted in (False, True):
        step = Step(hip, 32, [2], 40, half=True)
        step.vocab = step.stride = vocab
        step.logits = np.full((2, vocab), 3, np.float16)
        step.logits[:, ::5] = step.logits[:, 4500000:4700000] = -np.inf
        step.draft = None
        left = np.isfinite(step.logits[0])
        if drafted:                  # half of what p has, each twice as likely: the rest is the other half
            step.draft = step.logits.copy()
            step.draft[:, np.flatnonzero(left)[1::2]] = -np.inf
        step.tokens[1] = 10          # (10 is a multiple of 5: it cannot come)
        for u in (0, 0.25, 0.4999999, 0.7, 1 - 2 ** -24):
            step.uniforms[:] = u, 0.5
            step.upload().launch()
            ids = np.flatnonzero(left)[1::2] if drafted else np.flatnonzero(left)
            want = ids[int(float(np.float32(u)) * len(ids))]
            assert step.d_counts.download(np.int32, 1)[0] == 1
            assert abs(int(np.searchsorted(ids, step.d_next.download(np.int32, 1)[0])) -
                       int(np.searchsorted(ids, want))) <= (1 if drafted else 0)


@pytest.mark.parametrize("half", [False, True])
def test_rows_past_four_gigabytes(hip, half):
    """Rows 2 GiB apart."""
    for drafted in (False, True):
        step = Step(hip, 33, [2, 1], 5000, half=half, drafted=drafted).upload()
        step.stride = (1 << 31) // step.type().itemsize

        def spread(x):
            d = hip.DeviceArray((len(x) - 1) * (1 << 31) + x[0].nbytes)
            for r, row in enumerate(x):
                d.upload(row, r << 31)
            return d

        step.d_logits = spread(step.logits)
        step.d_draft = spread(step.draft) if drafted else None
        step.launch().check()


@pytest.mark.parametrize("scale", [1e4, 1e30, 3e38])
def test_logits_of_any_size(hip, scale):
    for heat in (1.0, 0.0, 1e30):
        step = Step(hip, 23, [3, 3], 2500, heat=heat)
        step.logits = np.clip(step.logits.astype(np.float64) * scale / 20, -3.4e38, 3.4e38).astype(np.float32)
        step.upload().launch().check()


def test_rows_past_the_bound_and_behind_the_last(hip):
    for tree in (False, True):
        for most in (1, 2, 5):
            Step(hip, 24, [6, 3, 0, 9], 800, tree=tree, max_query=most, behind=2).upload().launch().check()
    got = Step(hip, 25, [0, 0], 800, max_query=3, behind=1).upload().launch().check()
    assert got == [([], -1), ([], -1)]


def test_many_sequences(hip):
    Step(hip, 26, [2] * 1500, 130, drafted=True).upload().launch().check()


def test_two_graphs_and_eager_calls(hip):
    """Captured calls on a stream of their own, with other numbers, temperatures
    and drafts between the replays."""
    stream = hip.device.Stream()
    hip.device.set_stream(stream)
    try:
        steps = [Step(hip, 27, [4, 5, 3], 6000, drafted=True).upload(),
                 Step(hip, 28, [20, 9], 3000, tree=True, half=True).upload()]
        for s in steps:
            s.launch().check()
        graphs = [hip.device.Graph.capture(s.launch) for s in steps]
        rng = np.random.default_rng(5)
        for turn in range(4):
            for s in steps:
                s.uniforms = rng.random(s.rows).astype(np.float32)
                s.heat = rng.choice(np.float32([0, 0.5, 1]), len(s.sizes))
                s.d_uniforms.upload(s.uniforms)
                s.d_heat.upload(s.heat)
                s.d_probs.upload(np.full(s.rows, 77, np.float32))
            for g in graphs:
                g.launch()
            for s in steps:
                s.check()
            steps[turn % 2].launch().check()
        for g in graphs:
            g.close()
        hip.synchronize()
    finally:
        hip.device.set_stream(None)
        stream.close()


def test_results_repeat(hip):
    """The same bits every time."""
    step = Step(hip, 29, [6] * 20, 20011, drafted=True).upload()
    first = None
    for _ in range(3):
        step.launch().check()
        probs = step.d_probs.download(np.uint32, step.rows)
        assert first is None or np.array_equal(first, probs)
        first = probs


@pytest.mark.parametrize("half", [False, True])
def test_an_infinite_temperature_over_masked_logits(hip, half):
    """Logits of the type's lowest and largest value are as likely as the others.
    Weights of 1, whose sums are exact: token floor(u n) of the n that can come."""
    big = float(np.finfo(np.float16 if half else np.float32).max)
    for vocab in (1000, 9001, 40000):
        for drafted in (False, True):
            step = Step(hip, 34, [1] * 9 + [2], vocab, drafted=drafted, half=half, heat=np.inf)
            here = np.flatnonzero(np.arange(vocab) % 3 != 1)
            for x in (step.logits, step.draft) if drafted else (step.logits,):
                x[:, 2::3], x[:, 0::6] = -big, big
                x[:, 1::3] = -np.inf
            step.uniforms[:9] = 0, 0.1, 0.25, 1 / 3, 0.5, 0.6, 0.75, 0.9, 1 - 2 ** -24
            step.tokens[10] = here[7]            # p = 1 / n: u = 1 / n is rejected, and what is left is all but it
            step.uniforms[9:] = 0.3, 0.9
            step.upload().launch()
            after = step.d_next.download(np.int32, 10)
            n = len(here)
            assert after[:9].tolist() == [int(here[int(float(u) * n)]) for u in step.uniforms[:9]]
            probs = step.d_probs.download(np.float32, step.rows)
            assert abs(probs[10] * n - 1) <= 2 ** -24 + 1e-12
            if drafted:                          # p = q: accepted
                assert step.d_counts.download(np.int32, 10)[9] == 2
                assert after[9] == here[int(float(step.uniforms[9]) * n)]
            else:
                rest = np.delete(here, 7)
                assert step.d_counts.download(np.int32, 10)[9] == 1
                assert after[9] == rest[int(float(step.uniforms[9]) * (n - 1))]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("vocab,ids", [(5000, (17, 18, 19)), (5000, (17, 2500, 4999)), (40000, (4100, 39999, 5))])
def test_every_token_that_could_come_is_rejected(hip, half, vocab, ids):
    """Three tokens that can come, weights 1, a = e^-16 and b = e^-31.125, all rejected
    at u = 1 - 2^-24: nothing is left, and the token comes from p.  R is 1, a + b and
    b of p, so u R is below what is left by 2^-24 of it.  Token 1: 1 - 2^-24 >= 1 -
    1.1254e-7.  Token 2: b is 2.7e-7 of a, more than 2^-24.  Token 3: R is b and the
    rounding of 1 / s, for R = 1 - 1 / s - a / s, 6.3e-17 or 2e-3 of b too much (s is
    rounded up by a quarter of 2^-52 in every order of the three weights, 1 / s down)."""
    w = np.exp(np.float64([0, -16, -31.125]))
    assert (w[0] + w[1]) + w[2] == (w[0] + w[2]) + w[1] == w[0] + (w[1] + w[2])
    step = Step(hip, 35, [4, 5, 4], vocab, tree=True, half=half)
    step.parents = [[-1, 0, 0, 0], [-1, 0, 0, 0, 0], [-1, 0, 0, 0]]
    step.logits[:] = -np.inf
    step.logits[:, ids] = 0, -16, -31.125
    step.tokens[[1, 2, 3, 5, 6, 7, 8, 10, 11, 12]] = (*ids, *ids, ids[0], *ids)
    step.uniforms[:] = 1 - 2 ** -24
    step.uniforms[[4, 9]] = 0.3, 0
    got = step.upload().launch().check()
    assert [path for path, _ in got] == [[0]] * 3
    order = sorted(zip(ids, w))
    assert got[2][1] == order[0][0] and got[1][1] == ids[0]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("vocab", [5000, 32768, 32769, 151936])
def test_drafts_that_leave_nothing(hip, vocab, half):
    """p = q, and drafts that cannot come: rejected, and the token comes from p.  Rows
    of up to 16 segments are finished by the workgroup that finds the path."""
    step = Step(hip, 36, [2, 3, 2, 1], vocab, drafted=True, half=half, heat=[1, 0.6, 1.5, 1])
    step.logits[:, [17, vocab - 1]] = -np.inf
    step.draft[:] = step.logits
    step.tokens[[1, 3, 6]] = 17, vocab - 1, -1
    got = step.upload().launch().check()
    assert [path for path, _ in got] == [[0]] * 4
    for s in range(4):
        row = step.start[s]
        assert got[s][1] == tree_ref.draw(tree_ref.distribution(step.logits[row], step.heat[s]), step.uniforms[row])


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("vocab", [300, 5000, 151936])
def test_a_wide_tree_of_rejected_drafts(hip, vocab, half):
    """255 children of one row, with all but a fiftieth of p, each smaller than the
    next and rejected at u = 1 - 2^-24 (R is at least a fiftieth more than its p): the
    token comes from the others."""
    step = Step(hip, 37, [256, 256], vocab, tree=True, half=half)
    step.parents = [[-1] + [0] * 255] * 2
    rng = np.random.default_rng(38)
    step.logits[:] = rng.standard_normal(step.logits.shape)
    for s, spread in enumerate((vocab, min(vocab, 290))):       # all over the row, and close together
        ids = rng.permutation(spread)[:255]
        x = step.logits[256 * s].astype(np.float64)
        others = np.delete(np.exp(x), ids).sum()
        part = np.linspace(0.5, 1.5, 255)
        step.logits[256 * s, ids] = np.log(part / part.sum() * others * 49)
        step.tokens[256 * s + 1:256 * s + 256] = ids[np.argsort(step.logits[256 * s, ids], kind="stable")]
    step.uniforms[:] = 1 - 2 ** -24
    step.uniforms[[0, 256]] = 0.37, 0.81
    got = step.upload().launch().check()
    for s, (path, token) in enumerate(got):
        assert path == [0] and token not in step.tokens[256 * s + 1:256 * s + 256]


@pytest.mark.parametrize("half", [False, True])
def test_chains_of_256(hip, half):
    """As long as a sequence can be: drafts of the model's own distribution are all
    accepted, others are rejected somewhere."""
    step = Step(hip, 39, [256, 200, 256], 3001, drafted=True, half=half)
    step.draft[:456] = step.logits[:456]
    got = step.upload().launch().check()
    assert [len(path) for path, _ in got[:2]] == [256, 200] and len(got[2][0]) < 256


def test_draft_rows_of_another_stride(hip):
    for half in (False, True):
        step = Step(hip, 40, [3, 4, 2], 5003, drafted=True, half=half).upload()
        wide = np.full((step.rows, 5003 + 37), np.nan, step.type)
        wide[:, :5003] = step.draft
        step.d_draft = hip.DeviceArray.from_numpy(wide)
        hip.device.verify_drafts(step.d_logits, "fp16" if half else "fp32", 5003, 5003, step.d_draft, 5003 + 37,
                                 step.d_tokens, None, step.d_start, 3, step.rows, step.max_query, step.d_heat,
                                 step.d_uniforms, step.d_paths, step.d_counts, step.d_next, step.d_probs, step.d_ws,
                                 step.bytes)
        step.check()


def test_as_many_sequences_as_there_can_be(hip):
    Step(hip, 41, [1] * 65535, 21).upload().launch().check()
    Step(hip, 42, [2] * 65535, 9, drafted=True).upload().launch().check()
    _check_tree(hip, [[-1, 0]] * 65535, [5] * 65535, 2)
