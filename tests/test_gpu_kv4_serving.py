"""The 4-bit cache, the attention over it and the log probabilities together, as
a serving loop uses them: prompts of several sequences in pieces, then greedy
steps whose next tokens are the device's own picks; eagerly and from a graph.

Each stage is held against numpy in 64 bits on the device's inputs of that
stage: stored keys by their codes' definition, attention by kv4_ref.tolerance,
a log probability by the bound of test_gpu_logprobs.py."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref
from test_gpu_kv4_cache import EPS, THETA, _rotated, _table
from test_gpu_logprobs import _want

pytestmark = pytest.mark.gpu
HIDDEN, VOCAB, TOP, PAGE = 256, 2003, 4, 16


class Server:
    def __init__(self, hip, seed, heads, kv, hd, nseq, most_tokens, most_context):
        rng = np.random.default_rng(seed)
        self.hip, self.dims, self.nseq, self.most = hip, (heads, kv, hd), nseq, most_context
        self.width = (heads + 2 * kv) * hd
        half = lambda *s: rng.standard_normal(s).astype(np.float16)                     # noqa: E731
        self.host = {"embed": half(VOCAB, HIDDEN), "w_qkv": half(self.width, HIDDEN) / np.float16(16),
                     "q_norm": 1 + half(hd) / np.float16(8), "k_norm": 1 + half(hd) / np.float16(8),
                     "w_out": half(VOCAB, heads * hd) / np.float16(4), "rope": _table(most_context, hd)}
        up = hip.DeviceArray.from_numpy
        self.dev = {n: up(np.ascontiguousarray(x)) for n, x in self.host.items()}
        self.wide = -(-most_context // PAGE)
        self.cache = kv4_ref.Cache(nseq * self.wide + 3, PAGE, kv, hd)
        self.table = rng.permutation(self.cache.num_pages)[:nseq * self.wide].astype(np.int32).reshape(nseq, -1)
        self.d_pages, self.d_table = up(self.cache.raw), up(self.table)
        self.view = hip.device.kv4_cache(self.d_pages, self.cache.num_pages, PAGE, kv, hd)
        n = most_tokens
        self.d_x, self.d_qkv = hip.DeviceArray(n * HIDDEN * 2), hip.DeviceArray(n * self.width * 2)
        self.d_att, self.d_logits = hip.DeviceArray(n * heads * hd * 2), hip.DeviceArray(n * VOCAB * 4)
        self.d_at, self.d_slots, self.d_next = (hip.DeviceArray(n * 4) for _ in range(3))
        self.d_lens, self.d_start = hip.DeviceArray(nseq * 4), hip.DeviceArray(nseq * 4 + 4)
        self.d_lp, self.d_ent, self.d_rank = (hip.DeviceArray(n * 4) for _ in range(3))
        self.d_ids, self.d_top = (up(np.zeros(n * TOP, np.int32)) for _ in range(2))
        self.d_tokens = hip.DeviceArray(n * 4)
        self.lens = np.zeros(nseq, np.int32)

    def workspaces(self, tokens, most_query):
        heads, kv, hd = self.dims
        d = self.hip.device
        sizes = (d.kv4_attention_workspace_bytes(self.most, most_query, self.nseq, tokens, heads, kv, hd),
                 d.token_logprobs_workspace_bytes(tokens, VOCAB, TOP))
        return [(self.hip.DeviceArray(max(16, n)), n) for n in sizes]

    def place(self, counts):
        """Positions and slots of the sequences' next `counts` tokens."""
        at = np.concatenate([self.lens[s] + np.arange(n) for s, n in enumerate(counts)]).astype(np.int32)
        seq = np.repeat(np.arange(self.nseq), counts)
        slots = (self.table[seq, at // PAGE] * PAGE + at % PAGE).astype(np.int32)
        self.lens = (self.lens + counts).astype(np.int32)
        for d, x in ((self.d_at, at), (self.d_slots, slots), (self.d_lens, self.lens),
                     (self.d_start, np.concatenate(([0], np.cumsum(counts))).astype(np.int32))):
            d.upload(x)
        return at, slots

    def step(self, tokens, most_query, spaces, from_picks=False):
        heads, kv, hd = self.dims
        d, row = self.hip.device, heads * hd
        for r in range(tokens):
            token = self.d_ids.ptr + r * TOP * 4 if from_picks else self.d_tokens.ptr + r * 4
            d.embed_at(self.dev["embed"], token, VOCAB, self.d_x.ptr + r * HIDDEN * 2, HIDDEN)
            d.matvec("fp16", self.dev["w_qkv"], self.d_x.ptr + r * HIDDEN * 2, self.d_qkv.ptr + r * self.width * 2,
                     HIDDEN, self.width)
        base = self.d_qkv.ptr
        d.kv4_append(self.view, base, base + 2 * row, base + 2 * (row + kv * hd), self.width, self.width,
                     self.dev["q_norm"], self.dev["k_norm"], EPS, self.dev["rope"], self.most, self.d_at, self.d_slots,
                     tokens, heads, base, self.width)
        d.kv4_attention(self.view, base, self.width, None if most_query == 1 else self.d_start, self.d_lens,
                        self.d_table, self.wide, self.nseq, tokens, most_query, self.most, heads, *spaces[0],
                        self.d_att, row)
        for r in range(tokens):
            d.matvec("fp16", self.dev["w_out"], self.d_att.ptr + r * row * 2, self.d_logits.ptr + r * VOCAB * 4, row,
                     VOCAB, f32_out=True)
        d.token_logprobs(self.d_logits, "fp32", VOCAB, tokens, VOCAB, self.d_next, self.d_lp, self.d_rank, self.d_ent,
                         TOP, self.d_ids, self.d_top, *spaces[1])

    def results(self, tokens):
        get = [d.download(np.int32, tokens).copy() for d in (self.d_lp, self.d_ent, self.d_rank)]
        return get + [d.download(np.int32, tokens * TOP).copy() for d in (self.d_ids, self.d_top)]

    def check(self, tokens, counts, at, slots, embedded, given):
        """The step that just ran, stage by stage."""
        heads, kv, hd = self.dims
        x = self.host["embed"][embedded].astype(np.float64)
        assert np.array_equal(self.d_x.download(np.float16, tokens * HIDDEN).reshape(tokens, HIDDEN), x)
        qkv = (x @ self.host["w_qkv"].T.astype(np.float64)).reshape(tokens, -1, hd)
        q = self.d_qkv.download(np.float16, tokens * self.width).reshape(tokens, -1, hd)
        # fp16 projections and their fp32 sums: 2^-11 of the value, 2^-20 of its terms
        room = np.abs(x) @ np.abs(self.host["w_qkv"].T.astype(np.float64)) * 2.0 ** -20
        assert (np.abs(q[:, heads:] - qkv[:, heads:]) <= np.abs(qkv[:, heads:]) * 2.0 ** -11 + 2.0 ** -25
                + room.reshape(tokens, -1, hd)[:, heads:]).all()
        k = _rotated(q[:, heads:heads + kv], self.host["k_norm"], self.host["rope"], at)[0].astype(np.float32)
        for t in range(tokens):
            self.cache.write(slots[t], k[t], q[t, heads + kv:])
        assert np.array_equal(self.d_pages.download(np.uint8).reshape(self.cache.raw.shape), self.cache.raw)
        slot_k, slot_v = zip(*(self.cache.read(s) for s in slots))
        shape = (self.cache.num_pages, kv, PAGE, hd)
        if not hasattr(self.cache, "k"):
            self.cache.k, self.cache.v = np.zeros(shape, np.float16), np.zeros(shape, np.float16)
        for s, a, b in zip(slots, slot_k, slot_v):
            self.cache.k[s // PAGE, :, s % PAGE], self.cache.v[s // PAGE, :, s % PAGE] = a, b
        start = np.concatenate(([0], np.cumsum(counts)))
        want, spread, reach = kv4_ref.attention(self.cache, q[:, :heads], start, self.lens, self.table)
        att = self.d_att.download(np.float16, tokens * heads * hd).reshape(want.shape).astype(np.float64)
        assert (np.abs(att - want) <= kv4_ref.tolerance(want, spread, reach)).all()
        logits = self.d_logits.download(np.float32, tokens * VOCAB).reshape(tokens, VOCAB)
        lp, ent, order = _want(logits, given, TOP)
        near = lambda v: 2.0 ** -22 * (np.abs(v) + np.log(VOCAB) + 1) + 34 * 2.0 ** -24   # noqa: E731
        r = np.arange(tokens)
        got_lp, got_ent, rank, ids, top = self.results(tokens)
        assert np.array_equal(ids.reshape(tokens, TOP), order)
        want_lp = lp[r, given]
        assert (np.abs(got_lp.view(np.float32) - want_lp) <= near(want_lp)).all()
        assert (np.abs(got_ent.view(np.float32) - ent) <= near(ent) + 34 * 2.0 ** -24 * (np.log(VOCAB) + 1)).all()
        listed = np.take_along_axis(lp, order, 1)
        assert (np.abs(top.view(np.float32).reshape(tokens, TOP) - listed) <= near(listed)).all()
        mine = logits[r, given][:, None]
        ahead = (logits > mine) | ((logits == mine) & (np.arange(VOCAB) < given[:, None]))
        assert np.array_equal(rank, ahead.sum(1))


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64)])
def test_prompts_in_pieces_then_greedy_steps(hip, heads, kv, hd):
    assert THETA == 1e6
    rng = np.random.default_rng(hd)
    pieces = [[5, 40, 17], [30, 1, 18], [1, 2, 3]]            # tokens of each sequence in each call
    s = Server(hip, 1, heads, kv, hd, 3, 64, 160)
    stream = hip.device.Stream()
    hip.device.set_stream(stream)
    try:
        for counts in pieces:
            n = sum(counts)
            tokens = rng.integers(0, VOCAB, n).astype(np.int32)
            given = rng.integers(0, VOCAB, n).astype(np.int32)
            s.d_tokens.upload(tokens)
            s.d_next.upload(given)
            at, slots = s.place(counts)
            s.step(n, max(counts), s.workspaces(n, max(counts)))
            s.check(n, counts, at, slots, tokens, given)
        # the first picks: the last row of each sequence
        ends = np.cumsum(pieces[-1]) - 1
        first = s.d_ids.download(np.int32, n * TOP).reshape(n, TOP)[ends].copy()
        pages, lens = s.d_pages.download(np.uint8), s.lens.copy()
        spaces = s.workspaces(3, 1)
        s.d_next.upload(np.array([1, 2, 3], np.int32))
        want = []
        for i in range(5):
            if i == 0:
                s.d_ids.upload(first)
            embedded = s.d_ids.download(np.int32, 3 * TOP).reshape(3, TOP)[:, 0].copy()
            at, slots = s.place([1, 1, 1])
            s.step(3, 1, spaces, from_picks=True)
            s.check(3, [1, 1, 1], at, slots, embedded, np.array([1, 2, 3]))
            want.append(s.results(3))
        # the same steps from a graph, with eager work of other rows between
        graph = hip.device.Graph.capture(lambda: s.step(3, 1, spaces, from_picks=True))
        other = Server(hip, 2, heads, kv, hd, 3, 8, 40)
        other.d_tokens.upload(np.arange(8, dtype=np.int32))
        other.d_next.upload(np.arange(8, dtype=np.int32))
        for _ in range(2):
            s.d_pages.upload(pages)
            s.d_ids.upload(first)
            s.lens = lens.copy()
            for i in range(5):
                s.place([1, 1, 1])
                graph.launch()
                assert all(np.array_equal(a, b) for a, b in zip(s.results(3), want[i])), i
                if other.lens.max() < 30:
                    other.place([1, 2, 3])
                    other.step(6, 3, other.workspaces(6, 3))
        assert np.array_equal(s.d_pages.download(np.uint8).reshape(s.cache.raw.shape), s.cache.raw)
        graph.close()
        hip.synchronize()
    finally:
        hip.device.set_stream(None)
        stream.close()
