"""Speculative decoding as a serving loop runs it: trees of drafts over the 4-bit
cache, the drafts that stay, their keys and values moved up; eagerly and from a
graph.  Greedily it gives the tokens and the cache of decoding them one by one."""
from __future__ import annotations

import numpy as np
import pytest

import tree_ref
from test_gpu_kv4_cache import EPS
from test_gpu_kv4_serving import HIDDEN, PAGE, TOP, VOCAB, Server

pytestmark = pytest.mark.gpu
ROWS = 6                 # of a tree


class Speculator(Server):
    def __init__(self, *args):
        super().__init__(*args)
        n, up = self.nseq * ROWS, self.hip.DeviceArray.from_numpy
        self.d_parents, self.d_paths = (up(np.zeros(n, np.int32)) for _ in range(2))
        self.d_masks = up(np.zeros(n, np.uint64))
        self.d_uniforms, self.d_probs = (up(np.zeros(n, np.float32)) for _ in range(2))
        self.d_heat = up(np.zeros(self.nseq, np.float32))
        self.d_first, self.d_counts, self.d_after = (up(np.zeros(self.nseq, np.int32)) for _ in range(3))
        self.caches = self.hip.device.kv4_caches([self.view])
        self.d_start6 = up((np.arange(self.nseq + 1) * ROWS).astype(np.int32))
        heads, kv, hd = self.dims
        d = self.hip.device
        self.spaces = [(self.hip.DeviceArray(max(16, b)), b) for b in (
            d.kv4_tree_attention_workspace_bytes(self.most, ROWS, self.nseq, n, heads, kv, hd),
            d.verify_drafts_workspace_bytes(self.nseq, n, ROWS, VOCAB, False))]

    def speculate(self):
        """One step's launches; everything that changes from step to step is in device memory."""
        heads, kv, hd = self.dims
        d, row, n = self.hip.device, heads * hd, self.nseq * ROWS
        d.draft_tree(self.d_parents, self.d_start6, self.d_lens, self.nseq, n, ROWS, self.d_masks, self.d_at)
        for r in range(n):
            d.embed_at(self.dev["embed"], self.d_tokens.ptr + r * 4, VOCAB, self.d_x.ptr + r * HIDDEN * 2, HIDDEN)
            d.matvec("fp16", self.dev["w_qkv"], self.d_x.ptr + r * HIDDEN * 2, self.d_qkv.ptr + r * self.width * 2,
                     HIDDEN, self.width)
        base = self.d_qkv.ptr
        d.kv4_append(self.view, base, base + 2 * row, base + 2 * (row + kv * hd), self.width, self.width,
                     self.dev["q_norm"], self.dev["k_norm"], EPS, self.dev["rope"], self.most, self.d_at, self.d_slots,
                     n, heads, base, self.width)
        d.kv4_tree_attention(self.view, base, self.width, self.d_start6, self.d_lens, self.d_masks, self.d_table,
                             self.wide, self.nseq, n, ROWS, self.most, heads, *self.spaces[0], self.d_att, row)
        for r in range(n):
            d.matvec("fp16", self.dev["w_out"], self.d_att.ptr + r * row * 2, self.d_logits.ptr + r * VOCAB * 4, row,
                     VOCAB, f32_out=True)
        d.verify_drafts(self.d_logits, "fp32", VOCAB, VOCAB, None, 0, self.d_tokens, self.d_parents, self.d_start6,
                        self.nseq, n, ROWS, self.d_heat, self.d_uniforms, self.d_paths, self.d_counts, self.d_after,
                        self.d_probs, *self.spaces[1])
        d.kv4_keep(self.caches, self.d_table, self.wide, self.nseq, self.d_first, self.d_paths, ROWS, self.d_counts,
                   ROWS)

    def prompt(self, tokens):
        """Prompts of one length; the next tokens, greedily."""
        n = tokens.size
        self.d_tokens.upload(tokens.reshape(-1))
        self.d_next.upload(np.zeros(n, np.int32))
        self.place([tokens.shape[1]] * self.nseq)
        self.step(n, tokens.shape[1], self.workspaces(n, tokens.shape[1]))
        return self.d_ids.download(np.int32, n * TOP).reshape(self.nseq, -1, TOP)[:, -1, 0].copy()

    def kept(self):
        """Codes and scales of every sequence's positions (a page's layout is by position, so whole pages)."""
        raw = self.d_pages.download(np.uint8).reshape(self.cache.raw.shape)
        return [raw[self.table[s, :self.lens[s] // PAGE]] for s in range(self.nseq)]


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (4, 4, 64)])
@pytest.mark.parametrize("captured", [False, True])
def test_greedy_equals_one_by_one(hip, heads, kv, hd, captured):
    rng = np.random.default_rng(hd + 1)
    nseq, prompt, steps = 3, 21, 14
    tokens = rng.integers(0, VOCAB, (nseq, prompt)).astype(np.int32)
    stream = hip.device.Stream()
    hip.device.set_stream(stream)
    try:
        plain = Speculator(hip, 3, heads, kv, hd, nseq, nseq * prompt, 160)
        text = [plain.prompt(tokens)]
        one = plain.workspaces(nseq, 1)
        for _ in range(steps * ROWS):
            plain.place([1] * nseq)
            plain.d_tokens.upload(text[-1])
            plain.step(nseq, 1, one)
            text.append(plain.d_ids.download(np.int32, nseq * TOP).reshape(nseq, TOP)[:, 0].copy())
        text = np.array(text).T                                # [sequence][token]

        s = Speculator(hip, 3, heads, kv, hd, nseq, nseq * prompt, 160)
        out = [[t] for t in s.prompt(tokens)]
        graph = hip.device.Graph.capture(s.speculate) if captured else None
        lengths = set()
        for turn in range(steps):
            parents = [tree_ref.tree(rng, ROWS, wide=2) for _ in range(nseq)]
            drafts = rng.integers(0, VOCAB, (nseq, ROWS)).astype(np.int32)
            for q, ps in enumerate(parents):
                at = len(out[q]) - 1
                drafts[q, 0] = text[q, at]
                right = {0: at}                               # rows with the true text so far
                for i in range(1, ROWS):
                    if ps[i] in right and (turn + i + q) % 3 and right[ps[i]] + 1 not in right.values():
                        right[i] = right[ps[i]] + 1
                        drafts[q, i] = text[q, right[i]]
            s.d_first.upload(s.lens)
            first = s.lens.copy()
            s.place([ROWS] * nseq)                             # positions come from the tree, slots stay in order
            s.d_tokens.upload(drafts.reshape(-1))
            s.d_parents.upload(np.array(parents, np.int32).reshape(-1))
            s.d_uniforms.upload(rng.random(nseq * ROWS).astype(np.float32))
            graph.launch() if captured else s.speculate()
            counts = s.d_counts.download(np.int32, nseq)
            paths = s.d_paths.download(np.int32, nseq * ROWS).reshape(nseq, ROWS)
            after = s.d_after.download(np.int32, nseq)
            logits = s.d_logits.download(np.float32, nseq * ROWS * VOCAB).reshape(nseq, ROWS, VOCAB)
            for q in range(nseq):
                path, token, _ = tree_ref.verify(logits[q], None, drafts[q], parents[q], 0.0, np.zeros(ROWS), ROWS)
                assert path == paths[q, :counts[q]].tolist() and token == after[q]
                out[q] += [int(drafts[q, i]) for i in path[1:]] + [token]
                lengths.add(len(path))
            s.lens = (first + counts).astype(np.int32)
            for q in range(nseq):
                assert out[q] == text[q, :len(out[q])].tolist(), (turn, q)
        assert len(lengths) > 2
        plain.lens = s.lens                                    # the cache holds what one by one gives
        assert all(np.array_equal(a, b) for a, b in zip(s.kept(), plain.kept()))
        if captured:
            graph.close()
        hip.synchronize()
    finally:
        hip.device.set_stream(None)
        stream.close()


def test_draws_are_the_models(hip):
    """At a temperature: each step's path and token are what the definition makes
    of the device's own logits."""
    rng = np.random.default_rng(6)
    s = Speculator(hip, 4, 8, 2, 128, 3, 63, 160)
    after = s.prompt(rng.integers(0, VOCAB, (3, 21)).astype(np.int32))
    heat = np.float32([0.7, 1.3, 0.0])
    s.d_heat.upload(heat)
    ends = set()
    for _ in range(6):
        parents = [tree_ref.tree(rng, ROWS, wide=2) for _ in range(3)]
        drafts = rng.integers(0, VOCAB, (3, ROWS)).astype(np.int32)
        drafts[:, 0] = after
        uniforms = (rng.random((3, ROWS)) * 1e-4).astype(np.float32)      # so that unlikely drafts stay now and then
        uniforms[:, 0] = rng.random(3)
        s.d_first.upload(s.lens)
        first = s.lens.copy()
        s.place([ROWS] * 3)
        for d, x in ((s.d_tokens, drafts), (s.d_parents, np.array(parents, np.int32)), (s.d_uniforms, uniforms)):
            d.upload(x.reshape(-1))
        s.speculate()
        logits = s.d_logits.download(np.float32, 3 * ROWS * VOCAB).reshape(3, ROWS, VOCAB)
        counts, after = s.d_counts.download(np.int32, 3), s.d_after.download(np.int32, 3).copy()
        paths = s.d_paths.download(np.int32, 3 * ROWS).reshape(3, ROWS)
        for q in range(3):
            path, token, _ = tree_ref.verify(logits[q], None, drafts[q], parents[q], heat[q], uniforms[q], ROWS)
            assert path == paths[q, :counts[q]].tolist() and token == after[q]
            ends.add(len(path))
        s.lens = (first + counts).astype(np.int32)
    assert len(ends) > 1
