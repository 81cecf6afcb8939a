"""Moves of cached tokens within their sequences, byte for byte against numpy."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref
import tree_ref

pytestmark = pytest.mark.gpu


class Moves:
    def __init__(self, hip, seed, hd, page, kv, firsts, kept, layers=2, spare=2, stride=None):
        rng = np.random.default_rng(seed)
        self.hip, self.shape, self.firsts, self.kept, self.layers = hip, (page, kv, hd), firsts, kept, layers
        need = [max(1, -(-(max(0, f) + max([0] + list(k)) + 1) // page)) for f, k in zip(firsts, kept)]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(firsts), max(need)), -3, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        size = kv4_ref.head_layout(page, hd)[4]
        self.raw = rng.integers(0, 256, (layers, self.pages, kv, size), dtype=np.uint8)
        self.stride = stride or max(1, max(len(k) for k in kept))
        self.flat = np.full((len(kept), self.stride), 2 ** 31 - 1, np.int32)
        for s, k in enumerate(kept):
            self.flat[s, :len(k)] = k
        self.counts = np.array([len(k) for k in kept], np.int32)
        self.max_count = self.stride

    def upload(self):
        up = self.hip.DeviceArray.from_numpy
        page, kv, hd = self.shape
        self.d_raw = [up(x) for x in self.raw]
        self.caches = self.hip.device.kv4_caches(
            [self.hip.device.kv4_cache(d, self.pages, page, kv, hd) for d in self.d_raw])
        self.d = [up(x) for x in (self.table, np.array(self.firsts, np.int32), self.flat, self.counts)]
        return self

    def launch(self):
        table, first, kept, counts = self.d
        self.hip.device.kv4_keep(self.caches, table, self.table.shape[1], len(self.kept), first, kept, self.stride,
                                 counts, self.max_count)
        return self

    def expected(self):
        page, kv, hd = self.shape
        want = self.raw.copy()
        o = np.arange(page)[:, None]
        codes, pairs = np.arange(hd // 2), np.arange(hd // 8)
        kc, kp, vc, vp, _ = kv4_ref.head_layout(page, hd)
        byte = np.concatenate((kc + o * (hd // 2) + codes, kp + o * (hd // 8) + pairs,
                               vc + (o // 4 * (hd // 4) + codes // 2) * 8 + o % 4 * 2 + codes % 2,
                               vp + (o // 4 * (hd // 16) + pairs // 2) * 8 + o % 4 * 2 + pairs % 2), 1)
        for s, (first, kept) in enumerate(zip(self.firsts, self.kept)):
            if first < 0:
                continue

            def place(p):
                if p // page >= self.table.shape[1]:
                    return None
                at = self.table[s, p // page]
                return (at, byte[p % page]) if 0 <= at < self.pages else None

            def read(p):
                at = place(p)
                return None if at is None else want[:, at[0]][:, :, at[1]].copy()

            def write(p, what):
                at = place(p)
                if at is not None:
                    for layer in range(self.layers):
                        for h in range(kv):
                            want[layer, at[0], h, at[1]] = what[layer, h]

            tree_ref.keep(read, write, first, list(kept), min(self.counts[s], self.max_count))
        return want

    def check(self):
        want = self.expected()
        for layer, d in enumerate(self.d_raw):
            got = d.download(np.uint8, want[layer].size).reshape(want[layer].shape)
            assert np.array_equal(got, want[layer]), (layer, np.argwhere(got != want[layer])[:3])
        return want


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("kv", [1, 3, 8])
def test_paths(hip, hd, page, kv):
    Moves(hip, 1, hd, page, kv, [0, 13, 100, 255],
          [[0, 2, 5, 6], [0, 1, 2], [0, 3, 7, 20, 21, 40], [1, 2, 3, 4, 5]]).upload().launch().check()


@pytest.mark.parametrize("hd", [64, 128])
def test_positions_that_others_come_from(hip, hd):
    """Moves onto places that are sources themselves, over one turn of the
    workgroup and over many."""
    rng = np.random.default_rng(2)
    for n in (2, 15, 16, 17, 31, 32, 33, 64, 65, 300, 1000):
        drop = np.sort(rng.choice(n + 3, n, replace=False))
        Moves(hip, n, hd, 16, 2, [5, 0, 31], [np.arange(1, n + 1), drop, np.arange(n) + 17]).upload().launch().check()


def test_nothing_to_move(hip):
    """Chains whose drafts all stay, empty sequences, and no sequence at all."""
    b = Moves(hip, 3, 128, 16, 2, [9, 40, 3], [[0, 1, 2, 3], [], [0]]).upload().launch()
    assert np.array_equal(b.check(), b.raw)
    b.counts[:] = -1, 0, -2 ** 31
    b.upload().launch()
    assert np.array_equal(b.check(), b.raw)


def test_entries_that_move_nothing(hip):
    """Entries at or below their own place, a negative first, entries past the count."""
    b = Moves(hip, 4, 128, 16, 2, [9, -1, 3, -2 ** 31], [[0, 0, 5, 2, -7, 9], [2, 3], [4, 6, 8], [1, 2]], stride=9)
    b.counts[2] = 2
    b.upload().launch().check()
    b.counts[:] = 6, 2, 2 ** 31 - 1, 2
    b.max_count = 3
    b.upload().launch().check()


def test_pages_that_are_not_there(hip):
    b = Moves(hip, 5, 64, 16, 2, [0, 10, 0], [[20, 40, 60], [20, 25, 60, 61], [3, 70, 75]])
    b.table[0, 0] = -1                     # goes nowhere
    b.table[1, 1] = b.pages                # comes from nowhere
    b.table[2, 4] = 2 ** 31 - 1
    b.upload().launch().check()
    b = Moves(hip, 6, 64, 16, 2, [3, 4], [[1, 2, 3], [5, 9, 10]])
    b.firsts = [2 ** 31 - 1, 2 ** 31 - 3]  # far behind the table
    b.upload().launch()
    assert np.array_equal(b.check(), b.raw)


@pytest.mark.parametrize("layers", [1, 36, 128])
def test_layers(hip, layers):
    Moves(hip, 7, 128, 16, 1, [20, 30], [[0, 4, 5], [2, 9, 11]], layers=layers).upload().launch().check()


def test_many_sequences(hip):
    rng = np.random.default_rng(8)
    kept = [np.sort(rng.choice(12, int(rng.integers(0, 6)), replace=False)) for _ in range(500)]
    Moves(hip, 8, 64, 16, 2, list(rng.integers(0, 40, 500)), kept, layers=3).upload().launch().check()


def test_pages_past_four_gigabytes(hip):
    """The same moves with pages whose byte offsets pass 32 bits."""
    page, kv, hd = 256, 8, 128
    b = Moves(hip, 10, hd, page, kv, [250, 5], [[1, 5, 6, 300, 301], [0, 2, 3]], layers=1, spare=0).upload()
    want = b.launch().check()[0]
    size = hip.device.kv4_page_bytes(page, kv, hd)
    num = (1 << 32) // size + 9
    pages = hip.DeviceArray(num * size)
    for i in range(b.pages):
        pages.upload(b.raw[0, i], (num - 1 - i) * size)
    b.caches = hip.device.kv4_caches([hip.device.kv4_cache(pages, num, page, kv, hd)])
    b.d[0] = hip.DeviceArray.from_numpy(np.where(b.table >= 0, num - 1 - b.table, -1).astype(np.int32))
    b.launch()
    for i in range(b.pages):
        assert np.array_equal(pages.download(np.uint8, size, (num - 1 - i) * size).reshape(want[i].shape), want[i])


def test_graphs(hip):
    """A captured call moves what the buffers say at each replay."""
    stream = hip.device.Stream()
    hip.device.set_stream(stream)
    try:
        b = Moves(hip, 9, 128, 32, 2, [20, 30], [[0, 4, 5], [2, 9, 11]], layers=4).upload()
        graph = hip.device.Graph.capture(b.launch)
        rng = np.random.default_rng(9)
        for _ in range(3):
            b.kept = [np.sort(rng.choice(12, 3, replace=False)) for _ in range(2)]
            b.flat[:] = b.kept
            b.d[2].upload(b.flat)
            graph.launch()
            b.raw = b.check()
        graph.close()
        hip.synchronize()
    finally:
        hip.device.set_stream(None)
        stream.close()
