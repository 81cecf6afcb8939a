"""Timed operators of speculative decoding over a paged cache of 4-bit keys and values.

A step drafts a tree of tokens for each sequence, runs the model over all of
them at once, keeps one path and draws the token after it.  Row 0 of a
sequence's tree is the token that the step before ended with; a row's parent is
an earlier row of the same sequence (-1: only the positions before the tree are
above it).  Four kinds of case:

* ``tree``       from the parents: which rows of its tree each row sees, as bits,
  and its position in the text, once a step;
* ``attention``  every row's queries over the positions before the tree and over
  the rows on its own path, whose keys and values are the sequence's last cached
  positions;
* ``verify``     from the logits of every row and one random number a row: the
  path of drafted tokens that stays, the token after it, and the probability of
  every drafted token;
* ``keep``       the path's keys and values moved up behind the positions before
  the tree, in the caches of all layers.

Verification.  p is softmax(logits / temperature) of a row; where the temperature
is not above 0, p is 1 on the largest logit (the lowest id of equal ones).  From
row 0 on, the children of the current row are tried in order: child c with token
x is accepted if u_c R < p(x), where R starts as 1, and becomes the current row.
Else R becomes R - p(x), and p(x) 0.  A sequence's next token comes from what is
left of p at the last row: the first id whose running sum exceeds u_0 times the
total.  With draft logits (chains only) q is their distribution, x is accepted if
u_c q(x) < p(x), and what is left after it is rejected is max(p - q, 0).  Where
nothing is left, p is.

The cache.  A page holds ``page_size`` tokens of every kv head; a kv head's part
of a page is

* K codes   [page_size][head_dim / 2] bytes; 4 bytes hold 8 dims, byte 0 dims
  (0, 2), byte 1 (4, 6), byte 2 (1, 3), byte 3 (5, 7), first dim in the low bits;
* K params  [page_size][head_dim / 32] pairs of fp16 (d, m);
* V codes   [page_size / 4][head_dim / 4][4 tokens][2] bytes, 4 dims in order;
* V params  [page_size / 4][head_dim / 32][d, m][4 tokens] fp16.

A code of 0 .. 15 stands for fp16(d code + m).
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

GROUP = 32          # dims that share (d, m)
VOCAB = 151936
MOST = 256          # rows of a tree


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one sequence's small tree: latency
        dict(name="tree_one", op="tree", seqs=1, nodes=8, spread=1),
        # many sequences with the largest trees
        dict(name="tree_many", op="tree", seqs=128, nodes=256, spread=2),
        # one chat of a 0.6B-class model, a small tree: latency
        dict(name="attend_one", op="attention", seqs=1, lo=1000, hi=1000, nodes=8, heads=16, kv_heads=8, head_dim=128,
             page=16, spread=3),
        # a serving batch, 8B-class, small trees: bound by the cache's bytes
        dict(name="attend_batch", op="attention", seqs=48, lo=200, hi=4000, nodes=12, heads=32, kv_heads=8,
             head_dim=128, page=16, spread=4),
        # few sequences, 14B-class (5 heads per kv head), large trees behind long contexts
        dict(name="attend_long", op="attention", seqs=4, lo=8000, hi=32000, nodes=60, heads=40, kv_heads=8,
             head_dim=128, page=64, spread=5),
        # a small model with heads of 64, trees of unequal size
        dict(name="attend_hd64", op="attention", seqs=25, lo=150, hi=2500, nodes=33, heads=16, kv_heads=8, head_dim=64,
             page=32, spread=6),
        # one sequence, a chain of four drafts taken as given: latency
        dict(name="verify_one", op="verify", seqs=1, nodes=5, vocab=VOCAB, half=False, tree=False, drafted=False,
             heat="warm", spread=7),
        # a serving batch, chains drawn from a draft model whose logits are kept
        dict(name="verify_drawn", op="verify", seqs=40, nodes=6, vocab=VOCAB, half=False, tree=False, drafted=True,
             heat="mixed", spread=8),
        # trees of the most likely tokens, logits in fp16
        dict(name="verify_tree", op="verify", seqs=14, nodes=40, vocab=VOCAB, half=True, tree=True, drafted=False,
             heat="mixed", spread=9),
        # many sequences, short drafts, a vocabulary whose rows start on odd elements
        dict(name="verify_odd", op="verify", seqs=150, nodes=4, vocab=32003, half=True, tree=False, drafted=True,
             heat="mixed", spread=10),
        # a small batch's accepted tokens in the caches of a few layers
        dict(name="keep_path", op="keep", seqs=8, nodes=24, most=5, layers=8, kv_heads=8, head_dim=128, page=16,
             before=150, spread=11),
        # a window's worth of positions moved up after older ones are dropped
        dict(name="keep_window", op="keep", seqs=4, nodes=8000, most=3500, layers=12, kv_heads=8, head_dim=128,
             page=64, before=100, spread=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tree", "attention", "attention", "verify", "verify", "keep"))
    kv, hd, page = rng.choice((2, 4, 8)), rng.choice((64, 128, 128)), rng.choice((16, 32, 64, 128))
    spread = rng.randrange(1 << 20)
    if op == "tree":
        return dict(op=op, seqs=_log(rng, 1, 128), nodes=_log(rng, 1, MOST), spread=spread)
    if op == "attention":
        group = rng.randrange(1, 9)
        nodes = _log(rng, 1, MOST) if rng.random() < 0.3 else _log(rng, 2, 64)
        seqs = _log(rng, 1, 64)
        hi = max(nodes, min(_log(rng, 16, 30000), 100000 // seqs, 200000000 // (seqs * nodes * kv * group)))
        return dict(op=op, seqs=seqs, lo=max(nodes, hi // rng.choice((1, 4, 20))), hi=hi, nodes=nodes,
                    heads=kv * group, kv_heads=kv, head_dim=hd, page=page, spread=spread)
    if op == "verify":
        tree = rng.random() < 0.4
        drafted = not tree and rng.random() < 0.6
        nodes = _log(rng, 2, 100) if tree else rng.randrange(1, 9)
        vocab = rng.choice((_log(rng, 300, VOCAB), VOCAB))
        seqs = max(1, min(_log(rng, 1, 128), 70000000 // (vocab * nodes * (2 if drafted else 1))))
        return dict(op=op, seqs=seqs, nodes=nodes, vocab=vocab, half=rng.random() < 0.5, tree=tree, drafted=drafted,
                    heat=rng.choice(("cold", "warm", "mixed", "mixed")), spread=spread)
    layers = rng.randrange(1, 37)
    if rng.random() < 0.7:
        nodes, seqs = _log(rng, 4, MOST), _log(rng, 1, 64)
    else:
        nodes, seqs = _log(rng, MOST, 6000), _log(rng, 1, 4)
    layers = max(1, min(layers, 400000 // (seqs * nodes)))
    return dict(op=op, seqs=seqs, nodes=nodes, most=min(nodes // 2, 12) if nodes <= MOST else nodes * 2 // 5,
                layers=layers, kv_heads=kv, head_dim=hd, page=page, before=rng.randrange(0, 200), spread=spread)


def _sizes(r, seqs, nodes):
    """Rows of each sequence's tree."""
    return [nodes] + [r.randint((nodes + 1) // 2, nodes) for _ in range(seqs - 1)]


def _tree(r, n):
    """Parents of a tree of n rows, level after level, two to four children a row or so."""
    parents, at = [-1], 0
    for i in range(1, n):
        at = min(i - 1, at + (r.random() < 0.4))
        parents.append(at)
    return parents


def _plan(c):
    """Per sequence: rows, parents, cached positions (the rows' own included), as the case's spread gives them."""
    r = random.Random(c["spread"])
    sizes = _sizes(r, c["seqs"], c["nodes"])
    chain = c["op"] == "verify" and not c["tree"]
    parents = [list(range(-1, n - 1)) if chain else _tree(r, n) for n in sizes]
    lo, hi = c.get("lo", 300), c.get("hi", 3000)
    lens = [hi] + [r.randint(lo, hi) for _ in sizes[1:]]
    return sizes, parents, [max(n, m) for n, m in zip(lens, sizes)]


def _kept(c):
    """Per sequence, the rows that stay, ascending: none of them in a place that one moves to, but those already there."""
    r = random.Random(c["spread"])
    kept = []
    for n in [c["most"]] + [r.randint(c["most"] // 3, c["most"]) for _ in range(c["seqs"] - 1)]:
        stays = min(n, 1)                          # row 0 stays where it is
        kept.append(list(range(stays)) + sorted(r.sample(range(n, c["nodes"]), n - stays)))
    return kept


def work(case):
    c = case
    if c["op"] == "keep":
        moved = sum(max(0, len(k) - 1) for k in _kept(c)) * c["layers"]
        return {"bytes": 2 * moved * c["kv_heads"] * c["head_dim"] * 5 // 4, "flops": moved}
    sizes, parents, lens = _plan(c)
    rows = sum(sizes)
    if c["op"] == "tree":
        return {"bytes": rows * (4 + 4 + 8 * -(-c["nodes"] // 64)) + 8 * c["seqs"], "flops": rows * c["nodes"]}
    if c["op"] == "verify":
        n = rows * c["vocab"]
        if c["drafted"]:
            n += (rows - c["seqs"]) * c["vocab"]       # a sequence's last row has no child
        return {"bytes": n * (2 if c["half"] else 4) + 16 * rows, "flops": 4 * n}
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    seen = 0
    for n, p, length in zip(sizes, parents, lens):
        depth = []
        for a in p:
            depth.append(1 if a < 0 else depth[a] + 1)
        seen += n * (length - n) + sum(depth)
    return {"bytes": sum(lens) * kv * hd * 5 // 4 + 4 * rows * h * hd + 8 * rows * -(-c["nodes"] // 64),
            "flops": 4 * seen * h * hd}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator("cuda").manual_seed(int(seed) * 7919 + 29)


def _rows(g, n, width):
    """Normal activations with about one channel in 50 five times larger."""
    big = (torch.rand(width, generator=g, device="cuda") < 0.02).half() * 4 + 1
    return torch.randn((n, width), generator=g, device="cuda", dtype=torch.float16) * big


def _quantise(y):
    """Codes, d and m of y [..., head_dim] in fp32."""
    y = y.unflatten(-1, (-1, GROUP))
    m = y.amin(-1, keepdim=True).half().float()
    d = ((y.amax(-1, keepdim=True) - m) / 15).half().float()
    return torch.round((y - m) / d).clamp(0, 15).to(torch.uint8), d, m


def _pages(g, pages, page, kv, hd):
    """A cache full of normal keys (some channels larger) and values."""
    parts = []
    per = max(1, (1 << 26) // (page * kv * hd))
    for p0 in range(0, pages, per):
        n = min(per, pages - p0)
        k = _rows(g, n * page * kv, hd).float().view(n, page, kv, hd).transpose(1, 2).contiguous()
        u, d, m = _quantise(k)
        u = u.view(n, kv, page, hd // 8, 4, 2).transpose(-1, -2).reshape(n, kv, page, hd // 8, 4, 2)
        kc = (u[..., 0] | (u[..., 1] << 4)).reshape(n, kv, -1)
        kp = torch.cat((d, m), -1).half().view(n, kv, -1).view(torch.uint8)
        u, d, m = _quantise(torch.randn((n, kv, page, hd), generator=g, device="cuda"))
        u = u.view(n, kv, page // 4, 4, hd // 4, 2, 2).transpose(3, 4)
        vc = (u[..., 0] | (u[..., 1] << 4)).reshape(n, kv, -1)
        vp = torch.cat((d, m), -1).half().view(n, kv, page // 4, 4, hd // GROUP, 2).permute(0, 1, 2, 4, 5, 3)
        parts.append(torch.cat((kc, kp, vc, vp.reshape(n, kv, -1).view(torch.uint8)), -1))
    return torch.cat(parts)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(r, lens, page):
    """Pages in any order for sequences of these lengths: (number of pages, table)."""
    need = [-(-n // page) for n in lens]
    order = list(range(sum(need) + 1))
    r.shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at : at + n] + [0] * (max(need) - n))
        at += n
    return len(order), _int32(table)


def _starts(sizes):
    start = [0]
    for n in sizes:
        start.append(start[-1] + n)
    return start


def _logits(g, rows, vocab):
    """Rows whose most likely tokens take most of the probability, some rows more than others."""
    x = torch.randn((rows, vocab), generator=g, device="cuda") * 2
    at = torch.randint(0, vocab, (rows, 6), generator=g, device="cuda")
    peak = torch.rand((rows, 6), generator=g, device="cuda") * 6 + 8 + math.log(vocab / VOCAB)
    x.scatter_(1, at, peak)
    return x


def _prepare_verify(c, g, s, sizes, parents, start):
    n, v, rows = c["nodes"], c["vocab"], start[-1]
    r = random.Random(c["spread"] + 1)
    heat = [{"cold": 0.0, "warm": 0.8}.get(c["heat"], r.choice((0.0, 0.6, 1.0))) for _ in sizes]
    s["temps"] = torch.tensor(heat, device="cuda")
    kind = torch.half if c["half"] else torch.float32
    x = _logits(g, rows, v)
    near = x + 0.5 * torch.randn((rows, v), generator=g, device="cuda")      # a draft model's
    tokens = torch.randint(0, v, (rows,), generator=g, device="cuda", dtype=torch.int32)
    above = [start[i] + max(p, 0) for i, ps in enumerate(parents) for p in ps]
    child = [0] * rows                                                        # which child of its parent a row is
    seen = {}
    for i, a in enumerate(above):
        child[i] = seen.get(a, 0)
        seen[a] = child[i] + 1
    drawn = [i for i, p in enumerate(p for ps in parents for p in ps) if p >= 0]
    if drawn:
        at = torch.tensor(drawn, device="cuda")
        up = torch.tensor([above[i] for i in drawn], device="cuda")
        if c["drafted"]:                                                      # one drawn from the draft's distribution
            hot = torch.tensor([heat[i] for i, ps in enumerate(parents) for p in ps if p >= 0], device="cuda")[:, None]
            noise = -torch.log(-torch.log(torch.rand((len(drawn), v), generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
            tokens[at] = (near[up].to(kind).float() + hot * noise).argmax(-1).int()
        else:                                                                 # the draft's most likely ones in order
            top = torch.topk(near, min(v, max(child) + 1), -1).indices
            tokens[at] = top[up, torch.tensor([child[i] for i in drawn], device="cuda")].int()
    s["logits"] = x.to(kind)
    s["draft"] = near.to(kind) if c["drafted"] else None
    s["tokens"] = tokens
    s["uniforms"] = torch.rand(rows, generator=g, device="cuda")
    s["parents"] = _int32([p for ps in parents for p in ps]) if c["tree"] else None
    s["paths"] = torch.zeros((c["seqs"], n), dtype=torch.int32, device="cuda")
    s["counts"], s["next"] = (torch.zeros(c["seqs"], dtype=torch.int32, device="cuda") for _ in range(2))
    s["probs"] = torch.zeros(rows, device="cuda")
    if own:
        s["bytes"] = _hip().verify_drafts_workspace_bytes(c["seqs"], rows, n, v, c["drafted"])
        s["space"] = torch.empty(max(16, s["bytes"]), dtype=torch.uint8, device="cuda")


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    r = random.Random(seed * 31 + 7)
    s = {"case": c}
    if c["op"] == "keep":
        kept = _kept(c)
        kv, hd, page = c["kv_heads"], c["head_dim"], c["page"]
        first = random.Random(c["spread"] + 1).choices(range(c["before"] // 2, c["before"] + 1), k=c["seqs"])
        pages, s["table"] = _table(r, [n + c["nodes"] for n in first], page)
        one = _pages(g, pages, page, kv, hd)
        s["pages"] = torch.stack([one.roll(i, 0) for i in range(c["layers"])])
        s["first"], s["counts"] = _int32(first), _int32([len(k) for k in kept])
        s["kept"] = _int32([k + [-1] * (c["most"] - len(k)) for k in kept])
        if own:
            dev = _hip()
            s["caches"] = dev.kv4_caches([dev.kv4_cache(p.data_ptr(), pages, page, kv, hd) for p in s["pages"]])
        return s
    sizes, parents, lens = _plan(c)
    start = _starts(sizes)
    s["start"], s["lens"], s["rows"] = _int32(start), _int32(lens), start[-1]
    words = -(-c["nodes"] // 64)
    if c["op"] == "verify":
        _prepare_verify(c, g, s, sizes, parents, start)
        return s
    if c["op"] == "tree":
        s["parents"] = _int32([p for n in sizes for p in _tree(r, n)])
        s["masks"] = torch.zeros((start[-1], words), dtype=torch.int64, device="cuda")
        s["at"] = torch.zeros(start[-1], dtype=torch.int32, device="cuda")
        return s
    h, kv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    pages, s["table"] = _table(r, lens, page)
    s["pages"] = _pages(g, pages, page, kv, hd)
    s["max_context"] = max(lens)
    s["q"] = _rows(g, start[-1], h * hd)
    s["out"] = torch.zeros((start[-1], h * hd), dtype=torch.float16, device="cuda")
    # the bits that the step's `tree` call gave
    masks = []
    for ps in parents:
        at = len(masks)
        for i, p in enumerate(ps):
            masks.append((0 if p < 0 else masks[at + p]) | 1 << i)
    signed = [[(m >> 64 * w & (1 << 64) - 1) - (1 << 64) * (m >> 64 * w + 63 & 1) for w in range(words)] for m in masks]
    s["masks"] = torch.tensor(signed, dtype=torch.int64, device="cuda")
    if own:
        dev = _hip()
        s["cache"] = dev.kv4_cache(s["pages"].data_ptr(), pages, page, kv, hd)
        s["bytes"] = dev.kv4_tree_attention_workspace_bytes(s["max_context"], c["nodes"], c["seqs"], start[-1], h, kv,
                                                            hd)
        s["space"] = torch.empty(max(16, s["bytes"]), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------- the framework's calls
def _hip():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "citlali-llm-engine_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from pycitlali import device
    return device


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_tree(s):
    c = s["case"]
    _hip().draft_tree(s["parents"].data_ptr(), s["start"].data_ptr(), s["lens"].data_ptr(), c["seqs"], s["rows"],
                      c["nodes"], s["masks"].data_ptr(), s["at"].data_ptr())
    return s["masks"], s["at"]


def _own_attention(s):
    c = s["case"]
    width = c["heads"] * c["head_dim"]
    _hip().kv4_tree_attention(s["cache"], s["q"].data_ptr(), width, s["start"].data_ptr(), s["lens"].data_ptr(),
                              s["masks"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1], c["seqs"], s["rows"],
                              c["nodes"], s["max_context"], c["heads"], s["space"].data_ptr(), s["bytes"],
                              s["out"].data_ptr(), width)
    return s["out"]


def _own_verify(s):
    c = s["case"]
    _hip().verify_drafts(s["logits"].data_ptr(), "fp16" if c["half"] else "fp32", c["vocab"], c["vocab"],
                         _ptr(s["draft"]), c["vocab"], s["tokens"].data_ptr(), _ptr(s["parents"]),
                         s["start"].data_ptr(), c["seqs"], s["rows"], c["nodes"], s["temps"].data_ptr(),
                         s["uniforms"].data_ptr(), s["paths"].data_ptr(), s["counts"].data_ptr(), s["next"].data_ptr(),
                         s["probs"].data_ptr(), s["space"].data_ptr(), s["bytes"])
    return s["paths"], s["counts"], s["next"], s["probs"]


def _own_keep(s):
    c = s["case"]
    _hip().kv4_keep(s["caches"], s["table"].data_ptr(), s["table"].shape[1], c["seqs"], s["first"].data_ptr(),
                    s["kept"].data_ptr(), c["most"], s["counts"].data_ptr(), c["most"])
    return s["pages"]


# ---------------------------------------------------------------- plain forms
def _own_rows(s, n):
    """[seq][n] row numbers and whether the sequence has that many."""
    start = s["start"].long()
    i = torch.arange(n, device="cuda")
    real = i < (start[1:] - start[:-1])[:, None]
    return (start[:-1, None] + i).clamp(max=s["rows"] - 1), real


def _plain_tree(s):
    n = s["case"]["nodes"]
    row, real = _own_rows(s, n)
    i = torch.arange(n, device="cuda")
    parent = torch.where(real, s["parents"].long()[row], -1)
    see = ((parent[..., None] == i) | (i == i[:, None])).float()         # itself and the row above it
    for _ in range(max(1, n - 1).bit_length()):
        see = (torch.matmul(see, see) > 0).float()
    bits = torch.zeros((*see.shape[:2], -(-n // 64) * 64), dtype=torch.int64, device="cuda")
    bits[..., :n] = see.long()
    masks = (bits.unflatten(-1, (-1, 64)) << torch.arange(64, device="cuda")).sum(-1)
    before = s["lens"].long() - real.sum(-1)
    at = before[:, None] + see.sum(-1).long() - 1
    return masks[real], at[real].int()


def _unpack(pages, table, page, kv, hd):
    """K and V of every sequence as fp32 [seq][kv head][position][head_dim]."""
    n, wide = table.shape
    x = pages[table.long()]
    a, b = page * hd // 2, page * hd // 8
    kc, kp, vc, vp = (t.contiguous() for t in x.split((a, b, a, b), -1))
    u = torch.stack((kc & 15, kc >> 4), -1).view(n, wide, kv, page, hd // 8, 2, 4).transpose(-1, -2)
    p = kp.view(torch.float16).view(n, wide, kv, page, hd // GROUP, 1, 2).float()
    k = p[..., 0] * u.reshape(n, wide, kv, page, hd // GROUP, GROUP).float() + p[..., 1]
    u = torch.stack((vc & 15, vc >> 4), -1).view(n, wide, kv, page // 4, hd // 4, 4, 4).transpose(-2, -3)
    p = vp.view(torch.float16).view(n, wide, kv, page // 4, hd // GROUP, 2, 4).permute(0, 1, 2, 3, 6, 4, 5).float()
    v = p[..., :1] * u.reshape(n, wide, kv, page // 4, 4, hd // GROUP, GROUP).float() + p[..., 1:]
    return (t.half().reshape(n, wide, kv, page, hd).transpose(1, 2).reshape(n, kv, wide * page, hd).float()
            for t in (k, v))


def _plain_attention(s):
    c = s["case"]
    h, kv, hd, n = c["heads"], c["kv_heads"], c["head_dim"], c["nodes"]
    g = h // kv
    k, v = _unpack(s["pages"], s["table"], c["page"], kv, hd)
    row, real = _own_rows(s, n)
    before = s["lens"].long() - real.sum(-1)                              # positions that every row sees
    q = s["q"].float().view(-1, kv, g, hd)[row].permute(0, 2, 1, 3, 4)    # [seq][kv][row][g][hd]
    x = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)) * hd ** -0.5
    at = torch.arange(k.shape[2], device="cuda") - before[:, None]        # of the tree's rows
    word = (at.clamp(0, n - 1) // 64)[:, None].expand(-1, n, -1)
    on_path = (s["masks"][row].gather(2, word) >> (at.clamp(0, n - 1) % 64)[:, None]) & 1
    seen = (at < 0)[:, None] | ((at < n)[:, None] & (on_path == 1))
    x = x.masked_fill(~seen.repeat_interleave(g, 1)[:, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    o = o.unflatten(2, (-1, g)).permute(0, 2, 1, 3, 4).flatten(2)         # [seq][row][h * hd]
    return o[real].half()


def _distribution(x, temps):
    """Rows of probabilities in 64 bits: a token next to a border of the running sum has to be the right one."""
    x = x.double()
    top = x.amax(-1, keepdim=True)
    ids = torch.arange(x.shape[-1], device="cuda")
    first = torch.where(x == top, ids, x.shape[-1]).amin(-1, keepdim=True)
    hot = (temps > 0)[:, None]
    e = torch.exp((x - top) / torch.where(hot, temps.double()[:, None], 1.0))
    return torch.where(hot, e / e.sum(-1, keepdim=True), (ids == first).double())


def _plain_verify(s):
    c = s["case"]
    n, seqs = c["nodes"], c["seqs"]
    row, real = _own_rows(s, n)
    owner = torch.searchsorted(s["start"].long()[1:], torch.arange(s["rows"], device="cuda"), right=True)
    temps = s["temps"][owner]
    p = _distribution(s["logits"], temps)
    q = _distribution(s["draft"], temps) if c["drafted"] else None
    token, u = s["tokens"].long()[row], s["uniforms"].double()[row]
    parent = s["parents"].long()[row] if c["tree"] else (torch.arange(n, device="cuda") - 1).expand(seqs, n)
    current = torch.zeros(seqs, dtype=torch.long, device="cuda")
    left = torch.ones(seqs, dtype=torch.float64, device="cuda")
    gone = torch.zeros((seqs, n), dtype=torch.bool, device="cuda")        # rejected children of the current row
    path = torch.full((seqs, n + 1), -1, dtype=torch.long, device="cuda")
    path[:, 0] = 0
    count = torch.ones_like(current)
    for i in range(1, n):
        tried = real[:, i] & (parent[:, i] == current)
        at = row.gather(1, current[:, None])[:, 0]
        again = (gone & (token == token[:, i : i + 1])).any(-1)
        mine = torch.where(again, 0.0, p[at, token[:, i]])
        bar = q[at, token[:, i]] if c["drafted"] else left
        taken = tried & (u[:, i] * bar < mine)
        path.scatter_(1, torch.where(taken, count, n)[:, None], i)
        count += taken
        current = torch.where(taken, i, current)
        left = torch.where(taken, 1.0, torch.where(tried, left - mine, left))
        gone &= ~taken[:, None]
        gone[:, i] = tried & ~taken
    at = row.gather(1, current[:, None])[:, 0]
    rest = p[at]
    if c["drafted"]:
        rest = torch.where(gone.any(-1, keepdim=True), (rest - q[at]).clamp(min=0), rest)
    else:
        # each rejected token is taken out of its own sequence's row; the others write to a spare column
        rest = torch.cat((rest, torch.zeros_like(rest[:, :1])), 1)
        rest.scatter_(1, torch.where(gone, token, c["vocab"]), 0.0)
        rest = rest[:, :-1]
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p[at])
    run_sum = torch.cumsum(rest, -1)
    after = (run_sum <= u[:, :1] * run_sum[:, -1:]).sum(-1)
    above = row.gather(1, parent.clamp(0, n - 1))
    probs = torch.where(parent >= 0, p[above, token], 0.0)[real].float()
    return path[:, :n].int(), count.int(), after.clamp(max=c["vocab"] - 1).int(), probs


def _plain_keep(s):
    c = s["case"]
    page, hd = c["page"], c["head_dim"]
    j = torch.arange(c["most"], device="cuda")
    kept = s["kept"].long()
    moves = (j < s["counts"].long()[:, None]) & (kept != j)
    seq = torch.arange(c["seqs"], device="cuda")[:, None].expand_as(kept)[moves]
    src = (s["first"].long()[:, None] + kept)[moves]
    dst = (s["first"].long()[:, None] + j)[moves]

    def places(position):
        """(page, byte of each of the token's bytes in a head's part)."""
        o = (position % page)[:, None]
        codes, pairs = torch.arange(hd // 2, device="cuda"), torch.arange(hd // 8, device="cuda")
        kc = o * (hd // 2) + codes
        kp = page * hd // 2 + o * (hd // 8) + pairs
        vc = page * hd * 5 // 8 + (o // 4 * (hd // 4) + codes // 2) * 8 + o % 4 * 2 + codes % 2
        vp = page * hd * 9 // 8 + (o // 4 * (hd // 16) + pairs // 2) * 8 + o % 4 * 2 + pairs % 2
        return s["table"].long()[seq, position // page][:, None], torch.cat((kc, kp, vc, vp), 1)

    (p0, b0), (p1, b1) = places(src), places(dst)
    heads = torch.arange(c["kv_heads"], device="cuda")[:, None, None]
    for pages in s["pages"]:
        pages[p1, heads, b1] = pages[p0, heads, b0]
    return s["pages"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"tree": _own_tree, "attention": _own_attention, "verify": _own_verify, "keep": _own_keep}[op](state)
    return {"tree": _plain_tree, "attention": _plain_attention, "verify": _plain_verify, "keep": _plain_keep}[op](state)


# ---------------------------------------------------------------- in 64 bits
def _exact_attention(s):
    c = s["case"]
    h, kv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    sizes, parents, lens = _plan(c)
    half = s["pages"].view(torch.float16)
    dim = torch.arange(hd, device="cuda")
    out, at = [], 0
    for n, (length, ps) in enumerate(zip(lens, parents)):
        t = torch.arange(length, device="cuda")
        seen = torch.ones((len(ps), length), dtype=torch.bool)
        seen[:, length - len(ps) :] = False
        for i, p in enumerate(ps):
            if p >= 0:
                seen[i] |= seen[p]
            seen[i, length - len(ps) + i] = True
        hide = ~seen.cuda().repeat_interleave(h // kv, 0)
        p, o = s["table"][n].long()[t // page][:, None], (t % page)[:, None]
        heads = []
        for j in range(kv):
            byte = o * (hd // 2) + dim // 8 * 4 + dim % 2 * 2 + dim % 8 // 4
            code = (s["pages"][p, j, byte] >> (dim % 4 // 2 * 4)) & 15
            pair = (page * hd // 2 + (o * (hd // GROUP) + dim // GROUP) * 4) // 2
            k = (code.double() * half[p, j, pair].double() + half[p, j, pair + 1].double()).half().double()
            byte = page * hd * 5 // 8 + ((o // 4 * (hd // 4) + dim // 4) * 4 + o % 4) * 2 + dim % 4 // 2
            code = (s["pages"][p, j, byte] >> (dim % 2 * 4)) & 15
            pair = (page * hd * 9 // 8 + (o // 4 * (hd // GROUP) + dim // GROUP) * 16) // 2 + o % 4
            v = (code.double() * half[p, j, pair].double() + half[p, j, pair + 4].double()).half().double()
            q = s["q"][at : at + len(ps)].double().view(-1, h, hd)[:, j * (h // kv) : (j + 1) * (h // kv)]
            x = (q.reshape(-1, hd) @ k.T / math.sqrt(hd)).masked_fill(hide, -math.inf)
            heads.append((torch.softmax(x, -1) @ v).view(-1, h // kv, hd))
        out.append(torch.cat(heads, 1).flatten(1))
        at += len(ps)
    return torch.cat(out)


def _exact_probs(s):
    _, parents, _ = _plan(s["case"])
    start, heat, found = s["start"].tolist(), s["temps"].tolist(), []
    for at, hot, ps in zip(start, heat, parents):
        x = s["logits"][at : at + len(ps)].double()
        token = s["tokens"][at : at + len(ps)].long()
        up = torch.tensor(ps, device="cuda").clamp(min=0)
        if hot > 0:
            p = torch.exp(torch.log_softmax(x / hot, -1)[up, token])
        else:
            best = torch.sort(x, dim=-1, stable=True, descending=True).indices[:, 0]
            p = (best[up] == token).double()
        p[0] = 0.0
        found.append(p)
    return torch.cat(found)


def exact(case, seed):
    """Of the attention and of verification's probabilities; the rest is whole numbers, and bytes that stay as they were."""
    if case["op"] == "attention":
        return _exact_attention(prepare(case, seed))
    return (None, None, None, _exact_probs(prepare(case, seed))) if case["op"] == "verify" else None
