"""Timed operators of a serving step over a paged cache of 4-bit keys and values.

Three kinds of case:

* ``append``    ragged tokens of a step or a prompt: RMSNorm of the query and
  key heads and the rotary position in one pass, keys and values stored in the
  paged cache; the stored values are then read back as fp16;
* ``attention`` causal attention of each sequence's queries over its pages: one
  query per sequence (decode), a few (verifying drafted tokens) or a prompt;
* ``logprobs``  log probability and rank of a given token per row of logits, the
  row's entropy, and its most likely alternatives.

The cache.  A page holds ``page_size`` tokens of every kv head; a kv head's part
of a page is

* K codes   [page_size][head_dim / 2] bytes; 4 bytes hold 8 dims, byte 0 dims
  (0, 2), byte 1 (4, 6), byte 2 (1, 3), byte 3 (5, 7), first dim in the low bits;
* K params  [page_size][head_dim / 32] pairs of fp16 (d, m);
* V codes   [page_size / 4][head_dim / 4][4 tokens][2] bytes, 4 dims in order;
* V params  [page_size / 4][head_dim / 32][d, m][4 tokens] fp16.

32 dims of one token share m = fp16(min) and d = fp16((max - m) / 15); a code is
clamp(round((y - m) / d), 0, 15), 0 where d is 0, and stands for fp16(d code + m).
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
THETA = 1e6
GROUP = 32          # dims that share (d, m)
LIMIT = 61440.0     # values saturate here before they are quantised
VOCAB = 151936


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # the smallest call: one sequence's decode step of a 0.6B-class model
        dict(name="append_one", op="append", tokens=1, heads=16, kv_heads=8, head_dim=128, page=16, norm=True,
             positions=2048),
        # a decode step of many sequences, 8B-class, some rows of the batch unused
        dict(name="append_step", op="append", tokens=250, heads=32, kv_heads=8, head_dim=128, page=16, norm=True,
             positions=32768),
        # a long prompt, 8B-class
        dict(name="append_prompt", op="append", tokens=8192, heads=32, kv_heads=8, head_dim=128, page=64, norm=True,
             positions=32768),
        # one sequence's decode step at a short context: latency
        dict(name="decode_short", op="attention", seqs=1, lo=1024, hi=1024, queries=1, heads=16, kv_heads=8,
             head_dim=128, page=16, spread=1),
        # a serving batch, 8B-class, contexts of usual chats
        dict(name="decode_batch", op="attention", seqs=64, lo=200, hi=4000, queries=1, heads=32, kv_heads=8,
             head_dim=128, page=16, spread=2),
        # long contexts, 8B-class: bound by the cache's bytes
        dict(name="decode_long", op="attention", seqs=16, lo=4096, hi=32768, queries=1, heads=32, kv_heads=8,
             head_dim=128, page=64, spread=3),
        # many short sequences of a small model with heads of 64
        dict(name="decode_hd64", op="attention", seqs=100, lo=150, hi=1500, queries=1, heads=16, kv_heads=8,
             head_dim=64, page=32, spread=4),
        # verifying drafted tokens: up to four queries a sequence, 14B-class (5 heads per kv head)
        dict(name="verify_drafts", op="attention", seqs=24, lo=500, hi=6000, queries=4, heads=40, kv_heads=8,
             head_dim=128, page=16, spread=5),
        # a batch of fresh prompts of unequal length
        dict(name="prompt_batch", op="attention", seqs=6, lo=100, hi=2500, queries=2500, heads=16, kv_heads=8,
             head_dim=128, page=32, spread=6),
        # one chunk of a long prompt behind a long prefix, 8B-class: bound by the matrix products
        dict(name="prompt_long", op="attention", seqs=1, lo=16384, hi=16384, queries=2048, heads=32, kv_heads=8,
             head_dim=128, page=64, spread=7),
        # the picks of one decode step of a small batch
        dict(name="logprobs_step", op="logprobs", rows=8, vocab=VOCAB, half=False, top=20, masked=0.0),
        # scoring a prompt's tokens, logits kept in fp16
        dict(name="logprobs_prompt", op="logprobs", rows=2048, vocab=VOCAB, half=True, top=5, masked=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "logprobs"))
    kv = rng.choice((2, 4, 8))
    hd = rng.choice((64, 128, 128))
    page = rng.choice((16, 32, 64, 128))
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 8192), heads=kv * rng.randrange(1, 9 if kv < 8 else 5), kv_heads=kv,
                    head_dim=hd, page=page, norm=rng.random() < 0.7, positions=_log(rng, 16, 32768))
    if op == "logprobs":
        vocab = rng.choice((_log(rng, 300, VOCAB), VOCAB))
        return dict(op=op, rows=_log(rng, 1, 1500), vocab=vocab, half=rng.random() < 0.5, top=rng.randrange(1, 33),
                    masked=rng.choice((0.0, 0.0, 0.5, 0.99)))
    group = rng.randrange(1, 9)
    seqs = _log(rng, 1, 64)
    hi = _log(rng, 1, max(2, 250000 // seqs if seqs > 8 else 30000))
    queries = rng.choice((1, 1, rng.randrange(2, 9), _log(rng, 9, 1500)))
    if queries > 8:
        seqs = min(seqs, max(1, 2000 // queries))
        hi = min(max(hi, queries), 12000)
        if kv * group > 32:
            group = 32 // kv
    return dict(op=op, seqs=seqs, lo=max(1, hi // rng.choice((1, 4, 20))), hi=hi, queries=queries, heads=kv * group,
                kv_heads=kv, head_dim=hd, page=page, spread=rng.randrange(1 << 20))


def _lengths(c):
    """(context, queries) of each sequence; the queries are the context's last positions."""
    r = random.Random(c["spread"])
    lens = [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]
    lens[0] = c["hi"]
    asked = [c["queries"]] + [r.randint((c["queries"] + 1) // 2, c["queries"]) for _ in lens[1:]]
    if c["lo"] < c["queries"]:       # fresh prompts: every position is a query
        asked = [c["queries"]] * len(lens)
    return lens, [min(n, a) for n, a in zip(lens, asked)]


def work(case):
    c = case
    if c["op"] == "logprobs":
        size = 2 if c["half"] else 4
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size + c["rows"] * (16 + 8 * c["top"]), "flops": 6 * n}
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "append":
        cached = kv * hd * 5 // 4                     # K and V of one token in the cache
        row = 2 * hd * (h + 2 * kv) + 4 * hd + 2 * hd * h + cached
        back = cached + 4 * kv * hd                   # the stored values read back as fp16
        return {"bytes": c["tokens"] * (row + back), "flops": c["tokens"] * hd * (8 * h + 24 * kv)}
    lens, asked = _lengths(c)
    seen = sum(a * n - a * (a - 1) // 2 for n, a in zip(lens, asked))
    return {"bytes": sum(lens) * kv * hd * 5 // 4 + 4 * sum(asked) * h * hd, "flops": 4 * seen * h * hd}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator("cuda").manual_seed(int(seed) * 7919 + 13)


def _rows(g, n, width):
    """Normal activations with about one channel in 50 five times larger."""
    big = (torch.rand(width, generator=g, device="cuda") < 0.02).half() * 4 + 1
    return torch.randn((n, width), generator=g, device="cuda", dtype=torch.float16) * big


def _norm_weight(g, n):
    return (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).half()


def _quantise(y):
    """Codes, d and m of y [..., head_dim] in fp32."""
    y = y.clamp(-LIMIT, LIMIT).unflatten(-1, (-1, GROUP))
    m = y.amin(-1, keepdim=True).half().float()
    d = ((y.amax(-1, keepdim=True) - m) / 15).half().float()
    code = torch.where(d > 0, torch.round((y - m) / d), torch.zeros_like(y)).clamp(0, 15)
    return code, d, m


def _values(code, d, m):
    return (d * code + m).half().flatten(-2)


def _pages(g, pages, page, kv, hd):
    """A cache full of normal keys (some channels larger) and values."""
    parts = []
    per = max(1, (1 << 26) // (page * kv * hd))
    for p0 in range(0, pages, per):
        n = min(per, pages - p0)
        k = _rows(g, n * page * kv, hd).float().view(n, page, kv, hd).transpose(1, 2).contiguous()
        code, d, m = _quantise(k)
        u = code.to(torch.uint8).view(n, kv, page, hd // 8, 4, 2).transpose(-1, -2).reshape(n, kv, page, hd // 8, 4, 2)
        kc = (u[..., 0] | (u[..., 1] << 4)).reshape(n, kv, -1)
        kp = torch.cat((d, m), -1).half().view(n, kv, -1).view(torch.uint8)
        v = torch.randn((n, kv, page, hd), generator=g, device="cuda")
        code, d, m = _quantise(v)
        u = code.to(torch.uint8).view(n, kv, page // 4, 4, hd // 4, 2, 2).transpose(3, 4)
        vc = (u[..., 0] | (u[..., 1] << 4)).reshape(n, kv, -1)
        vp = torch.cat((d, m), -1).half().view(n, kv, page // 4, 4, hd // GROUP, 2).permute(0, 1, 2, 4, 5, 3)
        parts.append(torch.cat((kc, kp, vc, vp.reshape(n, kv, -1).view(torch.uint8)), -1))
    return torch.cat(parts)


def _rope_table(positions, hd):
    """(cos, sin) of every position and pair, from angles in 64 bits."""
    freq = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    r = random.Random(seed * 31 + 5)
    s = {"case": c}
    if c["op"] == "append":
        n, h, kv, hd = c["tokens"], c["heads"], c["kv_heads"], c["head_dim"]
        pages = n // c["page"] + 2
        s["qkv"] = _rows(g, n, (h + 2 * kv) * hd)     # one fused projection's rows
        s["q_norm"], s["k_norm"] = (_norm_weight(g, hd) if c["norm"] else None for _ in range(2))
        s["rope"] = _rope_table(c["positions"], hd)
        s["at"] = torch.randint(0, c["positions"], (n,), generator=g, device="cuda", dtype=torch.int32)
        slots = torch.randperm(pages * c["page"], generator=g, device="cuda")[:n].to(torch.int32)
        if n > 16:                                    # rows of the batch without a token
            slots[n // 3 : n // 3 + 3] = -1
            s["at"][n // 3 + 1 : n // 3 + 3] = -1
        s["slots"] = slots
        s["pages"] = torch.zeros(pages * kv * c["page"] * hd * 5 // 4, dtype=torch.uint8, device="cuda")
        s["q_out"] = torch.zeros((n, h * hd), dtype=torch.float16, device="cuda")
        s["k_out"], s["v_out"] = (torch.zeros((n, kv, hd), dtype=torch.float16, device="cuda") for _ in range(2))
        if own:
            s["cache"] = _hip().kv4_cache(s["pages"].data_ptr(), pages, c["page"], kv, hd)
    elif c["op"] == "attention":
        h, kv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
        lens, asked = _lengths(c)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 1
        order = list(range(pages))
        r.shuffle(order)
        wide = max(need)
        table, at = [], 0
        for n in need:
            table.append(order[at : at + n] + [0] * (wide - n))
            at += n
        start = [0]
        for a in asked:
            start.append(start[-1] + a)
        s["pages"] = _pages(g, pages, page, kv, hd)
        s["table"], s["lens"], s["start"] = _int32(table), _int32(lens), _int32(start)
        s["tokens"], s["max_query"], s["max_context"] = start[-1], max(asked), max(lens)
        s["q"] = _rows(g, start[-1], h * hd)
        s["out"] = torch.zeros((start[-1], h * hd), dtype=torch.float16, device="cuda")
        if own:
            dev = _hip()
            s["cache"] = dev.kv4_cache(s["pages"].data_ptr(), pages, page, kv, hd)
            s["bytes"] = dev.kv4_attention_workspace_bytes(s["max_context"], s["max_query"], c["seqs"], s["tokens"], h,
                                                           kv, hd)
            s["space"] = torch.empty(max(16, s["bytes"]), dtype=torch.uint8, device="cuda")
    else:
        n, v = c["rows"], c["vocab"]
        x = torch.randn((n, v), generator=g, device="cuda") * 2.5
        x[:, : v // 50] += 4                          # frequent tokens
        if c["masked"]:                               # a grammar allows part of the vocabulary
            x.masked_fill_(torch.rand(v, generator=g, device="cuda") < c["masked"], -math.inf)
            x[:, v // 2] = 1.0
        s["logits"] = x.half() if c["half"] else x
        s["tokens"] = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
        if c["masked"]:
            s["tokens"].fill_(v // 2)
        if n > 4:
            s["tokens"][n // 2] = -1                  # a row without a token
        s["logprob"], s["entropy"] = (torch.zeros(n, device="cuda") for _ in range(2))
        s["rank"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        s["top_ids"] = torch.zeros((n, c["top"]), dtype=torch.int32, device="cuda")
        s["top"] = torch.zeros((n, c["top"]), device="cuda")
        if own:
            s["bytes"] = _hip().token_logprobs_workspace_bytes(n, v, c["top"])
            s["space"] = torch.empty(max(16, s["bytes"]), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------- the framework's calls
def _hip():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "citlali-llm-engine_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from pycitlali import device
    return device


def _own_append(s):
    c, dev = s["case"], _hip()
    h, kv, hd, n = c["heads"], c["kv_heads"], c["head_dim"], c["tokens"]
    q = s["qkv"].data_ptr()
    stride = (h + 2 * kv) * hd
    norms = (s["q_norm"].data_ptr(), s["k_norm"].data_ptr()) if c["norm"] else (None, None)
    dev.kv4_append(s["cache"], q, q + 2 * h * hd, q + 2 * (h + kv) * hd, stride, stride, *norms, EPS,
                   s["rope"].data_ptr(), c["positions"], s["at"].data_ptr(), s["slots"].data_ptr(), n, h,
                   s["q_out"].data_ptr(), h * hd)
    dev.kv4_read(s["cache"], s["slots"].data_ptr(), n, s["k_out"].data_ptr(), s["v_out"].data_ptr())
    return s["q_out"], s["k_out"], s["v_out"]


def _own_attention(s):
    c = s["case"]
    width = c["heads"] * c["head_dim"]
    _hip().kv4_attention(s["cache"], s["q"].data_ptr(), width, s["start"].data_ptr(), s["lens"].data_ptr(),
                         s["table"].data_ptr(), s["table"].shape[1], c["seqs"], s["tokens"], s["max_query"],
                         s["max_context"], c["heads"], s["space"].data_ptr(), s["bytes"], s["out"].data_ptr(), width)
    return s["out"]


def _own_logprobs(s):
    c = s["case"]
    _hip().token_logprobs(s["logits"].data_ptr(), "fp16" if c["half"] else "fp32", c["vocab"], c["rows"], c["vocab"],
                          s["tokens"].data_ptr(), s["logprob"].data_ptr(), s["rank"].data_ptr(),
                          s["entropy"].data_ptr(), c["top"], s["top_ids"].data_ptr(), s["top"].data_ptr(),
                          s["space"].data_ptr(), s["bytes"])
    return s["logprob"], s["rank"], s["entropy"], s["top_ids"], s["top"]


# ---------------------------------------------------------------- plain forms
def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _plain_append(s):
    c = s["case"]
    h, kv, hd, n = c["heads"], c["kv_heads"], c["head_dim"], c["tokens"]
    q, k, v = (t.unflatten(-1, (-1, hd)) for t in s["qkv"].split((h * hd, kv * hd, kv * hd), -1))
    at = s["at"].long()
    known = (at >= 0)[:, None, None]
    cos, sin = s["rope"][at.clamp(min=0)][:, None].unbind(-1)

    def head(x, w, wide):
        x = x.to(wide)
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(wide)
        return _rotate(x, cos.to(wide), sin.to(wide))

    q_out = torch.where(known, head(q, s["q_norm"], torch.float32).half(), 0.0).flatten(1)
    # a key next to the border of two codes takes the right one: 64 bits up to the code
    k = head(k, s["k_norm"], torch.float64).float()
    kept = known & (s["slots"] >= 0)[:, None, None]
    return (q_out.half(), torch.where(kept, _values(*_quantise(k)), 0.0).half(),
            torch.where(kept, _values(*_quantise(v.float())), 0.0).half())


def _unpack(pages, table, page, kv, hd):
    """K and V of every sequence as fp32 [seq][kv head][position][head_dim]."""
    n, wide = table.shape
    x = pages[table.long()]
    a, b = page * hd // 2, page * hd // 8
    kc, kp, vc, vp = (t.contiguous() for t in x.split((a, b, a, b), -1))
    u = torch.stack((kc & 15, kc >> 4), -1).view(n, wide, kv, page, hd // 8, 2, 4).transpose(-1, -2)
    p = kp.view(torch.float16).view(n, wide, kv, page, hd // GROUP, 1, 2).float()
    k = _values(u.reshape(n, wide, kv, page, hd // GROUP, GROUP).float(), p[..., 0], p[..., 1])
    u = torch.stack((vc & 15, vc >> 4), -1).view(n, wide, kv, page // 4, hd // 4, 4, 4).transpose(-2, -3)
    p = vp.view(torch.float16).view(n, wide, kv, page // 4, hd // GROUP, 2, 4).permute(0, 1, 2, 3, 6, 4, 5).float()
    v = _values(u.reshape(n, wide, kv, page // 4, 4, hd // GROUP, GROUP).float(), p[..., :1], p[..., 1:])
    return (t.reshape(n, wide, kv, page, hd).transpose(1, 2).reshape(n, kv, wide * page, hd).float() for t in (k, v))


def _plain_attention(s):
    c = s["case"]
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    g = h // kv
    k, v = _unpack(s["pages"], s["table"], c["page"], kv, hd)
    start, lens = s["start"].long(), s["lens"].long()
    asked = start[1:] - start[:-1]
    i = torch.arange(s["max_query"], device="cuda")
    real = i < asked[:, None]                                             # [seq][query]
    row = (start[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"].float().view(-1, kv, g, hd)[row].permute(0, 2, 1, 3, 4)    # [seq][kv][query][g][hd]
    x = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)) * hd ** -0.5
    seen = torch.arange(k.shape[2], device="cuda") < (lens - asked)[:, None, None] + i[:, None] + 1
    x = x.masked_fill(~seen.repeat_interleave(g, 1)[:, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    o = o.unflatten(2, (-1, g)).permute(0, 2, 1, 3, 4).flatten(2)         # [seq][query][h * hd]
    return o[real].half()


def _plain_logprobs(s):
    c = s["case"]
    x, token = s["logits"].float(), s["tokens"].long()
    ids = torch.arange(c["vocab"], device="cuda")
    y = x - x.amax(-1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(-1, keepdim=True)
    y = y - torch.log(total)
    entropy = -(torch.where(e > 0, y, 0.0) * e).sum(-1) / total[:, 0]
    given = token >= 0
    at = token.clamp(min=0)[:, None]
    mine = x.gather(1, at)
    logprob = torch.where(given, y.gather(1, at)[:, 0], 0.0)
    rank = torch.where(given, ((x > mine) | ((x == mine) & (ids < at))).sum(-1), -1).int()
    # ties go to the lowest token: (ordered bits of the logit, complement of the token) as one number
    bits = (x + 0.0).view(torch.int32)
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32) | (0xFFFFFFFF - ids)
    top = 0xFFFFFFFF - (torch.topk(key, c["top"], -1).values & 0xFFFFFFFF)
    return logprob, rank, entropy, top.int(), y.gather(1, top)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "logprobs": _own_logprobs}[op](state)
    return {"append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs}[op](state)


# ---------------------------------------------------------------- in 64 bits
def _exact_append(s):
    c = s["case"]
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].double()
    known = s["at"] >= 0
    freq = THETA ** (-torch.arange(hd // 2, device="cuda").double() * 2 / hd)
    turn = torch.polar(torch.ones_like(freq), s["at"].clamp(min=0).double()[:, None] * freq)[:, None]

    def heads(lo, n, w):
        y = x[:, lo * hd : (lo + n) * hd].reshape(-1, n, hd)
        if w is not None:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / hd + EPS) * w.double()
        z = torch.complex(y[..., : hd // 2].contiguous(), y[..., hd // 2 :].contiguous()) * turn
        return torch.cat((z.real, z.imag), -1)

    def stored(y):
        y = y.reshape(*y.shape[:2], hd // GROUP, GROUP)
        low = y.min(-1).values.half().double()
        step = ((y.max(-1).values - low) / 15).half().double()
        code = torch.round((y - low[..., None]) / step[..., None].clamp(min=1e-30)).clamp(0, 15)
        back = (code * step[..., None] + low[..., None]).half().double().reshape(*y.shape[:2], hd)
        return back * (known & (s["slots"] >= 0))[:, None, None]

    q = heads(0, h, s["q_norm"]).flatten(1) * known[:, None]
    return q, stored(heads(h, kv, s["k_norm"])), stored(x[:, (h + kv) * hd :].reshape(-1, kv, hd))


def _exact_attention(s):
    c = s["case"]
    h, kv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lens, asked = _lengths(c)
    half = s["pages"].view(torch.float16)
    dim = torch.arange(hd, device="cuda")
    out, at = [], 0
    for n, (length, a) in enumerate(zip(lens, asked)):
        t = torch.arange(length, device="cuda")
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
            q = s["q"][at : at + a].double().view(a, h, hd)[:, j * (h // kv) : (j + 1) * (h // kv)]
            for i in range(0, a, 512):                # queries i .. i + 511
                x = q[i : i + 512].reshape(-1, hd) @ k.T / math.sqrt(hd)
                last = length - a + torch.arange(i, min(a, i + 512), device="cuda").repeat_interleave(h // kv)
                x[t > last[:, None]] = -math.inf
                heads.append((torch.softmax(x, -1) @ v).view(-1, h // kv, hd))
        blocks = len(heads) // kv
        out.append(torch.cat([torch.cat(heads[j * blocks : (j + 1) * blocks]) for j in range(kv)], 1).flatten(1))
        at += a
    return torch.cat(out)


def _exact_logprobs(s):
    c = s["case"]
    found = []
    for x, token in zip(s["logits"].split(256), s["tokens"].long().split(256)):
        x = x.double()
        y = x - torch.logsumexp(x, -1, keepdim=True)
        p = torch.exp(y)
        entropy = -torch.where(p > 0, p * y, 0.0).sum(-1)
        mine = torch.where(token >= 0, y.gather(1, token.clamp(min=0)[:, None])[:, 0], 0.0)
        found.append((mine, entropy, torch.sort(y, -1, descending=True).values[:, : c["top"]]))
    logprob, entropy, top = (torch.cat(t) for t in zip(*found))
    return logprob, None, entropy, None, top


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["op"]](s)
