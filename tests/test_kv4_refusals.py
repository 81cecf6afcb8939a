"""What the 4-bit cache's and the log probabilities' entry points refuse, on the
host, before anything touches the GPU: each call is a valid one with a single
argument changed."""
from __future__ import annotations

import ctypes

import pytest

import pycitlali
from pycitlali import device

A = 0x10000          # an aligned address nobody reads
INVALID, UNSUPPORTED = 1, 2


def _cache(**kw):
    f = dict(pages=A, num_pages=10, page_size=16, kv_heads=2, head_dim=128)
    f.update(kw)
    return device.kv4_cache(**f)


APPEND = dict(q=A, k=A, v=A, q_stride=1024, kv_stride=256, q_norm=A, k_norm=A, eps=1e-6, rope=A, rope_positions=9,
              positions=A, slots=A, tokens=0, heads=8, q_out=A + 4096, q_out_stride=1024)
READ = dict(slots=A, count=0, k_out=A, v_out=A)
ATTENTION = dict(q=A, q_stride=1024, query_start=None, context_lens=A, page_table=A, pages_per_seq=4, nseq=0,
                 tokens=0, max_query=1, max_context=64, heads=8, workspace=None, workspace_bytes=0, out=A,
                 out_stride=1024)
LOGPROBS = dict(logits=A, kind="fp32", row_stride=1000, rows=0, vocab=1000, tokens=A, logprobs=A, ranks=A, entropies=A,
                top_k=5, top_ids=A, top_logprobs=A, workspace=None, workspace_bytes=0)


def _refused(call, status, *args, **kw):
    with pytest.raises(pycitlali.CitlaliError) as e:
        call(*args, **kw)
    assert e.value.status == status and str(e.value)


CACHES = [(dict(pages=None), INVALID), (dict(num_pages=0), INVALID), (dict(num_pages=-1), INVALID),
          (dict(kv_heads=0), INVALID), (dict(kv_heads=4097), INVALID), (dict(page_size=24), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED),
          (dict(page_size=512), UNSUPPORTED), (dict(page_size=0), UNSUPPORTED), (dict(page_size=-16), UNSUPPORTED),
          (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=256), UNSUPPORTED), (dict(pages=A + 8), INVALID),
          (dict(num_pages=1 << 27), INVALID)]


@pytest.mark.parametrize("change,status", CACHES)
def test_caches(change, status):
    c = _cache(**change)
    _refused(device.kv4_append, status, c, **APPEND)
    _refused(device.kv4_read, status, c, **READ)
    _refused(device.kv4_attention, status, c, **ATTENTION)


def test_calls_of_nothing_launch_nothing():
    device.kv4_append(_cache(), **APPEND)
    device.kv4_append(_cache(), **{**APPEND, "q": None, "q_out": None, "heads": 0})
    device.kv4_read(_cache(), **READ)
    device.kv4_attention(_cache(), **ATTENTION)
    device.token_logprobs(**LOGPROBS)


@pytest.mark.parametrize("change", [
    dict(tokens=-1), dict(heads=-1), dict(heads=5000), dict(k=None), dict(v=None), dict(rope=None),
    dict(positions=None), dict(slots=None), dict(q=None), dict(q_out=None), dict(heads=0), dict(rope_positions=0),
    dict(q_stride=1016), dict(kv_stride=248), dict(q_out_stride=0), dict(q_stride=1028), dict(kv_stride=260),
    dict(q_out_stride=1025), dict(q=A + 2), dict(k=A + 8), dict(v=A + 4), dict(q_out=A + 2), dict(q_norm=A + 2),
    dict(k_norm=A + 8), dict(rope=A + 4), dict(tokens=1 << 24), dict(q_out=A, q_out_stride=2048, tokens=2)])
def test_append(change):
    _refused(device.kv4_append, INVALID, _cache(), **{**APPEND, **change})


@pytest.mark.parametrize("change", [dict(count=-1), dict(slots=None), dict(k_out=None), dict(v_out=None),
                                    dict(k_out=A + 2), dict(v_out=A + 8), dict(count=(1 << 25) + 1)])
def test_read(change):
    _refused(device.kv4_read, INVALID, _cache(), **{**READ, **change})


@pytest.mark.parametrize("change,status", [
    (dict(nseq=-1), INVALID), (dict(tokens=-1), INVALID), (dict(max_query=0), INVALID), (dict(max_context=0), INVALID),
    (dict(heads=0), INVALID), (dict(heads=9), INVALID), (dict(heads=34), UNSUPPORTED), (dict(nseq=1 << 16), INVALID),
    (dict(max_query=1 << 24), INVALID), (dict(max_context=(1 << 26) - 1023, pages_per_seq=1 << 22), INVALID),
    (dict(tokens=1 << 29, query_start=A), INVALID), (dict(q=None), INVALID), (dict(context_lens=None), INVALID), (dict(page_table=None), INVALID),
    (dict(out=None), INVALID), (dict(tokens=3), INVALID), (dict(pages_per_seq=0), INVALID),
    (dict(max_context=65), INVALID), (dict(q_stride=1016), INVALID), (dict(out_stride=8), INVALID),
    (dict(q_stride=1025), INVALID), (dict(out_stride=1028), INVALID), (dict(q=A + 4), INVALID),
    (dict(out=A + 8), INVALID)])
def test_attention(change, status):
    _refused(device.kv4_attention, status, _cache(), **{**ATTENTION, **change})


def test_attention_of_too_many_sequences():
    _refused(device.kv4_attention, INVALID, _cache(kv_heads=256),
             **{**ATTENTION, "heads": 256, "q_stride": 32768, "out_stride": 32768, "nseq": 65535, "tokens": 65535})


def test_attention_workspace():
    """A plan that splits long contexts needs room for its parts, and says so."""
    lib = pycitlali.load()
    need = device.kv4_attention_workspace_bytes(100000, 1, 1, 1, 8, 2, 128)
    call = {**ATTENTION, "nseq": 1, "tokens": 1, "max_context": 100000, "pages_per_seq": 100000 // 16}
    if need:
        _refused(device.kv4_attention, INVALID, _cache(), **{**call, "workspace": A, "workspace_bytes": need - 1})
        _refused(device.kv4_attention, INVALID, _cache(), **{**call, "workspace": None, "workspace_bytes": need})
        _refused(device.kv4_attention, INVALID, _cache(), **{**call, "workspace": A + 4, "workspace_bytes": need})
    for bad in ((0, 1, 1, 1, 8, 2, 128), (9, 0, 1, 1, 8, 2, 128), (9, 1, -1, 1, 8, 2, 128), (9, 1, 1, 1, 9, 2, 128),
                (9, 1, 1, 1, 8, 2, 100), (9, 1, 1, 1, 34, 2, 128), (9, 1, 0, 0, 8, 2, 128),
                (2 ** 31 - 1, 1, 1, 1, 8, 2, 128), (9, 1, 1, 2 ** 31 - 1, 8, 2, 128)):
        assert lib.citlali_hip_kv4_attention_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("change", [
    dict(rows=-1), dict(rows=(1 << 23) + 1), dict(vocab=0),
    dict(vocab=(1 << 30) + 1, row_stride=1 << 31), dict(logits=None), dict(row_stride=999), dict(logits=A + 2),
    dict(kind="fp16", logits=A + 1), dict(tokens=None), dict(tokens=None, logprobs=None), dict(top_k=-1),
    dict(top_k=65), dict(top_ids=None), dict(top_logprobs=None)])
def test_logprobs(change):
    _refused(device.token_logprobs, INVALID, **{**LOGPROBS, **change})


def test_logprobs_type_and_workspace():
    lib = pycitlali.load()
    args = [ctypes.c_void_p(A), 8, 1000, 0, 1000] + [ctypes.c_void_p(A)] * 4 + [0, None, None, None, 0]
    assert lib.citlali_hip_token_logprobs(*args) == INVALID
    need = device.token_logprobs_workspace_bytes(1, 151936, 20)
    if need:
        call = {**LOGPROBS, "rows": 1, "vocab": 151936, "row_stride": 151936, "top_k": 20}
        _refused(device.token_logprobs, INVALID, **{**call, "workspace": A, "workspace_bytes": need - 1})
        _refused(device.token_logprobs, INVALID, **{**call, "workspace": A + 8, "workspace_bytes": need})
    for bad in ((0, 5, 1), ((1 << 23) + 1, 5, 1), (1, 0, 1), (1, 2 ** 31 - 1, 1), (1, 5, -1), (1, 5, 65)):
        assert lib.citlali_hip_token_logprobs_workspace_bytes(*bad) == 0


def test_page_bytes():
    assert device.kv4_page_bytes(16, 8, 128) == 16 * 8 * 160
    assert device.kv4_page_bytes(256, 1, 64) == 256 * 80
    for bad in ((16, 0, 128), (16, 4097, 128), (12, 8, 128), (16, 8, 80), (0, 8, 128), (512, 8, 128)):
        assert device.kv4_page_bytes(*bad) == 0


@pytest.mark.parametrize("args", [(None, 5, 64, 1e4), (A, 0, 64, 1e4), (A, 5, 63, 1e4), (A, 5, 0, 1e4),
                                  (A, 5, 4096, 1e4), (A, 5, 64, 0.0), (A, 5, 64, float("inf")), (A + 4, 5, 64, 1e4),
                                  (A, 2 ** 31 - 1, 64, 1e4)])
def test_rope_table(args):
    _refused(device.rope_table, INVALID, *args)


def test_short_workspaces_are_refused():
    """The sizes that the queries give are what the calls insist on."""
    need = device.kv4_attention_workspace_bytes(100000, 1, 1, 1, 8, 2, 128)
    call = {**ATTENTION, "nseq": 1, "tokens": 1, "max_context": 100000, "pages_per_seq": 100000 // 16}
    assert need > 0 and need % (8 * (128 + 2) * 4) == 0        # parts of 8 heads
    for change in (dict(workspace=A, workspace_bytes=need - 1), dict(workspace=A, workspace_bytes=0),
                   dict(workspace=None, workspace_bytes=need), dict(workspace=A + 4, workspace_bytes=need)):
        _refused(device.kv4_attention, INVALID, _cache(), **{**call, **change})
    need = device.token_logprobs_workspace_bytes(1, 151936, 20)
    call = {**LOGPROBS, "rows": 1, "vocab": 151936, "row_stride": 151936, "top_k": 20}
    assert need > 0 and need % (16 + 8 * 20) == 0              # sums and 20 listed of each piece
    for change in (dict(workspace=A, workspace_bytes=need - 1), dict(workspace=A, workspace_bytes=0),
                   dict(workspace=None, workspace_bytes=need), dict(workspace=A + 8, workspace_bytes=need)):
        _refused(device.token_logprobs, INVALID, **{**call, **change})
