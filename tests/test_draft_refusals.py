"""What the calls on trees of drafted tokens refuse, on the host, before anything
touches the GPU: each call is a valid one with a single argument changed."""
from __future__ import annotations

import ctypes

import pytest

import pycitlali
from pycitlali import device

A = 0x10000          # an aligned address nobody reads
INVALID, UNSUPPORTED = 1, 2

TREE = dict(parents=A, query_start=A, context_lens=A, nseq=0, tokens=0, max_query=8, masks=A, positions=A)
ATTENTION = dict(q=A, q_stride=1024, query_start=A, context_lens=A, masks=A, page_table=A, pages_per_seq=4, nseq=0,
                 tokens=0, max_query=8, max_context=64, heads=8, workspace=None, workspace_bytes=0, out=A,
                 out_stride=1024)
VERIFY = dict(logits=A, kind="fp32", row_stride=1000, vocab=1000, draft_logits=None, draft_row_stride=0, tokens=A,
              parents=A, query_start=A, nseq=0, rows=0, max_query=8, temperatures=A, uniforms=A, paths=A, counts=A,
              next_tokens=A, token_probs=A, workspace=None, workspace_bytes=0)
KEEP = dict(page_table=A, pages_per_seq=4, nseq=0, first=A, kept=A, kept_stride=8, counts=A, max_count=8)


def _cache(**kw):
    return device.kv4_cache(**{**dict(pages=A, num_pages=10, page_size=16, kv_heads=2, head_dim=128), **kw})


def _refused(call, status, *args, **kw):
    with pytest.raises(pycitlali.CitlaliError) as e:
        call(*args, **kw)
    assert e.value.status == status and str(e.value)


def test_calls_of_nothing_launch_nothing():
    device.draft_tree(**TREE)
    device.kv4_tree_attention(_cache(), **ATTENTION)
    device.verify_drafts(**VERIFY)
    device.verify_drafts(**{**VERIFY, "tokens": None, "max_query": 1, "query_start": None})
    device.verify_drafts(**{**VERIFY, "parents": None, "draft_logits": A, "draft_row_stride": 1000, "paths": None,
                            "counts": None, "token_probs": None, "temperatures": None})
    caches = device.kv4_caches([_cache(), _cache(pages=2 * A)])
    device.kv4_keep(caches, **KEEP)
    device.kv4_keep(caches, **{**KEEP, "nseq": 5, "max_count": 0})


@pytest.mark.parametrize("change", [
    dict(nseq=-1), dict(tokens=-1), dict(max_query=0), dict(max_query=257), dict(nseq=1 << 16), dict(parents=None),
    dict(context_lens=None), dict(masks=None), dict(masks=A + 4), dict(query_start=None, tokens=3)])
def test_tree(change):
    _refused(device.draft_tree, INVALID, **{**TREE, **change})


@pytest.mark.parametrize("change,status", [
    (dict(masks=None), INVALID), (dict(masks=A + 4), INVALID), (dict(max_query=257), INVALID),
    (dict(max_query=0), INVALID), (dict(nseq=-1), INVALID), (dict(heads=9), INVALID), (dict(heads=34), UNSUPPORTED),
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(context_lens=None), INVALID),
    (dict(page_table=None), INVALID), (dict(query_start=None, tokens=3), INVALID), (dict(max_context=65), INVALID),
    (dict(q_stride=1016), INVALID), (dict(out_stride=1028), INVALID), (dict(q=A + 4), INVALID)])
def test_attention(change, status):
    _refused(device.kv4_tree_attention, status, _cache(), **{**ATTENTION, **change})


def test_attention_names_itself_and_its_workspace():
    call = {**ATTENTION, "nseq": 1, "tokens": 8, "max_context": 100000, "pages_per_seq": 100000 // 16}
    need = device.kv4_tree_attention_workspace_bytes(100000, 8, 1, 8, 8, 2, 128)
    assert need > 0
    for change in (dict(workspace=A, workspace_bytes=need - 1), dict(workspace=None, workspace_bytes=need),
                   dict(workspace=A + 4, workspace_bytes=need)):
        _refused(device.kv4_tree_attention, INVALID, _cache(), **{**call, **change})
        assert "kv4_tree_attention" in pycitlali.last_error()
    lib = pycitlali.load()
    for bad in ((0, 8, 1, 8, 8, 2, 128), (9, 0, 1, 8, 8, 2, 128), (9, 257, 1, 8, 8, 2, 128), (9, 8, -1, 8, 8, 2, 128),
                (9, 8, 1, 8, 9, 2, 128), (9, 8, 1, 8, 8, 2, 100), (9, 8, 1, 8, 34, 2, 128), (9, 8, 0, 0, 8, 2, 128)):
        assert lib.citlali_hip_kv4_tree_attention_workspace_bytes(*bad) == 0
    for cache in (_cache(page_size=24), _cache(head_dim=96)):
        _refused(device.kv4_tree_attention, UNSUPPORTED, cache, **ATTENTION)


@pytest.mark.parametrize("change", [
    dict(nseq=-1), dict(rows=-1), dict(vocab=0), dict(max_query=0), dict(max_query=257), dict(nseq=1 << 16),
    dict(vocab=(1 << 30) + 1, row_stride=1 << 31), dict(rows=(1 << 24)), dict(logits=None), dict(uniforms=None),
    dict(next_tokens=None), dict(tokens=None), dict(query_start=None, rows=3), dict(row_stride=999),
    dict(draft_logits=A, draft_row_stride=1000), dict(draft_logits=A, draft_row_stride=999, parents=None),
    dict(logits=A + 2), dict(kind="fp16", logits=A + 1),
    dict(draft_logits=A + 2, draft_row_stride=1000, parents=None),
    dict(nseq=65535, max_query=256, vocab=1 << 20, row_stride=1 << 20)])
def test_verify(change):
    _refused(device.verify_drafts, INVALID, **{**VERIFY, **change})


def test_verify_type_and_workspace():
    lib = pycitlali.load()
    p = ctypes.c_void_p(A)
    args = [p, 8, 1000, 1000, None, 0, p, p, p, 0, 0, 8, p, p, p, p, p, p, None, 0]
    assert lib.citlali_hip_verify_drafts(*args) == INVALID
    for parents, drafts in ((A, None), (None, A)):
        need = device.verify_drafts_workspace_bytes(2, 16, 8, 1000, drafts is not None)
        call = {**VERIFY, "nseq": 2, "rows": 16, "parents": parents, "draft_logits": drafts, "draft_row_stride": 1000}
        assert need >= 16 * 16
        for change in (dict(workspace=A, workspace_bytes=need - 1), dict(workspace=A, workspace_bytes=0),
                       dict(workspace=None, workspace_bytes=need), dict(workspace=A + 8, workspace_bytes=need)):
            _refused(device.verify_drafts, INVALID, **{**call, **change})
    for bad in ((-1, 5, 1, 9, 0), (1, -1, 1, 9, 0), (1, 5, 0, 9, 0), (1, 5, 257, 9, 0), (1, 5, 1, 0, 0),
                (1, 5, 1, (1 << 30) + 1, 0), (0, 0, 1, 9, 0), (65535, 5, 256, 1 << 20, 0)):
        assert lib.citlali_hip_verify_drafts_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("change", [
    dict(page_table=None), dict(first=None), dict(kept=None), dict(counts=None), dict(pages_per_seq=0),
    dict(nseq=-1), dict(nseq=1 << 16), dict(max_count=-1), dict(max_count=9),
    dict(max_count=(1 << 30) + 1, kept_stride=1 << 31)])
def test_keep(change):
    _refused(device.kv4_keep, INVALID, device.kv4_caches([_cache()]), **{**KEEP, **change})


@pytest.mark.parametrize("second,status", [
    (dict(pages=None), INVALID), (dict(pages=2 * A + 8), INVALID), (dict(pages=2 * A, num_pages=9), INVALID),
    (dict(pages=2 * A, page_size=32), INVALID), (dict(pages=2 * A, kv_heads=4), INVALID),
    (dict(pages=2 * A, head_dim=64), INVALID), (dict(pages=2 * A, head_dim=96), UNSUPPORTED), (dict(), INVALID)])
def test_keep_of_caches(second, status):
    _refused(device.kv4_keep, status, device.kv4_caches([_cache(), _cache(**second)]), **KEEP)


def test_keep_of_too_many():
    lib = pycitlali.load()
    p = ctypes.c_void_p(A)
    many = device.kv4_caches([_cache(pages=A * (i + 1)) for i in range(129)])
    _refused(device.kv4_keep, INVALID, many, **KEEP)
    assert lib.citlali_hip_kv4_keep(many, 0, p, 4, 0, p, p, 8, p, 8) == INVALID
    assert lib.citlali_hip_kv4_keep(None, 1, p, 4, 0, p, p, 8, p, 8) == INVALID
    _refused(device.kv4_keep, INVALID, device.kv4_caches([_cache(kv_heads=4096)]), **{**KEEP, "nseq": 2049})
