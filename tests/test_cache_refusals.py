"""What the cache, its attention and the log probabilities refuse on the
host, before anything reaches a GPU (no GPU needed)."""
from __future__ import annotations

import ctypes
import math

import pytest

from omnivoice_b200 import _native as N

A = 1 << 20  # an aligned address that no check before the device's follows


def cache(**change):
    fields = dict(keys=A, values=A, key_scales=A, value_scales=A, page_table=A, pages=4,
                  page_tokens=64, kv_heads=2, head_dim=128, num_seqs=1, max_pages=4)
    fields.update(change)
    return N.KvCache(**fields)


def write(lib, c, **change):
    a = dict(k=A, ld_k=256, v=A, ld_v=256, rows=3, cu=A, starts=A, max_rows=3)
    a.update(change)
    return lib.ov_kv_cache_write(ctypes.byref(c) if c else None, a["k"], a["ld_k"], a["v"],
                                 a["ld_v"], a["rows"], a["cu"], a["starts"], a["max_rows"], None)


def read(lib, c, **change):
    a = dict(k=A, ld_k=256, v=A, ld_v=256, rows=3, cu=A, starts=A, max_rows=3)
    a.update(change)
    return lib.ov_kv_cache_read(ctypes.byref(c) if c else None, a["cu"], a["starts"], a["rows"],
                                a["max_rows"], a["k"], a["ld_k"], a["v"], a["ld_v"], None)


def attend(lib, c, **change):
    a = dict(q=A, ld_q=512, rows=3, cu=A, max_rows=3, lengths=A, max_length=200, heads=4, causal=1,
             scale=0.1, out=A, ld_out=512, workspace=None, bytes=0)
    a.update(change)
    return lib.ov_attention_kv_cache(ctypes.byref(c) if c else None, a["q"], a["ld_q"], a["rows"],
                                     a["cu"], a["max_rows"], a["lengths"], a["max_length"],
                                     a["heads"], a["causal"], a["scale"], a["out"], a["ld_out"],
                                     a["workspace"], a["bytes"], None)


def logprobs(lib, **change):
    a = dict(logits=A, type=N.OV_LOGITS_F32, ld=100, rows=3, codebooks=1, vocab=100, targets=A,
             top_k=5, logprob=A, entropy=A, rank=A, ids=A, tops=A)
    a.update(change)
    return lib.ov_token_logprobs(a["logits"], a["type"], a["ld"], a["rows"], a["codebooks"],
                                 a["vocab"], a["targets"], a["top_k"], a["logprob"], a["entropy"],
                                 a["rank"], a["ids"], a["tops"], None)


def refused(status, word):
    assert status == N.OV_ERR_INVALID
    assert word in N.last_error(), N.last_error()


CACHE = [(dict(head_dim=64), "head_dim"), (dict(page_tokens=48), "page_tokens"),
         (dict(page_tokens=0), "page_tokens"), (dict(kv_heads=0), "kv_heads"),
         (dict(num_seqs=65536), "sequences"), (dict(pages=0), "no pages"),
         (dict(max_pages=0), "no pages"), (dict(pages=1 << 24), "2^31"),
         (dict(max_pages=1 << 25), "2^31"), (dict(keys=None), "keys"),
         (dict(values=A + 8), "values must be 16-byte aligned"), (dict(key_scales=A + 2), "key_scales"),
         (dict(value_scales=None), "value_scales"), (dict(page_table=A + 1), "page_table")]


@pytest.mark.parametrize("call", [write, read, attend])
@pytest.mark.parametrize("change,word", CACHE)
def test_cache_descriptions(native, call, change, word):
    refused(call(native, cache(**change)), word)


@pytest.mark.parametrize("call", [write, read, attend])
def test_no_cache(native, call):
    refused(call(native, None), "cache must not be null")


@pytest.mark.parametrize("call", [write, read])
@pytest.mark.parametrize("change,word", [
    (dict(ld_k=255), "k stride"), (dict(ld_k=248), "k stride"), (dict(ld_v=260), "v stride"),
    (dict(rows=1 << 31), "rows"), (dict(k=None), "k must not be null"), (dict(v=A + 2), "v must be"),
    (dict(cu=None), "cu_rows"), (dict(starts=A + 2), "starts")])
def test_cache_rows(native, call, change, word):
    refused(call(native, cache(), **change), word)


@pytest.mark.parametrize("change,word", [
    (dict(heads=3), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"),
    (dict(heads=2048), "1024"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"), (dict(rows=1 << 31), "rows"),
    (dict(max_length=257), "page table"), (dict(ld_q=504), "q stride"), (dict(ld_q=514), "q stride"),
    (dict(ld_out=128), "out stride"), (dict(q=None), "q must not"), (dict(out=A + 8), "out must"),
    (dict(cu=None), "cu_rows"), (dict(lengths=None), "lengths"), (dict(workspace=A + 4), "workspace")])
def test_attention(native, change, word):
    refused(attend(native, cache(), **change), word)


@pytest.mark.parametrize("change,word", [
    (dict(type=2), "logits type"), (dict(codebooks=0), "codebooks"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 20) + 1, ld=1 << 21), "vocab"), (dict(ld=99), "logits stride"),
    (dict(codebooks=2), "logits stride"), (dict(top_k=33), "top_k"), (dict(vocab=4), "top_k"),
    (dict(rows=1 << 27), "rows"), (dict(logits=None), "logits"), (dict(logits=A + 2), "logits"),
    (dict(targets=None), "targets"), (dict(logprob=None), "logprob"), (dict(entropy=A + 1), "entropy"),
    (dict(rank=A + 2), "rank"), (dict(ids=None), "top_ids"), (dict(tops=None), "top_logprobs")])
def test_logprobs(native, change, word):
    refused(logprobs(native, **change), word)


def test_nothing_to_do_is_no_error(native):
    assert write(native, cache(), rows=0) == 0 and write(native, cache(num_seqs=0)) == 0
    assert read(native, cache(), max_rows=0) == 0
    assert attend(native, cache(), rows=0, q=None) == 0
    assert logprobs(native, rows=0, logits=None) == 0


@pytest.mark.parametrize("page_tokens", [16, 32, 64, 128])
@pytest.mark.parametrize("rows", [1, 3])
def test_lengths_that_the_kernels_sums_would_overflow(native, page_tokens, rows):
    """A page table may name almost 2^31 tokens; lengths stay so far below
    that rounding them up to a step of the kernels holds in 32 bits."""
    tokens = (1 << 31) - page_tokens
    c = cache(page_tokens=page_tokens, max_pages=tokens // page_tokens)
    for length in (tokens, (1 << 31) - 1023):
        if length <= tokens:
            refused(attend(native, c, rows=rows, max_length=length), "max_length")
    # The largest length passes this check and fails a later one.
    refused(attend(native, c, rows=rows, max_length=(1 << 31) - 1024, q=None), "q must not")


@pytest.mark.parametrize("change,word", [(c, w) for c, w in CACHE if not any(
    n in c for n in ("keys", "values", "key_scales", "value_scales", "page_table"))])
def test_no_workspace_size_for_a_cache_that_is_refused(native, change, word):
    """By the same check as the call's, whatever its pointers are."""
    c = cache(**(dict(keys=None, page_table=None) | change))
    assert native.ov_attention_kv_cache_workspace_bytes(ctypes.byref(c), 3, 3, 200, 4) == 0
    assert word in N.last_error(), N.last_error()


def test_no_workspace_size_without_a_cache(native):
    assert native.ov_attention_kv_cache_workspace_bytes(None, 3, 3, 200, 4) == 0
    assert "cache must not be null" in N.last_error()
