"""Paged key / value cache, what can be checked without a GPU: the index arithmetic with lists that point outside
everything, and every refusal of the entry points (all of them come before anything is enqueued)."""
import ctypes as C
import os
import subprocess
import sys
import tempfile

import pytest

from bolt_amd import capi
from bolt_amd.capi import (DT_BF16, DT_F16, DT_F32, DT_I8, DT_U8_Q, NOT_MATCH, NOT_SUPPORTED, NULL_POINTER, SUCCESS, BoltPagedBatch,
                           BoltPagedKvCache, BoltRotary, lib)

HERE = os.path.dirname(os.path.abspath(__file__))
P = 0x10000  # stands for a device address: a refused call looks at it and follows it nowhere


def test_index_arithmetic_on_the_host():
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "check")
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                               os.path.join(HERE, "paged_index_check.cpp"), "-o", exe])
        assert subprocess.check_output([exe]).decode() == "ok\n"


def test_index_arithmetic_reads_nothing_outside_its_lists():
    """the same program with address checks: offsets, lengths and table rows are on the heap there"""
    with tempfile.TemporaryDirectory() as d:
        exe = os.path.join(d, "check")
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                               os.path.join(HERE, "paged_index_check.cpp"), "-o", exe])
        assert subprocess.check_output([exe]).decode() == "ok\n"


def pool(**kw):
    c = BoltPagedKvCache(DT_F16, 10, 16, 2, 64, P, P, None, None)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def rows(offsets=P, **kw):
    b = BoltPagedBatch(3, 4, 5 if offsets else 3, P, P, offsets)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def rotary(**kw):
    r = BoltRotary(64, 64, 0, P, P)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def append(c=None, b=None, dt=DT_F16, k=P, ks=128, v=P, vs=128, heads=4, q=P, qs=256, qo=2 * P, qos=256, r=None):
    return lib().bolt_gfx950_kv_cache_append(c or pool(), b or rows(), dt, k, ks, v, vs, heads, q, qs, qo, qos, r)


def attend(prompt, c=None, b=None, dt=DT_F16, heads=4, q=P, qs=256, out=2 * P, os_=256, scale=0.125, window=0, ws=P, n=None):
    c, b = c or pool(), b or rows(P if prompt else None)
    fn = lib().bolt_gfx950_paged_attention_prompt if prompt else lib().bolt_gfx950_paged_attention_decode
    return fn(c, b, dt, heads, q, qs, out, os_, scale, window, ws, 1 << 40 if n is None else n)


CALLS = [append, lambda **kw: attend(False, **kw), lambda **kw: attend(True, **kw)]


@pytest.mark.parametrize("call", CALLS, ids=["append", "decode", "prompt"])
def test_refusals_of_the_cache_and_the_types(call):
    for c in (pool(k=None), pool(v=None), pool(dt=DT_I8), pool(dt=DT_I8, kScale=P)):
        assert call(c=c) == NULL_POINTER
    for c in (pool(dt=DT_F32), pool(dt=DT_U8_Q), pool(headDim=0), pool(headDim=96), pool(headDim=256), pool(pageSize=0), pool(pageSize=24),
              pool(pageSize=8192), pool(kvHeads=0), pool(kvHeads=2000), pool(numPages=0), pool(numPages=1 << 31), pool(k=P + 8),
              pool(v=P + 2), pool(dt=DT_I8, kScale=P + 2, vScale=P)):
        assert call(c=c) == NOT_SUPPORTED and lib().bolt_gfx950_last_error()
    for dt, cache in ((DT_F32, DT_BF16), (DT_F16, DT_BF16), (DT_BF16, DT_F16), (DT_I8, DT_I8), (DT_U8_Q, DT_F16), (99, DT_F16)):
        assert call(c=pool(dt=cache, kScale=P, vScale=P), dt=dt) == NOT_SUPPORTED


@pytest.mark.parametrize("call", CALLS, ids=["append", "decode", "prompt"])
def test_refusals_of_rows_and_heads(call):
    assert call(heads=3) == NOT_MATCH                      # 2 key heads
    assert call(heads=16386) == NOT_SUPPORTED
    assert call(qs=255) == NOT_MATCH and call(q=None) == NULL_POINTER and call(q=P + 8) == NOT_SUPPORTED
    assert call(qs=260) == NOT_SUPPORTED                   # 520 bytes between rows
    assert call(qs=0) == NOT_MATCH
    offsets = None if call is CALLS[1] else P
    for b in (rows(offsets, pageTable=None), rows(offsets, lengths=None)):
        assert call(b=b) == NULL_POINTER
    for b in (rows(offsets, batch=65536, numTokens=65536), rows(offsets, maxPages=0), rows(offsets, maxPages=1 << 27), rows(offsets, pageTable=P + 1),
              rows(offsets, lengths=P + 2)):
        assert call(b=b) == NOT_SUPPORTED
    assert call(b=rows(P, numTokens=1 << 31)) == NOT_SUPPORTED
    assert call(b=rows(None, numTokens=4)) == NOT_MATCH    # 3 sequences, one row each


def test_refusals_of_append():
    for kw in ({"k": None}, {"v": None}, {"q": None}, {"qo": None}):
        assert append(**kw) == NULL_POINTER
    assert append(ks=127) == NOT_MATCH and append(vs=64) == NOT_MATCH and append(qos=200) == NOT_MATCH
    assert append(k=P + 4) == NOT_SUPPORTED and append(vs=132) == NOT_SUPPORTED and append(qo=P + 2) == NOT_SUPPORTED
    assert append(qo=P, qos=512) == NOT_MATCH              # in place with another stride
    for r in (rotary(cosine=None), rotary(sine=None)):
        assert append(r=r) == NULL_POINTER
    for r in (rotary(dim=0), rotary(dim=8), rotary(dim=72), rotary(dim=128), rotary(cosine=P + 4), rotary(sine=P + 8)):
        assert append(r=r) == NOT_SUPPORTED


@pytest.mark.parametrize("prompt", [False, True])
def test_refusals_of_attention(prompt):
    assert attend(prompt, heads=0) == NOT_SUPPORTED
    assert attend(prompt, out=None) == NULL_POINTER and attend(prompt, ws=None) == NULL_POINTER
    assert attend(prompt, out=P) == NOT_SUPPORTED          # over q
    assert attend(prompt, os_=128) == NOT_MATCH and attend(prompt, out=P + 8) == NOT_SUPPORTED
    assert attend(prompt, ws=P + 16) == NOT_SUPPORTED and attend(prompt, n=0) == NOT_MATCH
    n = C.c_size_t(0)
    b = rows(P if prompt else None)
    assert lib().bolt_gfx950_paged_attention_workspace_bytes(pool(), b, 4, C.byref(n)) == SUCCESS and n.value > 0
    assert attend(prompt, n=n.value - 1) == NOT_MATCH
    assert attend(False, b=rows(P)) == NOT_MATCH           # decode has no offsets,
    assert attend(True, b=rows(None)) == NULL_POINTER      # prompt needs them


def test_more_row_tiles_than_a_launch_can_have():
    """128 rows to a workgroup of 256 threads, fewer than 2^32 threads to a launch: fewer than 2^24 (rows * heads / 128 + batch * key
    heads)"""
    n = C.c_size_t(0)
    size = lib().bolt_gfx950_paged_attention_workspace_bytes
    for batch, tokens, kv, heads, code in ((65535, 65535, 512, 512, NOT_SUPPORTED), (65535, 65535, 254, 254, SUCCESS), (1, 1 << 27, 16, 16, NOT_SUPPORTED),
                                           (1, (1 << 27) - 4096, 16, 16, SUCCESS)):
        b = rows(P, batch=batch, numTokens=tokens)
        assert size(pool(kvHeads=kv), b, heads, C.byref(n)) == code
        if code:
            assert attend(True, c=pool(kvHeads=kv), b=b, heads=heads, qs=heads * 64, os_=heads * 64) == code


def test_nothing_to_do_is_success():
    for b in (rows(P, batch=0, numTokens=0), rows(P, numTokens=0), rows(P, batch=0)):
        assert append(b=b) == SUCCESS and attend(True, b=b) == SUCCESS
    assert attend(False, b=rows(None, batch=0, numTokens=0)) == SUCCESS
    assert append(b=rows(None, batch=0, numTokens=0), k=None, v=None, q=None, qo=None) == SUCCESS


def test_workspace_query_refuses_what_the_calls_refuse():
    f, n = lib().bolt_gfx950_paged_attention_workspace_bytes, C.c_size_t(0)
    assert f(pool(), rows(), 4, None) == NULL_POINTER and f(pool(k=None), rows(), 4, C.byref(n)) == NULL_POINTER
    assert f(pool(), rows(), 5, C.byref(n)) == NOT_MATCH and f(pool(headDim=32), rows(), 4, C.byref(n)) == NOT_SUPPORTED
    assert f(pool(), None, 4, C.byref(n)) == NULL_POINTER


def test_host_mirror_refuses_what_the_library_cannot_see():
    import torch
    from bolt_amd import host_paged as hp
    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    for args in ((k, k.float()), (k[:, :, ::2], k[:, :, ::2]), (k.to(torch.int8), k.to(torch.int8)), (k[0], k[0]), (k, k)):
        with pytest.raises(capi.BoltError):   # the last: not on a GPU
            hp.PagedKvCache(*args)
    t, n = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for args in ((t.long(), n), (t, n.long()), (t[:2], n), (t, n, torch.zeros(3, dtype=torch.int32), 3), (t, n, torch.zeros(4, dtype=torch.int32)), (t, n)):
        with pytest.raises(capi.BoltError):
            hp.PagedBatch(*args)
    with pytest.raises(capi.BoltError):
        hp.Rotary(torch.zeros(4, 8), torch.zeros(4, 7))
