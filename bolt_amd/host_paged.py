"""Host-side mirrors of the paged key / value cache entry points on torch CUDA tensors: append with position rotation,
attention of one new token per sequence, attention of prompts. All arithmetic is in libbolt_gfx950.so; the calls enqueue
on the library's stream (bolt_gfx950_set_stream) and return. What they allocate belongs to that stream. For inference:
nothing is recorded for a gradient.

    cache = PagedKvCache(k, v)                                   # [pages, kv_heads, page_size, head_dim]
    batch = PagedBatch(page_table, lengths)                      # lengths include the new tokens
    q = kv_cache_append(cache, batch, k_new, v_new, q_new, Rotary(cos, sin))
    out = paged_attention_decode(cache, batch, q, workspace=paged_attention_workspace(cache, batch, heads))
"""
import ctypes as C
import math

import torch

from . import capi
# (torch._C: what torch.cuda.current_device() and current_stream() wrap; a call on a decoder's path costs the host 8 us)
from .capi import BoltError, BoltPagedBatch, BoltPagedKvCache, BoltRotary, check, lib

DT_OF = {torch.float32: capi.DT_F32, torch.float16: capi.DT_F16, torch.bfloat16: capi.DT_BF16, torch.int8: capi.DT_I8}


def _want(ok, why):
    if not ok:
        raise BoltError(why)


def _list32(t, name, shape):
    _want(t.dtype == torch.int32 and t.is_contiguous() and tuple(t.shape) == shape, "%s: contiguous int32 %s" % (name, list(shape)))


class PagedKvCache:
    """k, v: contiguous [pages, kv_heads, page_size, head_dim] of float16, bfloat16 or int8; int8 with fp32 scales
    [pages, kv_heads, page_size] (stored = real * scale). The tensors are updated in place."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _want(k.dtype in DT_OF and k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.is_contiguous() and v.is_contiguous(),
              "k and v: contiguous [pages, kv_heads, page_size, head_dim] of one type")
        for s in (k_scale, v_scale):
            _want((s is None) == (k.dtype != torch.int8), "an int8 cache has scales, another has none")
            _want(s is None or (s.dtype == torch.float32 and s.is_contiguous() and s.shape == k.shape[:3]),
                  "scales: contiguous float32 [pages, kv_heads, page_size]")
        self.keep = (k, v, k_scale, v_scale)
        self.device = _one_device(*self.keep)
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.scale = 1.0 / math.sqrt(self.head_dim)
        self.struct = BoltPagedKvCache(DT_OF[k.dtype], self.pages, self.page_size, self.kv_heads, self.head_dim, k.data_ptr(), v.data_ptr(),
                                       None if k_scale is None else k_scale.data_ptr(), None if v_scale is None else v_scale.data_ptr())
        self.ref = C.byref(self.struct)


class PagedBatch:
    """page_table: int32 [batch, max_pages]; lengths: int32 [batch], the new tokens included; offsets: int32 [batch + 1], the
    first packed row of every sequence's new tokens, with `rows` rows in all (at least offsets[batch]); None: one new token
    per sequence. The contents may change between calls and between replays of a captured graph."""

    def __init__(self, page_table, lengths, offsets=None, rows=None):
        batch = lengths.shape[0]
        _want(page_table.dim() == 2, "page_table: [batch, max_pages]")
        _list32(page_table, "page_table", (batch, page_table.shape[1]))
        _list32(lengths, "lengths", (batch,))
        if offsets is not None:
            _list32(offsets, "offsets", (batch + 1,))
            _want(rows is not None, "rows: how many packed rows the buffers have")
        self.keep = (page_table, lengths, offsets)
        self.device = _one_device(*self.keep)
        self.rows = batch if rows is None else int(rows)
        self.struct = BoltPagedBatch(batch, page_table.shape[1], self.rows, page_table.data_ptr(), lengths.data_ptr(),
                                     None if offsets is None else offsets.data_ptr())
        self.ref = C.byref(self.struct)


class Rotary:
    """cos, sin: contiguous float32 [positions, dim / 2]."""

    def __init__(self, cos, sin, interleaved=False):
        _want(cos.dim() == 2 and cos.shape == sin.shape and all(t.dtype == torch.float32 and t.is_contiguous() for t in (cos, sin)),
              "cos and sin: contiguous float32 [positions, dim / 2]")
        self.keep = (cos, sin)
        self.device = _one_device(cos, sin)
        self.struct = BoltRotary(2 * cos.shape[1], cos.shape[0], int(bool(interleaved)), cos.data_ptr(), sin.data_ptr())
        self.ref = C.byref(self.struct)


def _one_device(*tensors):
    found = {t.device for t in tensors if t is not None}
    _want(len(found) == 1 and next(iter(found)).type == "cuda", "tensors of one GPU")
    return next(iter(found))


def _empty(shape, dtype, device):
    """A new tensor that the library's stream uses. torch hands memory out again in the order of the stream it was allocated on, so
    it is allocated on that one; and the stream that is current in torch has to be done with it, too, before it is."""
    ours = lib().bolt_gfx950_get_stream() or 0
    if ours == torch._C._cuda_getCurrentRawStream(device.index):
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(torch.cuda.ExternalStream(ours, device) if ours else torch.cuda.default_stream(device)):
        t = torch.empty(shape, dtype=dtype, device=device)
    t.record_stream(torch.cuda.current_stream(device))
    return t


def _rows(t, name, shape, dtype, device):
    """Checks rows of heads, [rows, heads, dim] with dense heads; returns the elements between rows. (On the path of every call:
    no message is made before it is needed.)"""
    if t.shape != shape or t.dtype != dtype or t.device != device:
        raise BoltError("%s: %s %s on %s, not %s %s on %s" % (name, list(shape), dtype, device, list(t.shape), t.dtype, t.device))
    s = t.stride()
    if s[2] != 1 or (s[1] != shape[2] and shape[1] != 1):
        raise BoltError("%s: the heads of a row are dense" % name)
    if shape[0] < 2:
        return shape[1] * shape[2]
    if s[0] > 0xffffffff:  # (ctypes would pass its low 32 bits)
        raise BoltError("%s: rows are fewer than 2^32 elements apart" % name)
    return s[0]


def _here(cache, batch):
    if cache.device != batch.device or cache.device.index != torch._C._cuda_getDevice():
        raise BoltError("cache and batch belong to the current GPU")


def kv_cache_append(cache, batch, k, v, q=None, rotary=None, q_out=None):
    """k, v: [rows, kv_heads, head_dim], q: [rows, heads, head_dim], rows any number of elements apart. Returns q_out, the
    rotated queries (None without q). Rows that belong to no sequence, or whose position lies behind the angles, are left as they are
    in q_out (where the call makes q_out, they hold anything): the angles have to reach as far as the lengths do."""
    _here(cache, batch)
    device, dtype, shape = cache.device, k.dtype, (batch.rows, cache.kv_heads, cache.head_dim)
    if rotary is not None and rotary.device != device:
        raise BoltError("the angles are on the cache's GPU")
    dt = DT_OF.get(dtype)
    if dt is None:
        raise BoltError("float32, float16 or bfloat16 rows")
    ks, vs = _rows(k, "k", shape, dtype, device), _rows(v, "v", shape, dtype, device)
    heads, qs, qo, qp, qop = 0, 0, 0, None, None
    if q is not None:
        if q.dim() != 3:
            raise BoltError("q: [rows, heads, head_dim]")
        heads = q.shape[1]
        shape = (shape[0], heads, shape[2])
        qs = _rows(q, "q", shape, dtype, device)
        if q_out is None:
            q_out = _empty(shape, dtype, device)
            qo = heads * shape[2]
        else:
            qo = _rows(q_out, "q_out", shape, dtype, device)
        qp, qop = q.data_ptr(), q_out.data_ptr()
    code = lib().bolt_gfx950_kv_cache_append(cache.ref, batch.ref, dt, k.data_ptr(), ks, v.data_ptr(), vs, heads, qp, qs, qop, qo,
                                             None if rotary is None else rotary.ref)
    if code:
        check(code, "kv_cache_append")
    return q_out


def paged_attention_workspace(cache, batch, heads):
    """Device memory for the attention calls of this cache and batch shape; calls that may overlap need one each."""
    n = C.c_size_t(0)
    check(lib().bolt_gfx950_paged_attention_workspace_bytes(cache.ref, batch.ref, heads, C.byref(n)), "paged_attention_workspace_bytes")
    return _empty(n.value, torch.uint8, cache.device)


def _attention(fn, what, cache, batch, q, out, scale, window, workspace):
    _here(cache, batch)
    device, dtype = cache.device, q.dtype
    dt = DT_OF.get(dtype)
    if dt is None or q.dim() != 3:
        raise BoltError("q: [rows, heads, head_dim] of float32, float16 or bfloat16")
    if not 0 <= window <= 0xffffffff:
        raise BoltError("window: 0 (every key) to 2^32 - 1 keys")
    heads = q.shape[1]
    shape = (batch.rows, heads, cache.head_dim)
    qs = _rows(q, "q", shape, dtype, device)
    if workspace is None:
        workspace = paged_attention_workspace(cache, batch, heads)
    elif workspace.dtype != torch.uint8 or workspace.device != device or not workspace.is_contiguous():
        raise BoltError("workspace: contiguous uint8 on the cache's GPU")
    if out is None:
        out, os = _empty(shape, dtype, device), heads * shape[2]
    else:
        os = _rows(out, "out", shape, dtype, device)
    code = fn(cache.ref, batch.ref, dt, heads, q.data_ptr(), qs, out.data_ptr(), os, cache.scale if scale is None else scale, window,
              workspace.data_ptr(), workspace.numel())
    if code:
        check(code, what)
    return out


def paged_attention_decode(cache, batch, q, out=None, scale=None, window=0, workspace=None):
    """One new token per sequence (batch without offsets): q and out [batch, heads, head_dim]. scale: 1 / sqrt(head_dim)."""
    return _attention(lib().bolt_gfx950_paged_attention_decode, "paged_attention_decode", cache, batch, q, out, scale, window, workspace)


def paged_attention_prompt(cache, batch, q, out=None, scale=None, window=0, workspace=None):
    """Any number of new tokens per sequence (batch with offsets): q and out [rows, heads, head_dim]. Rows that belong to no
    sequence are left as they are."""
    return _attention(lib().bolt_gfx950_paged_attention_prompt, "paged_attention_prompt", cache, batch, q, out, scale, window, workspace)
