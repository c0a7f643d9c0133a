"""Serving operators: rows in a paged key-value cache, and the attention of one new token per sequence over it.

They take over where ``optimized_attention`` ends: its prepared keys (``kn``) and values, or a projection's raw ones, go
into the cache with ``append_rows``; each generated token is one ``decode_step`` (or ``append_rows`` and
``decode_attention``); ``read_rows`` gives cached rows back as [B, Hkv, S, D].  Asynchronous calls on the current stream,
capturable into CUDA graphs: lengths and page tables are read on the device, so a captured step follows them.

The cache is two pools of pages [n_pages, Hkv, page_size, D] (``PagedCache``) and an int32 table [B, max_pages]: row p of
sequence b lies in row p % page_size of page ``pages[b, p // page_size]``.  Sequences may share pages that they only read.
An e4m3 cache halves what a step reads: each row is e4m3 values times one power of two, kept as an exponent byte.

K rows and queries are normed (``gk`` / ``gq``; None: not) and rotated (``cos`` and ``sin`` [positions, D]; None: not) in
fp32 and rounded once; ``optimized_attention`` rounds at every step of its reference's contract, so rows that have to equal
its ``kn`` bit for bit are appended from ``kn``, with ``gk`` and the tables left out.

Lengths and tables on the device are not looked at by the host.  A table entry outside the cache, a length or position
that the table cannot hold or one behind the rotary tables is reported through the status word (``check_status`` raises);
nothing is read or written out of bounds.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from .api import _DTYPES, _call, _major, _on_device, _raw_stream, status_word

_CACHE_DTYPES = {**_DTYPES, torch.float8_e4m3fn: _lib.KF_E4M3}
# The structs of include/kf_b200.h: 8-byte fields throughout.
_CACHE = "5P17q"
_APPEND = struct.Struct("@" + _CACHE + "8P10qd")
_READ = struct.Struct("@" + _CACHE + "4P9q")
_DECODE = struct.Struct("@" + _CACHE + "11P12q2d")


class PagedCache(NamedTuple):
    """The pools of a cache: ``k`` and ``v`` [n_pages, Hkv, page_size, D], and for an e4m3 cache ``k_scale`` and
    ``v_scale`` [n_pages, Hkv, page_size] (float8_e8m0fnu).  The operators take any (k, v) or (k, v, k_scale, v_scale)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None

    @classmethod
    def allocate(cls, n_pages, page_size, kv_heads, head_dim, dtype=torch.bfloat16, device="cuda"):
        """Pools of the given sizes, not cleared; ``dtype`` torch.bfloat16, torch.float16 or torch.float8_e4m3fn."""
        if dtype not in _CACHE_DTYPES:
            raise ValueError("Expected a BF16, FP16 or float8_e4m3fn cache")
        k, v = (torch.empty(n_pages, kv_heads, page_size, head_dim, dtype=dtype, device=device) for _ in range(2))
        if dtype != torch.float8_e4m3fn:
            return cls(k, v)
        return cls(k, v, *(torch.empty(n_pages, kv_heads, page_size, dtype=torch.float8_e8m0fnu, device=device)
                           for _ in range(2)))


def _cache_fields(cache, pages, b, dtype, index):
    """The kf_paged_cache of a call, after the checks that need no device."""
    if len(cache) == 2:
        (k, v), ks, vs = cache, None, None
    else:
        k, v, ks, vs = cache
    if k.ndim != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _CACHE_DTYPES:
        raise ValueError("Expected cache pools [n_pages, Hkv, page_size, D] of one type (BF16, FP16 or float8_e4m3fn)")
    n, h, page, d = k.shape
    if d not in (128, 256) or n < 1 or h < 1 or page < 16 or page % 16:
        raise ValueError("Expected D=128/256 and a page size that is a multiple of 16")
    e8 = k.dtype == torch.float8_e4m3fn
    if not e8 and k.dtype != dtype:
        raise ValueError("Expected a cache of the tensors' type, or of float8_e4m3fn")
    if pages.ndim != 2 or pages.shape[0] != b or pages.shape[1] < 1 or pages.dtype != torch.int32 or (
            pages.shape[1] > 1 and pages.stride(1) != 1):
        raise ValueError("Expected an int32 page table [B, max_pages] with contiguous rows")
    ok = k.is_cuda and k.get_device() == index and v.get_device() == index and pages.get_device() == index
    sk, sv = k.stride(), v.stride()
    ok = ok and sk[3] == 1 and sv[3] == 1
    scale = (0, 0, 0, 0)
    if e8:
        if ks is None or vs is None or ks.shape != k.shape[:3] or vs.shape != k.shape[:3] or (
                ks.dtype != torch.float8_e8m0fnu or vs.dtype != torch.float8_e8m0fnu):
            raise ValueError("Expected float8_e8m0fnu scales [n_pages, Hkv, page_size] with an e4m3 cache")
        ok = ok and ks.get_device() == index and vs.get_device() == index and ks.stride(2) == 1 and vs.stride(2) == 1
        scale = ks.stride()[:2] + vs.stride()[:2]
    elif ks is not None or vs is not None:
        raise ValueError("Scales belong to an e4m3 cache only")
    if not ok:
        raise ValueError("The cache and its table must lie on the tensors' CUDA device, with contiguous rows")
    return (k.data_ptr(), v.data_ptr(), ks.data_ptr() if e8 else 0, vs.data_ptr() if e8 else 0, pages.data_ptr(),
            pages.stride(0), n, pages.shape[1], page, h, d, _CACHE_DTYPES[k.dtype], *sk[:3], *sv[:3], *scale)


def _check_ints(name, t, b, index):
    if t.dtype != torch.int32 or t.shape != (b,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"Expected {name} as contiguous int32 [B] on the tensors' CUDA device")


def _check_rows(tensors):
    """Every tensor in rows of a contiguous head dimension, on one CUDA device that is a B200, in one 16-bit type."""
    first = tensors[0]
    dtype, index = first.dtype, first.get_device()
    ok = dtype in _DTYPES and first.is_cuda
    for t in tensors:
        if t.requires_grad:
            raise ValueError("This API is forward-only")
        ok = ok and t.get_device() == index and t.dtype == dtype and t.stride(-1) == 1
    if not ok:
        raise ValueError("Inputs must be BF16 (or FP16) with a contiguous head dimension on one CUDA device")
    if _major(index) != 10:
        raise ValueError("This implementation is written for SM100/Blackwell")
    return index


def _small(d, gammas, cos, sin):
    """Checks of weights and tables; the number of positions and the ones that are there."""
    if (cos is None) != (sin is None):
        raise ValueError("Provide both rotary tables or neither")
    there = [g for g in gammas if g is not None]
    for g in there:
        if g.shape != (d,):
            raise ValueError("Expected gamma [D]")
    if cos is None:
        return 0, there
    if cos.ndim != 2 or cos.shape[1] != d or cos.shape[0] < 1 or sin.shape != cos.shape or not (
            cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("Expected contiguous rotary tables [positions, D]")
    return cos.shape[0], [*there, cos, sin]


def _p(t):
    return 0 if t is None else t.data_ptr()


def append_rows(cache, k, v, pages, start, gk=None, cos=None, sin=None, *, counts=None, eps=1e-6):
    """Rows ``k`` and ``v`` [B, Hkv, S, D] into the cache, row s of sequence b at position ``start[b] + s``.

    K rows are normed with ``gk`` and rotated with the tables' row of their position on the way (each only if given); V rows
    are stored as they are.  ``counts`` [B] (int32): only the rows s < counts[b] exist, for padded batches.  k and v may be
    head-transposed views of a projection's [B, S, Hkv*D].  Two rows of one call must not go to the same place.
    Writes into the cache's tensors and returns ``cache``."""
    if k.ndim != 4 or k.shape != v.shape or min(k.shape) < 1:
        raise ValueError("Expected K/V [B,Hkv,S,D]")
    b, h, s, d = k.shape
    n_pos, small = _small(d, (gk,), cos, sin)
    if not (eps > 0):
        raise ValueError("eps must be positive")
    index = _check_rows([k, v, *small])
    fields = _cache_fields(cache, pages, b, k.dtype, index)
    if cache[0].shape[1] != h or cache[0].shape[3] != d:
        raise ValueError("Expected K/V with the heads and the head dimension of the cache")
    _check_ints("start", start, b, index)
    if counts is not None:
        _check_ints("counts", counts, b, index)
    with _on_device(index):
        _call(_lib.load().kf_append_rows(_APPEND.pack(
            *fields, k.data_ptr(), v.data_ptr(), _p(gk), _p(cos), _p(sin), start.data_ptr(), _p(counts),
            status_word(k.device).data_ptr(), b, s, _DTYPES[k.dtype], n_pos, *k.stride()[:3], *v.stride()[:3], eps),
            _raw_stream(index)))
    return cache


def read_rows(cache, pages, lengths, s, *, dtype=None, k_out=None, v_out=None):
    """The first ``s`` rows of every sequence as (k, v), each [B, Hkv, s, D]; rows at and behind ``lengths[b]`` are zero.

    ``dtype`` of the result: the cache's own, or torch.bfloat16 (default, exact) or torch.float16 from an e4m3 cache.
    ``k_out`` / ``v_out`` take preallocated (also strided) results."""
    pool = cache[0]
    if pool.ndim != 4 or lengths.ndim != 1 or lengths.shape[0] < 1 or s < 1:
        raise ValueError("Expected a cache, lengths [B] and s >= 1")
    if dtype is None:
        dtype = k_out.dtype if k_out is not None else torch.bfloat16 if pool.dtype == torch.float8_e4m3fn else pool.dtype
    if dtype not in _DTYPES:
        raise ValueError("Rows are read as BF16 or FP16")
    b, shape = lengths.shape[0], (lengths.shape[0], pool.shape[1], int(s), pool.shape[3])
    index = pool.get_device()
    if not pool.is_cuda:
        raise ValueError("The cache and its table must lie on the tensors' CUDA device, with contiguous rows")
    fields = _cache_fields(cache, pages, b, dtype, index)
    _check_ints("lengths", lengths, b, index)
    k = torch.empty(shape, dtype=dtype, device=pool.device) if k_out is None else k_out
    v = torch.empty(shape, dtype=dtype, device=pool.device) if v_out is None else v_out
    if k.shape != shape or v.shape != shape or k.dtype != dtype or v.dtype != dtype:
        raise ValueError("k_out / v_out must be [B,Hkv,s,D] of the result's type")
    _check_rows([k, v])
    if k.get_device() != index:
        raise ValueError("k_out / v_out must lie on the cache's device")
    with _on_device(index):
        _call(_lib.load().kf_read_rows(_READ.pack(
            *fields, k.data_ptr(), v.data_ptr(), lengths.data_ptr(), status_word(pool.device).data_ptr(), b, shape[2],
            _DTYPES[dtype], *k.stride()[:3], *v.stride()[:3]), _raw_stream(index)))
    return k, v


_workspace_bytes = {}  # (device, D, e4m3, more than eight query heads per KV head) -> bytes


def _decode(q, new_k, new_v, cache, pages, lengths, gq, gk, cos, sin, eps, scale, out, workspace):
    pool = cache[0]
    if q.ndim != 4 or q.shape[2] != 1 or min(q.shape) < 1:
        raise ValueError("Expected Q [B,Hq,1,D]: one token per sequence")
    b, hq, _, d = q.shape
    if pool.ndim != 4 or pool.shape[3] != d or pool.shape[1] < 1 or hq % pool.shape[1]:
        raise ValueError("Expected a cache of the queries' head dimension and valid GQA")
    hkv = pool.shape[1]
    n_pos, rows = _small(d, (gq, gk), cos, sin)
    if not (eps > 0):
        raise ValueError("eps must be positive")
    scale = d ** -0.5 if scale is None else scale
    rows.insert(0, q)
    strides = (0, 0, 0, 0)
    if new_k is not None:
        if new_k.shape != (b, hkv, 1, d) or new_v.shape != new_k.shape:
            raise ValueError("Expected K/V [B,Hkv,1,D]: one token per sequence")
        rows += (new_k, new_v)
        strides = new_k.stride()[:2] + new_v.stride()[:2]
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise ValueError("out must match q in shape and dtype")
    rows.append(out)
    index = _check_rows(rows)
    fields = _cache_fields(cache, pages, b, q.dtype, index)
    _check_ints("lengths", lengths, b, index)
    lib = _lib.load()
    with _on_device(index):
        key = (index, d, fields[11], hq > 8 * hkv)
        need = _workspace_bytes.get(key)
        if need is None:
            need = _workspace_bytes[key] = lib.kf_decode_workspace_bytes(b, hq, hkv, d, fields[11])
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        elif (workspace.numel() * workspace.element_size() < need or workspace.get_device() != index or
              not workspace.is_contiguous()):
            raise ValueError(f"workspace must be contiguous, on the queries' device and hold {need} bytes")
        _call(lib.kf_decode_attention(_DECODE.pack(
            *fields, q.data_ptr(), _p(gq), _p(cos), _p(sin), out.data_ptr(), lengths.data_ptr(), _p(new_k), _p(new_v),
            _p(gk), workspace.data_ptr(), status_word(q.device).data_ptr(), b, hq, _DTYPES[q.dtype], n_pos,
            *q.stride()[:2], *out.stride()[:2], *strides, eps, scale), _raw_stream(index)))
    return out


def decode_workspace_bytes(q, cache):
    """Bytes of device memory that a ``decode_attention`` or ``decode_step`` of these tensors works in."""
    with _on_device(q.get_device()):
        return _lib.load().kf_decode_workspace_bytes(q.shape[0], q.shape[1], cache[0].shape[1], q.shape[3],
                                                     _CACHE_DTYPES[cache[0].dtype])


def decode_attention(q, cache, pages, lengths, gq=None, cos=None, sin=None, *, eps=1e-6, scale=None, out=None,
                     workspace=None):
    """Attention of one query token per sequence over its ``lengths[b]`` cached rows, the newest of which is its own.

    ``q`` [B, Hq, 1, D] (also a head-transposed view of a projection's [B, 1, Hq*D]) is normed with ``gq`` and rotated to
    position ``lengths[b] - 1`` in the kernel's prologue (each only if given); query head h reads KV head
    h // (Hq // Hkv).  A sequence with ``lengths[b] <= 0`` (padding) gets zeros.  ``out`` takes a preallocated (also
    strided) result; ``workspace`` (``decode_workspace_bytes``) memory that no other call uses meanwhile, else both come
    from torch's allocator.  Returns [B, Hq, 1, D]."""
    return _decode(q, None, None, cache, pages, lengths, gq, None, cos, sin, eps, scale, out, workspace)


def decode_step(q, k, v, cache, pages, lengths, gq=None, gk=None, cos=None, sin=None, *, eps=1e-6, scale=None, out=None,
                workspace=None):
    """One generated token of every sequence: its ``k`` and ``v`` [B, Hkv, 1, D] are appended at position
    ``lengths[b] - 1`` (as ``append_rows`` does) and its query attends to all ``lengths[b]`` rows (``decode_attention``).
    ``lengths`` counts the new token; a sequence with ``lengths[b] <= 0`` appends nothing and gets zeros."""
    return _decode(q, k, v, cache, pages, lengths, gq, gk, cos, sin, eps, scale, out, workspace)
