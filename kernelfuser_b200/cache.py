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

Attention sums in fp32.  Prepared queries and probabilities enter its products as two 16-bit numbers each, which leaves 2^-16
(bf16) or 2^-22 (fp16) of a value; in a bf16 call on an e4m3 cache as ONE f16 number, off by 2^-12 of it or less, an eighth of
what rounding the result to bf16 costs.

The layout that decoding reads fastest is the one of ``PagedCache.allocate``, rows of a head D apart.  Any pool with contiguous
rows is taken, [n_pages, page_size, Hkv, D] viewed as [n_pages, Hkv, page_size, D] among them, but copied row by row: long
16-bit sequences take the same time from it, a ragged step of 32 short ones a sixth more, an e4m3 cache a quarter more.

Lengths and tables on the device are not looked at by the host.  A table entry outside the cache, a length or position
that the table cannot hold or one behind the rotary tables is reported through the status word (``check_status`` raises);
nothing is read or written out of bounds.
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from .api import _DTYPES, _call, _current_device, _major, _on_device, _raw_stream, _status, status_word

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


_E8, _SCALE, _INT = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.int32
_16 = frozenset(_DTYPES)

# These calls are a few microseconds of GPU work when the batch is small, so their host path is written for few Python
# operations: each tensor is looked at once, in line.


def _bad_cache(k, v, ks, vs, pages, b, dtype, index):
    """The error of a cache or table that does not fit."""
    if k.requires_grad or v.requires_grad:
        raise ValueError("This API is forward-only")
    if k.ndim != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _CACHE_DTYPES:
        raise ValueError("Expected cache pools [n_pages, Hkv, page_size, D] of one type (BF16, FP16 or float8_e4m3fn)")
    n, h, page, d = k.shape
    if d not in (128, 256) or n < 1 or h < 1 or page < 16 or page % 16:
        raise ValueError("Expected D=128/256 and a page size that is a multiple of 16")
    if k.dtype is not _E8 and k.dtype != dtype:
        raise ValueError("Expected a cache of the tensors' type, or of float8_e4m3fn")
    if pages.ndim != 2 or pages.shape[0] != b or pages.shape[1] < 1 or pages.dtype != _INT or (
            pages.shape[1] > 1 and pages.stride(1) != 1):
        raise ValueError("Expected an int32 page table [B, max_pages] with contiguous rows")
    if k.dtype is not _E8 and not (ks is None and vs is None):
        raise ValueError("Scales belong to an e4m3 cache only")
    if k.dtype is _E8 and (ks is None or vs is None or ks.shape != k.shape[:3] or vs.shape != k.shape[:3] or
                           ks.dtype != _SCALE or vs.dtype != _SCALE):
        raise ValueError("Expected float8_e8m0fnu scales [n_pages, Hkv, page_size] with an e4m3 cache")
    raise ValueError("The cache and its table must lie on the tensors' CUDA device, with contiguous rows")


def _cache_fields(cache, pages, b, dtype, index):
    """The kf_paged_cache of a call, after the checks that need no device."""
    if len(cache) == 2:
        (k, v), ks, vs = cache, None, None
    else:
        k, v, ks, vs = cache
    shape, kind, sk, sv, sp, table = k.shape, k.dtype, k.stride(), v.stride(), pages.stride(), pages.shape
    e8 = kind is _E8
    ok = (len(shape) == 4 and v.shape == shape and v.dtype is kind and (e8 or kind is dtype) and len(table) == 2 and
          table[0] == b and table[1] >= 1 and pages.dtype is _INT and (sp[1] == 1 or table[1] == 1) and
          k.get_device() == v.get_device() == pages.get_device() == index >= 0 and sk[3] == 1 == sv[3] and
          not (k.requires_grad or v.requires_grad))
    if ok:
        n, h, page, d = shape
        ok = (d == 128 or d == 256) and n >= 1 and h >= 1 and page >= 16 and page % 16 == 0
    if ok and e8:
        ok = (ks is not None and vs is not None and ks.dtype is _SCALE and vs.dtype is _SCALE and
              ks.shape == vs.shape == shape[:3] and ks.get_device() == vs.get_device() == index)
        if ok:
            a, c = ks.stride(), vs.stride()
            if a[2] == 1 == c[2]:
                return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages.data_ptr(), sp[0], n, table[1], page,
                        h, d, _lib.KF_E4M3, sk[0], sk[1], sk[2], sv[0], sv[1], sv[2], a[0], a[1], c[0], c[1])
    elif ok and ks is None and vs is None:
        return (k.data_ptr(), v.data_ptr(), 0, 0, pages.data_ptr(), sp[0], n, table[1], page, h, d, _DTYPES[kind], sk[0], sk[1],
                sk[2], sv[0], sv[1], sv[2], 0, 0, 0, 0)
    _bad_cache(k, v, ks, vs, pages, b, dtype, index)


def _check_ints(name, t, b, index):
    if t.dtype is not _INT or t.shape != (b,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"Expected {name} as contiguous int32 [B] on the tensors' CUDA device")


def _check_rows(tensors, first, small):
    """Every tensor in rows of a contiguous head dimension, on one CUDA device that is a B200, in one 16-bit type; the rows
    that are read, weights and tables need no gradient."""
    dtype, index = first.dtype, first.get_device()
    ok = dtype in _16 and index >= 0
    for t in tensors:
        if t.requires_grad:
            raise ValueError("This API is forward-only")
        ok = ok and t.get_device() == index and t.dtype is dtype and t.stride(-1) == 1
    for t in small:
        if t is not None:
            if t.requires_grad:
                raise ValueError("This API is forward-only")
            ok = ok and t.get_device() == index and t.dtype is dtype and t.is_contiguous()
    if not ok:
        raise ValueError("Inputs must be BF16 (or FP16) with a contiguous head dimension on one CUDA device")
    if _major(index) != 10:
        raise ValueError("This implementation is written for SM100/Blackwell")
    return index


def _check_small(d, gq, gk, cos, sin):
    """Shapes of weights and tables; the number of positions."""
    if (gq is not None and gq.shape != (d,)) or (gk is not None and gk.shape != (d,)):
        raise ValueError("Expected gamma [D]")
    if cos is None:
        if sin is not None:
            raise ValueError("Provide both rotary tables or neither")
        return 0
    if sin is None:
        raise ValueError("Provide both rotary tables or neither")
    shape = cos.shape
    if len(shape) != 2 or shape[1] != d or shape[0] < 1 or sin.shape != shape:
        raise ValueError("Expected contiguous rotary tables [positions, D]")
    return shape[0]


def _status_ptr(index):
    w = _status.get(index)
    return (status_word(torch.device("cuda", index)) if w is None else w).data_ptr()


def append_rows(cache, k, v, pages, start, gk=None, cos=None, sin=None, *, counts=None, eps=1e-6):
    """Rows ``k`` and ``v`` [B, Hkv, S, D] into the cache, row s of sequence b at position ``start[b] + s``.

    K rows are normed with ``gk`` and rotated with the tables' row of their position on the way (each only if given); V rows
    are stored as they are.  ``counts`` [B] (int32): only the rows s < counts[b] exist, for padded batches.  k and v may be
    head-transposed views of a projection's [B, S, Hkv*D].  Two rows of one call must not go to the same place.
    Writes into the cache's tensors and returns ``cache``."""
    if k.ndim != 4 or k.shape != v.shape or min(k.shape) < 1:
        raise ValueError("Expected K/V [B,Hkv,S,D]")
    b, h, s, d = k.shape
    n_pos = _check_small(d, gk, None, cos, sin)
    if not (eps > 0):
        raise ValueError("eps must be positive")
    index = _check_rows((k, v), k, (gk, cos, sin))
    fields = _cache_fields(cache, pages, b, k.dtype, index)
    if fields[9] != h or fields[10] != d:
        raise ValueError("Expected K/V with the heads and the head dimension of the cache")
    _check_ints("start", start, b, index)
    if counts is not None:
        _check_ints("counts", counts, b, index)
    packed = (k.data_ptr(), v.data_ptr(), 0 if gk is None else gk.data_ptr(), 0 if cos is None else cos.data_ptr(),
              0 if sin is None else sin.data_ptr(), start.data_ptr(), 0 if counts is None else counts.data_ptr(),
              _status_ptr(index), b, s, _DTYPES[k.dtype], n_pos)
    with _on_device(index):
        params = _APPEND.pack(*fields, *packed, *k.stride()[:3], *v.stride()[:3], eps)
        _call(_lib.load().kf_append_rows(params, _raw_stream(index)))
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
    if _check_rows((k, v), k, ()) != index:
        raise ValueError("k_out / v_out must lie on the cache's device")
    with _on_device(index):
        _call(_lib.load().kf_read_rows(_READ.pack(
            *fields, k.data_ptr(), v.data_ptr(), lengths.data_ptr(), _status_ptr(index), b, shape[2],
            _DTYPES[dtype], *k.stride()[:3], *v.stride()[:3]), _raw_stream(index)))
    return k, v


_workspace_bytes = {}  # (device, D, e4m3, more than eight query heads per KV head) -> bytes


def _decode(q, new_k, new_v, cache, pages, lengths, gq, gk, cos, sin, eps, scale, out, workspace):
    shape = q.shape
    if len(shape) != 4 or shape[2] != 1 or shape[0] < 1 or shape[1] < 1:
        raise ValueError("Expected Q [B,Hq,1,D]: one token per sequence")
    b, hq, _, d = shape
    pool = cache[0].shape
    if len(pool) != 4 or pool[3] != d or pool[1] < 1 or hq % pool[1]:
        raise ValueError("Expected a cache of the queries' head dimension and valid GQA")
    hkv = pool[1]
    n_pos = _check_small(d, gq, gk, cos, sin)
    if not (eps > 0):
        raise ValueError("eps must be positive")
    fresh = out is None
    if fresh:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape:
        raise ValueError("out must match q in shape and dtype")
    if new_k is None:
        index = _check_rows((q,) if fresh else (q, out), q, (gq, cos, sin))
        new = (0, 0, 0)
        new_strides = (0, 0, 0, 0)
    else:
        if new_k.shape != (b, hkv, 1, d) or new_v.shape != new_k.shape:
            raise ValueError("Expected K/V [B,Hkv,1,D]: one token per sequence")
        index = _check_rows((q, new_k, new_v) if fresh else (q, new_k, new_v, out), q, (gq, gk, cos, sin))
        new = (new_k.data_ptr(), new_v.data_ptr(), 0 if gk is None else gk.data_ptr())
        nk, nv = new_k.stride(), new_v.stride()
        new_strides = (nk[0], nk[1], nv[0], nv[1])
    fields = _cache_fields(cache, pages, b, q.dtype, index)
    _check_ints("lengths", lengths, b, index)
    lib = _lib.load()
    if _current_device() != index:
        with torch.cuda.device(index):
            return _decode(q, new_k, new_v, cache, pages, lengths, gq, gk, cos, sin, eps, scale, out, workspace)
    key = (index, d, fields[11], hq > 8 * hkv)
    need = _workspace_bytes.get(key)
    if need is None:
        need = _workspace_bytes[key] = lib.kf_decode_workspace_bytes(b, hq, hkv, d, fields[11])
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    elif (workspace.numel() * workspace.element_size() < need or workspace.get_device() != index or
          not workspace.is_contiguous()):
        raise ValueError(f"workspace must be contiguous, on the queries' device and hold {need} bytes")
    sq, so = q.stride(), out.stride()
    rc = lib.kf_decode_attention(_DECODE.pack(
        *fields, q.data_ptr(), 0 if gq is None else gq.data_ptr(), 0 if cos is None else cos.data_ptr(),
        0 if sin is None else sin.data_ptr(), out.data_ptr(), lengths.data_ptr(), *new, workspace.data_ptr(),
        _status_ptr(index), b, hq, _DTYPES[q.dtype], n_pos, sq[0], sq[1], so[0], so[1], *new_strides, eps,
        d ** -0.5 if scale is None else scale), _raw_stream(index))
    if rc:
        _call(rc)
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
    if k is None or v is None:  # (without rows it would be decode_attention, over a row that nothing has written)
        raise ValueError("Expected K/V [B,Hkv,1,D]: one token per sequence")
    return _decode(q, k, v, cache, pages, lengths, gq, gk, cos, sin, eps, scale, out, workspace)
