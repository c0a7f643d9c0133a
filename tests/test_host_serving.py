"""CPU tests of the serving operators' boundary: every misuse is a ValueError (an error code from the C entry points) before
anything is launched."""
import ctypes

import pytest
import torch

import kernelfuser_b200 as kf
from kernelfuser_b200 import _lib, cache as kc

BF = torch.bfloat16


def parts(b=2, hq=4, hkv=2, d=128, n=5, page=16, dtype=BF, cache=BF):
    pool = kf.PagedCache.allocate(n, page, hkv, d, cache, device="cpu")
    return dict(q=torch.zeros(b, hq, 1, d, dtype=dtype), k=torch.zeros(b, hkv, 1, d, dtype=dtype), cache=pool,
                pages=torch.zeros(b, 2, dtype=torch.int32), lengths=torch.ones(b, dtype=torch.int32),
                g=torch.ones(d, dtype=dtype), cos=torch.zeros(9, d, dtype=dtype))


def attend(x, **kw):
    kw = {**x, **kw}
    return kf.decode_attention(kw["q"], kw["cache"], kw["pages"], kw["lengths"], kw["g"], kw["cos"], kw.get("sin", kw["cos"]))


def append(x, **kw):
    kw = {**x, **kw}
    return kf.append_rows(kw["cache"], kw["k"], kw.get("v", kw["k"]), kw["pages"], kw["lengths"], kw["g"], kw["cos"],
                          kw.get("sin", kw["cos"]), eps=kw.get("eps", 1e-6))


def test_misuse_raises_value_error():
    x = parts()
    for call in (attend, append):
        with pytest.raises(ValueError, match="both rotary"):
            call(x, sin=None)
        with pytest.raises(ValueError, match="gamma"):
            call(x, g=x["g"][:64])
        with pytest.raises(ValueError, match="rotary tables"):
            call(x, cos=x["cos"][:, :64], sin=x["cos"][:, :64])
        with pytest.raises(ValueError, match="CUDA"):  # there is no CPU path
            call(x)
    with pytest.raises(ValueError, match="forward-only"):
        append(x, k=x["k"].float().requires_grad_().to(BF))
    with pytest.raises(ValueError, match="one token"):
        attend(x, q=torch.zeros(2, 4, 3, 128, dtype=BF))
    with pytest.raises(ValueError, match="GQA"):
        attend(x, q=torch.zeros(2, 5, 1, 128, dtype=BF))
    with pytest.raises(ValueError, match="GQA"):
        attend(x, q=torch.zeros(2, 4, 1, 256, dtype=BF), g=torch.ones(256, dtype=BF))
    with pytest.raises(ValueError, match="Expected K/V"):
        append(x, v=x["k"][:, :1])
    with pytest.raises(ValueError, match="Expected K/V"):
        kf.decode_step(x["q"], x["k"][:1], x["k"][:1], x["cache"], x["pages"], x["lengths"])
    with pytest.raises(ValueError, match="eps"):
        append(x, eps=0.0)
    with pytest.raises(ValueError, match="s >= 1"):
        kf.read_rows(x["cache"], x["pages"], x["lengths"], 0)
    with pytest.raises(ValueError, match="BF16 or FP16"):
        kf.read_rows(x["cache"], x["pages"], x["lengths"], 4, dtype=torch.float32)
    with pytest.raises(ValueError, match="CUDA"):
        kf.read_rows(x["cache"], x["pages"], x["lengths"], 4)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        kf.PagedCache.allocate(2, 16, 1, 128, torch.float32, device="cpu")


def fields(x, dtype=BF):
    return kc._cache_fields(x["cache"], x["pages"], 2, dtype, -1)


@pytest.mark.parametrize("change,match", [
    (dict(cache=(torch.zeros(5, 2, 16, 128, dtype=BF), torch.zeros(5, 2, 32, 128, dtype=BF))), "pools"),
    (dict(cache=(torch.zeros(5, 2, 16, 128), torch.zeros(5, 2, 16, 128))), "pools"),
    (dict(cache=(torch.zeros(5, 2, 16, 64, dtype=BF),) * 2), "128/256"),
    (dict(cache=(torch.zeros(5, 2, 24, 128, dtype=BF),) * 2), "page size"),
    (dict(cache=(torch.zeros(5, 2, 16, 128, dtype=torch.float16),) * 2), "tensors' type"),
    (dict(cache=(torch.zeros(5, 2, 16, 128, dtype=torch.float8_e4m3fn),) * 2), "scales"),
    (dict(cache=(torch.zeros(5, 2, 16, 128, dtype=torch.float8_e4m3fn),) * 2 + (torch.zeros(5, 2, 16),) * 2), "scales"),
    (dict(cache=(torch.zeros(5, 2, 16, 128, dtype=BF),) * 2 + (torch.zeros(5, 2, 16),) * 2), "e4m3 cache only"),
    (dict(pages=torch.zeros(3, 2, dtype=torch.int32)), "page table"),
    (dict(pages=torch.zeros(2, 2, dtype=torch.int64)), "page table"),
    (dict(pages=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]), "page table"),
])
def test_cache_and_table_are_checked(change, match):
    with pytest.raises(ValueError, match=match):
        fields({**parts(), **change})


def test_lengths_are_checked():
    for bad in (torch.ones(2), torch.ones(3, dtype=torch.int32), torch.ones(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="lengths"):
            kc._check_ints("lengths", bad, 2, -1)


def c_cache(p, **kw):
    v = dict(pages_stride=2, n=5, max_pages=2, page=16, h=2, d=128, dtype=0, kp=4096, kh=2048, ks=128, vp=4096, vh=2048, vs=128,
             sc=(0, 0, 0, 0), pools=(p, p, 0, 0, p))
    v.update(kw)
    return (*v["pools"], v["pages_stride"], v["n"], v["max_pages"], v["page"], v["h"], v["d"], v["dtype"], v["kp"], v["kh"],
            v["ks"], v["vp"], v["vh"], v["vs"], *v["sc"])


def test_c_abi_rejects_bad_arguments_before_launch():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 15) & ~15

    def decode(cache=(), b=2, hq=4, dtype=0, q=p, out=p, strides=(512, 128) * 2, new=(0, 0), ws=p, status=p, eps=1e-6, scale=0.1,
               cos=0, sin=0, n_pos=0, lengths=p):
        return lib.kf_decode_attention(kc._DECODE.pack(*(cache or c_cache(p)), q, 0, cos, sin, out, lengths, *new, 0, ws, status, b, hq,
                                                       dtype, n_pos, *strides, 256, 128, 256, 128, eps, scale), None)

    for kw, code, text in [
            (dict(dtype=7), -1, b"dtype"), (dict(hq=5), -1, b"multiple"), (dict(b=0), -1, b"B must"), (dict(q=0), -1, b"q must"),
            (dict(q=p + 2), -2, b"aligned"), (dict(strides=(516, 128, 512, 128)), -2, b"multiples of 8"),
            (dict(strides=(512, 128, 512, 0)), -2, b"multiples of 8"), (dict(new=(p, 0)), -1, b"both new"),
            (dict(ws=0), -1, b"workspace"), (dict(ws=p + 4), -2, b"aligned"), (dict(status=0), -1, b"status"),
            (dict(eps=0.0), -1, b"eps"), (dict(eps=float("nan")), -1, b"eps"), (dict(scale=-1.0), -1, b"scale"),
            (dict(scale=float("inf")), -1, b"scale"), (dict(cos=p), -1, b"both rotary"), (dict(cos=p, sin=p), -1, b"n_positions"),
            (dict(cache=c_cache(p, d=64)), -1, b"head dim"), (dict(cache=c_cache(p, page=24)), -1, b"multiple of 16"),
            (dict(cache=c_cache(p, page=0)), -1, b"multiple of 16"), (dict(cache=c_cache(p, n=0)), -1, b"n_pages"),
            (dict(cache=c_cache(p, n=1 << 40)), -1, b"n_pages"), (dict(cache=c_cache(p, max_pages=0)), -1, b"max_pages"),
            (dict(cache=c_cache(p, h=0)), -1, b"Hkv"), (dict(cache=c_cache(p, dtype=1)), -1, b"dtype"),
            (dict(cache=c_cache(p, kp=4100)), -2, b"16 bytes"), (dict(cache=c_cache(p, vs=0)), -2, b"16 bytes"),
            (dict(cache=c_cache(p, ks=64)), -1, b"row stride"), (dict(cache=c_cache(p, pages_stride=-1)), -1, b"pages_stride"),
            (dict(cache=c_cache(p, dtype=2)), -1, b"k_scale"),
            (dict(cache=c_cache(p, dtype=2, pools=(p, p, p, p, p), sc=(32, 8, 32, 16))), -2, b"scale strides"),
            (dict(cache=c_cache(p, pools=(0, p, 0, 0, p))), -1, b"NULL"), (dict(cache=c_cache(p, pools=(p, p + 8, 0, 0, p))), -2, b"aligned")]:
        assert decode(**kw) == code and text in lib.kf_last_error(), (kw, lib.kf_last_error())
    for fn in (lib.kf_append_rows, lib.kf_read_rows, lib.kf_decode_attention):
        assert fn(None, None) == -1

    def append(b=2, s=3, start=p, status=p, strides=(768, 128, 256)):
        return lib.kf_append_rows(kc._APPEND.pack(*c_cache(p), p, p, 0, 0, 0, start, 0, status, b, s, 0, 0, *strides, *strides, 1e-6), None)

    def read(b=2, s=3, lengths=p, strides=(768, 128, 256)):
        return lib.kf_read_rows(kc._READ.pack(*c_cache(p), p, p, lengths, p, b, s, 0, *strides, *strides), None)

    for fn in (append, read):
        assert fn(s=0) == -1 and fn(b=1 << 40) == -1 and fn(strides=(768, 128, 64)) == -1 and fn(strides=(768, 0, 256)) == -2
    assert append(start=0) == -1 and append(status=0) == -1 and read(lengths=0) == -1 and append(b=1 << 16, s=1 << 16) == -1


def test_workspace_size():
    lib = _lib.load()
    assert lib.kf_decode_workspace_bytes(0, 4, 2, 128, 0) == 0 and lib.kf_decode_workspace_bytes(1, 4, 2, 64, 0) == 0
    one, two = lib.kf_decode_workspace_bytes(1, 8, 1, 128, 0), lib.kf_decode_workspace_bytes(1, 16, 1, 128, 0)
    assert 0 < one < two
