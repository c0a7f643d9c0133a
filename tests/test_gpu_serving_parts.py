"""Attention over long sequences, whose parts meet from many warps and CTAs: against a bound that a result without some of its
keys is outside of, with value rows that say where in the sequence they stand."""
import pytest
import torch

import kernelfuser_b200 as kf
from serving import Paged, tables
from serving_close import LONG, attention_close, region_values

pytestmark = pytest.mark.gpu

BF, FP, E8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.mark.parametrize("values", ["random", "regions"])
@pytest.mark.parametrize("cache,dtype", [("16", BF), ("16", FP), ("e4m3", BF), ("e4m3", FP)])
@pytest.mark.parametrize("lengths,hq,hkv,d", LONG)
def test_every_part_counts_once(values, cache, dtype, lengths, hq, hkv, d):
    p = Paged(lengths, hkv, d, 64, E8 if cache == "e4m3" else dtype, seed=140)
    if values == "regions":
        region_values(p, lengths)
    g = torch.Generator().manual_seed(141)
    q = torch.randn(len(lengths), hq, 1, d, generator=g).to("cuda", dtype)
    gq = (1.4 + 0.2 * torch.randn(d, generator=g)).to("cuda", dtype)
    cos, sin = tables(max(lengths), d, dtype, "cuda")
    got = kf.decode_attention(q, p.cache, p.pages, torch.tensor(lengths, dtype=torch.int32, device="cuda"), gq, cos, sin)
    torch.cuda.synchronize()
    kf.check_status()
    some = [i for i in range(len(lengths)) if i < 8 or i % 37 == 0 or i == len(lengths) - 1]
    want, bound = attention_close(p, q, lengths, gq, cos, sin, only=some)
    off = (got[some].double() - want[some]).abs()
    assert torch.isfinite(got.double()).all()
    assert (off <= bound[some]).all(), float((off / bound[some]).max())
