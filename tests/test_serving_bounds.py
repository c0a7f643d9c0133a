"""CPU test of the tests' own bound: results with a mistake planted in the 64-bit oracle are outside of it."""
import pytest
import torch

from serving import Paged, tables, transform
from serving_close import LONG, attention_close, region_values

BF, FP, E8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.mark.parametrize("cache,dtype", [("16", BF), ("16", FP), ("e4m3", BF), ("e4m3", FP)])
@pytest.mark.parametrize("lengths,d", sorted({(max(x[0]), x[3]) for x in LONG}))
def test_lost_and_repeated_keys_are_seen(cache, dtype, lengths, d):
    # the longest sequence of each launch, two query heads of one KV head
    n = lengths
    p = Paged([n], 1, d, 64, E8 if cache == "e4m3" else dtype, seed=140, device="cpu")
    region_values(p, [n])
    g = torch.Generator().manual_seed(141)
    q = torch.randn(1, 2, 1, d, generator=g).to(dtype)
    gq = (1.4 + 0.2 * torch.randn(d, generator=g)).to(dtype)
    cos, sin = tables(n, d, dtype, "cpu")
    want, bound = (x[0, :, 0] for x in attention_close(p, q, [n], gq, cos, sin))
    k, v = p.rows("k", 0, n)[0], p.rows("v", 0, n)[0]
    weight = torch.softmax(transform(q[0, :, 0], gq, cos[n - 1], sin[n - 1])[0] @ k.t() * d ** -0.5, -1)

    def outside(times):  # the attention over rows that count 0, 1 or 2 times
        x = weight * times
        return ((x @ v / x.sum(-1, keepdim=True) - want).abs() > bound).any()

    assert not outside(torch.ones(n)) and (want > bound).any()
    step = 32 if cache == "e4m3" else 16  # what a warp takes at a time
    if cache == "e4m3" and dtype == BF:  # one f16 number in the products: what a CTA takes of one long sequence
        step = max(step, n // 148)
    for lo, hi in ((0, step), (n // 2 // 64 * 64, n // 2 // 64 * 64 + step), (n - step, n), (n - n // 8, n), (0, n // 2)):
        for wrong in (0.0, 2.0):
            times = torch.ones(n)
            times[lo:hi] = wrong
            assert outside(times), (lo, hi, wrong)
