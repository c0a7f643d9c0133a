"""Attention over caches whose values are as large, or as small, as the cache's type holds."""
import pytest
import torch

import kernelfuser_b200 as kf
from serving import Paged, tables
from serving_close import attention_close

pytestmark = pytest.mark.gpu

BF, E8 = torch.bfloat16, torch.float8_e4m3fn


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rand(seed, *shape, dtype=BF):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(*shape, generator=g).to("cuda", dtype)


def check(got, want, bound):
    got = got.double()
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    assert (off <= bound).all(), float((off / bound).max())


# whole items of one and of many steps, broken ones joined once and in groups
LENGTHS = [[40, 1, 0, 700], [70001], [9000, 13, 5000]]


@pytest.mark.parametrize("low,high", [(244, 246), (200, 246), (1, 3), (1, 246)])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 1, 128), (2, 1, 256), (11, 1, 256)])
def test_value_scales_at_the_ends_of_their_range(low, high, lengths, hq, hkv, d):
    p = Paged(lengths, hkv, d, 16, E8, seed=70)
    g = torch.Generator().manual_seed(71)
    p.v_scale = torch.randint(low, high + 1, p.v_scale.shape, generator=g, dtype=torch.uint8).cuda().view(torch.float8_e8m0fnu)
    q = rand(72, len(lengths), hq, 1, d)
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    torch.cuda.synchronize()
    kf.check_status()
    check(got, *attention_close(p, q, lengths, None, None, None))


@pytest.mark.parametrize("lengths", LENGTHS)
def test_the_largest_row_of_an_e4m3_cache(lengths):
    # every value row is the largest one that append_rows makes, 448 * 2^119: so is the result, whatever the weights
    p = Paged(lengths, 1, 128, 16, E8, seed=73)
    p.v.copy_(torch.full(p.v.shape, 448.0).to(E8))
    p.v_scale.view(torch.uint8).fill_(246)
    q = rand(74, len(lengths), 4, 1, 128)
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    torch.cuda.synchronize()
    kf.check_status()
    for b, n in enumerate(lengths):
        assert (got[b].double() == (448 * 2.0 ** 119 if n > 0 else 0)).all()


def test_a_large_value_row_that_a_step_appends():
    # a bf16 value of 2^126 goes through append, read and attention, with the step's own row the largest
    lengths = [33, 700]
    p = Paged(lengths, 2, 128, 16, E8, seed=75)
    q, k, v = rand(76, 2, 8, 1, 128), rand(77, 2, 2, 1, 128), rand(78, 2, 2, 1, 128) * 2.0 ** 124
    cos, sin = tables(700, 128, BF, "cuda")
    got = kf.decode_step(q, k, v, p.cache, p.pages, ints(lengths), None, None, cos, sin)
    torch.cuda.synchronize()
    kf.check_status()
    check(got, *attention_close(p, q, lengths, None, cos, sin))


@pytest.mark.parametrize("power", [127, 122, -90])
@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 1, 128), (2, 1, 256), (11, 1, 256)])
def test_values_at_the_ends_of_bf16(power, lengths, hq, hkv, d):
    # below 2^power, and half of them near it: the result is a mean of them, whatever their sum
    p = Paged(lengths, hkv, d, 16, BF, seed=79)
    p.v.clamp_(-0.99, 0.99).mul_(2.0 ** power)
    q = rand(80, len(lengths), hq, 1, d)
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    torch.cuda.synchronize()
    kf.check_status()
    check(got, *attention_close(p, q, lengths, None, None, None))
