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


# (len, heads): whole items of many steps; one item over every CTA, joined in groups; a few parts joined at once
BROKEN = [([900] * 150, 4), ([70001], 4), ([70001], 16), ([9000, 13, 5000], 8)]


def minus_infinite_keys(p, b, first, last):
    """Keys first .. last-1 of sequence b whose scores are -inf for queries with a one in column 0."""
    at = torch.arange(first, last, device="cuda")
    page, row = p.pages[b].long()[at // p.page], at % p.page
    p.k[page, :, row] = 0
    p.k[page, :, row, 0] = -float("inf")


@pytest.mark.parametrize("lengths,hq", BROKEN)
def test_parts_without_any_weight(lengths, hq):
    # keys of whole CTAs' pieces score -inf: the rest alone counts; if all do, nothing is defined
    p = Paged(lengths, 1, 128, 16, BF, seed=81)
    q = rand(82, len(lengths), hq, 1, 128)
    q[..., 0] = 1.0
    n = lengths[0]
    for first, last in ((0, n // 2), (n // 2, n - 1), (1, n // 2)):
        clean = p.k.clone()
        minus_infinite_keys(p, 0, first, last)
        got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
        torch.cuda.synchronize()
        kf.check_status()
        keep = [r for r in range(n) if not first <= r < last]
        cut = Paged.__new__(Paged)
        cut.__dict__.update(p.__dict__)
        cut.rows = lambda name, b, m: p.rows(name, 0, n)[:, keep]
        want, bound = attention_close(cut, q[:1], [len(keep)], None, None, None)
        assert torch.isfinite(got.double()).all()
        assert ((got[:1].double() - want).abs() <= bound).all()
        p.k.copy_(clean)
    minus_infinite_keys(p, 0, 0, n)
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    torch.cuda.synchronize()
    kf.check_status()
    assert torch.isnan(got[0]).all() and torch.isfinite(got[1:].double()).all()


@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("cache", ["16", "e4m3"])
@pytest.mark.parametrize("lengths,hq", BROKEN)
def test_nan_and_infinity_in_one_part(lengths, hq, cache, what):
    p = Paged(lengths, 1, 128, 16, E8 if cache == "e4m3" else BF, seed=83)
    q, n = rand(84, len(lengths), hq, 1, 128), lengths[0]
    clean = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    page, row = int(p.pages[0, (n - 100) // 16]), (n - 100) % 16
    if cache == "e4m3":
        getattr(p, what + "_scale").view(torch.uint8)[page, 0, row] = 255
    else:
        getattr(p, what)[page, 0, row] = float("nan")
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    torch.cuda.synchronize()
    kf.check_status()
    assert torch.isnan(got[0]).all() and torch.equal(got[1:], clean[1:])
    if cache == "16" and what == "v":  # an infinity stays in its column
        getattr(p, what)[page, 0, row] = 1.0
        clean = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
        p.v[page, 0, row, 5], p.v[page, 0, row, 9] = float("inf"), -float("inf")
        got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
        torch.cuda.synchronize()
        assert (got[0, ..., 5] == float("inf")).all() and (got[0, ..., 9] == -float("inf")).all()
        keep = [c for c in range(128) if c not in (5, 9)]
        assert torch.equal(got[..., keep], clean[..., keep]) and torch.equal(got[1:], clean[1:])
