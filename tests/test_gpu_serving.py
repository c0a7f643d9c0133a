"""The serving operators against their definition in 64 bits: rows into a paged cache and back, the attention of one token
over it, and both together, at the sizes, layouts and masks where they can go wrong."""
import math

import pytest
import torch

import kernelfuser_b200 as kf
from serving import EPS, Paged, U, attention, quantise, tables, transform, two

pytestmark = pytest.mark.gpu

BF, FP, E8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rand(seed, *shape, dtype=BF):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(*shape, generator=g).to("cuda", dtype)


def weights(seed, d, dtype):
    return (1.4 + 0.2 * rand(seed, d, dtype=torch.float32)).to(dtype)


def done():
    torch.cuda.synchronize()
    kf.check_status()


def check(got, want, bound):
    off = (got.double() - want).abs() - bound
    assert torch.isfinite(got.double()).all()
    assert (off <= 0).all(), (float(off.max()), float((got.double() - want).abs().max()))


def fill_nan_behind(p, lengths):
    """NaN in every row of the pools that no sequence holds: nothing may depend on them."""
    hold = torch.zeros(p.k.shape[0], p.page, dtype=torch.bool)
    table = p.pages.cpu()
    for b, n in enumerate(lengths):
        for r in range(max(n, 0)):
            hold[table[b, r // p.page], r % p.page] = True
    hold = hold.cuda()[:, None, :]
    for pool, scale in ((p.k, p.k_scale), (p.v, p.v_scale)):
        if scale is None:
            pool.masked_fill_(~hold[..., None], math.nan)
        else:
            pool.view(torch.uint8).masked_fill_(~hold[..., None], 0x7f)
            scale.view(torch.uint8).masked_fill_((~hold).expand(scale.shape), 255)


# ---- attention ---------------------------------------------------------------------------------------------------------
EDGE = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 0, 127, 128, 129, 255, 257, -3, 300]


@pytest.mark.parametrize("cache", ["16", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,hq,hkv,page,norm,rope", [
    (128, 8, 2, 16, True, True),     # four query heads to a KV head
    (128, 3, 3, 48, False, True),    # heads without sharing, pages that are no power of two
    (128, 12, 1, 32, True, False),   # two n8 blocks, the second half full
    (128, 40, 2, 64, True, True),    # two blocks of 16 rows, the second one short
    (128, 35, 1, 16, False, True),   # three blocks
    (256, 4, 2, 16, True, True),
    (256, 11, 1, 80, False, False),
    (256, 17, 1, 16, True, True),    # a block of 16 rows and a single one
])
def test_attention_at_edge_lengths(cache, dtype, d, hq, hkv, page, norm, rope):
    p = Paged(EDGE, hkv, d, page, E8 if cache == "e4m3" else dtype, seed=1, max_pages=20)
    fill_nan_behind(p, EDGE)
    q = rand(2, len(EDGE), hq, 1, d, dtype=dtype)
    gq = weights(3, d, dtype) if norm else None
    cos, sin = tables(300, d, dtype, "cuda") if rope else (None, None)
    out = torch.full_like(q, math.nan)
    got = kf.decode_attention(q, p.cache, p.pages, ints(EDGE), gq, cos, sin, out=out)
    done()
    assert got is out
    check(got, *attention(p, q, EDGE, gq, cos, sin))
    for b, n in enumerate(EDGE):
        if n <= 0:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("cache", ["16", "e4m3"])
@pytest.mark.parametrize("lengths,hq,hkv,d", [
    ([70001], 8, 1, 128),                 # one item over every CTA
    ([9000, 1, 0, 5000, 13], 4, 2, 128),  # broken items next to whole ones
    ([20000, 64], 2, 1, 256),
    ([4097] * 3, 16, 1, 256),
    ([6000, 700], 24, 1, 128),
    ([900] * 150, 24, 1, 128),            # whole items of many units: every slot of a ring is used, again and again
    ([1500] * 150, 16, 1, 256),
    ([1300] * 300, 2, 1, 256),
    ([2100] * 450, 3, 1, 128),
    ([900] * 40, 8, 4, 128),
])
def test_long_sequences_are_split_and_joined(cache, lengths, hq, hkv, d):
    p = Paged(lengths, hkv, d, 64, E8 if cache == "e4m3" else BF, seed=4)
    q, gq = rand(5, len(lengths), hq, 1, d), weights(6, d, BF)
    cos, sin = tables(max(lengths), d, BF, "cuda")
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths), gq, cos, sin)
    done()
    check(got, *attention(p, q, lengths, gq, cos, sin))
    for _ in range(3):  # the same bits every time
        assert torch.equal(kf.decode_attention(q, p.cache, p.pages, ints(lengths), gq, cos, sin), got)


@pytest.mark.parametrize("cache", ["16", "e4m3"])
@pytest.mark.parametrize("lengths,hq,hkv,d", [
    ([70, 0, 400], 4800, 1, 128),         # more blocks of 16 query heads than CTAs
    ([9000, 77], 40, 1, 128),             # the last block half full, broken items
    ([3000, 1, 0, 801], 100, 2, 256),
])
def test_many_query_heads_share_a_step(cache, lengths, hq, hkv, d):
    p = Paged(lengths, hkv, d, 16, E8 if cache == "e4m3" else BF, seed=91)
    q, k, v = rand(92, len(lengths), hq, 1, d), rand(93, len(lengths), hkv, 1, d), rand(94, len(lengths), hkv, 1, d)
    got = kf.decode_step(q, k, v, p.cache, p.pages, ints(lengths))  # (writes the last row, once)
    again = kf.decode_step(q, k, v, p.cache, p.pages, ints(lengths))
    done()
    check(got, *attention(p, q, lengths, None, None, None))
    assert torch.equal(got, again)


def test_more_captured_launches_than_join_words():
    # a captured launch has words of its own to count in, 4096 at a time; a further one gets them from its workspace
    lengths, most = [3000, 70], 4300
    p = Paged(lengths, 1, 128, 64, BF, seed=50)
    q, n = rand(51, 2, 4, 1, 128), ints(lengths)
    want = kf.decode_attention(q, p.cache, p.pages, n)
    out = torch.empty_like(want)
    ws = torch.empty(kf.decode_workspace_bytes(q, p.cache), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(most):
                kf.decode_attention(q, p.cache, p.pages, n, out=out, workspace=ws)
        out.zero_()
        for _ in range(2):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        g.reset()
        del g
    done()


def test_joins_after_a_status():
    # CTAs that find the status word set still count, so that the words are clear for the next launch
    lengths = [40000, 9000]
    p = Paged(lengths, 1, 128, 64, BF, seed=52)
    q, n = rand(53, 2, 4, 1, 128), ints(lengths)
    want = kf.decode_attention(q, p.cache, p.pages, n)
    done()
    for _ in range(1100):  # every row of words in turn
        bad = p.pages.clone() if _ == 0 else bad
        if _ == 0:
            bad[0, 3] = -1
        kf.decode_attention(q, p.cache, bad, n)
    with pytest.raises(kf.KernelStatusError, match="911"):
        kf.check_status()
    for _ in range(1100):
        got = kf.decode_attention(q, p.cache, p.pages, n)
    done()
    assert torch.equal(got, want)


def test_many_sequences():
    # more sequences than threads of a CTA, runs of empty ones among them
    lengths = [(37 * b) % 150 if b % 7 and not 200 < b < 420 else 0 for b in range(700)]
    p = Paged(lengths, 2, 128, 16, BF, seed=7)
    q = rand(8, 700, 4, 1, 128)
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    done()
    check(got, *attention(p, q, lengths, None, None, None))


@pytest.mark.parametrize("cache", ["16", "e4m3"])
def test_strided_tensors_and_shared_pages(cache):
    # projections' layouts, a pool of [n_pages, page, Hkv, D], a table that every sequence shares, an output inside a larger one
    lengths = [200, 150, 33]
    p = Paged([200], 2, 128, 16, E8 if cache == "e4m3" else BF, seed=9, strided=True)
    p.pages = p.pages.expand(3, -1)
    q = rand(10, 3, 1, 8 * 128).view(3, 1, 8, 128).transpose(1, 2)
    big = torch.full((3, 16, 1, 128), 7.0, dtype=BF, device="cuda")
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths), out=big[:, 4:12])
    done()
    check(got, *attention(p, q, lengths, None, None, None))
    assert (big[:, :4] == 7).all() and (big[:, 12:] == 7).all()


def test_scale_and_peaked_scores():
    # scores of hundreds: all but a few probabilities vanish, and the running maximum moves many times
    lengths = [3000, 777]
    p = Paged(lengths, 2, 128, 32, FP, seed=11)
    q = rand(12, 2, 4, 1, 128, dtype=FP)
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths), scale=1.0)
    done()
    check(got, *attention(p, q, lengths, None, None, None, scale=1.0))


def test_value_rows_of_very_different_sizes():
    # an 8-bit cache whose value scales differ by up to 2^60: each row's scale acts in the exponent of its probability
    lengths = [500, 40]
    p = Paged(lengths, 2, 128, 16, E8, seed=13)
    g = torch.Generator().manual_seed(14)
    p.v_scale = torch.randint(90, 150, p.v_scale.shape, generator=g, dtype=torch.uint8).cuda().view(torch.float8_e8m0fnu)
    q = rand(15, 2, 4, 1, 128)
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    done()
    want, bound = attention(p, q, lengths, None, None, None)
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("cache", ["16", "e4m3"])
@pytest.mark.parametrize("what", ["k", "v", "q"])
def test_nan_spoils_what_sees_it_and_nothing_else(cache, what):
    lengths = [100, 5, 400]
    p = Paged(lengths, 2, 128, 16, E8 if cache == "e4m3" else BF, seed=16)
    q = rand(17, 3, 4, 1, 128)
    clean = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    if what == "q":
        q = q.clone()
        q[2, 3, 0, 5] = math.nan
    else:
        page, row = int(p.pages[2, 333 // 16]), 333 % 16
        if cache == "e4m3":
            getattr(p, what + "_scale").view(torch.uint8)[page, 1, row] = 255
        else:
            getattr(p, what)[page, 1, row] = math.nan
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    done()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[2, 3 if what == "q" else slice(2, 4)] = True
    assert torch.isnan(got[hit]).all()
    assert torch.equal(got[~hit], clean[~hit])


def test_infinite_scores_give_nan_and_minus_infinite_ones_nothing():
    lengths = [70, 70]
    p = Paged(lengths, 1, 128, 16, BF, seed=18)
    q = rand(19, 2, 1, 1, 128)
    q[..., 0] = 1.0
    for b, x in ((0, math.inf), (1, -math.inf)):
        p.k[int(p.pages[b, 2]), 0, 3] = 0
        p.k[int(p.pages[b, 2]), 0, 3, 0] = x
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    done()
    assert torch.isnan(got[0]).all()
    rows = [r for r in range(70) if r != 35]
    want, bound = attention(p, q, lengths, None, None, None, keys=lambda b, n: (p.rows("k", b, n)[:, rows], p.rows("v", b, n)[:, rows]))
    check(got[1], want[1], bound[1])


def test_infinities_in_the_cache_stay_what_they_are():
    # a value row with +inf or -inf gives that infinity in its column, both give NaN, no other column changes
    for dtype in (BF, FP):
        p = Paged([150], 1, 128, 16, dtype, seed=60)
        q = rand(61, 1, 4, 1, 128, dtype=dtype)
        clean = kf.decode_attention(q, p.cache, p.pages, ints([150]))
        at = [(int(p.pages[0, r // 16]), r % 16) for r in (3, 77, 149)]
        p.v[at[0][0], 0, at[0][1], 5], p.v[at[1][0], 0, at[1][1], 9] = math.inf, -math.inf
        p.v[at[0][0], 0, at[0][1], 40], p.v[at[2][0], 0, at[2][1], 40] = math.inf, -math.inf
        got = kf.decode_attention(q, p.cache, p.pages, ints([150]))
        done()
        assert (got[..., 5] == math.inf).all() and (got[..., 9] == -math.inf).all() and torch.isnan(got[..., 40]).all()
        keep = [c for c in range(128) if c not in (5, 9, 40)]
        assert torch.equal(got[..., keep], clean[..., keep])


def test_pools_inside_one_tensor():
    # K and V pages side by side, [n_pages, 2, Hkv, page, D], as one allocation
    p = Paged([100, 37], 2, 128, 32, BF, seed=62)
    both = torch.stack((p.k, p.v), 1)
    q, new = rand(63, 2, 4, 1, 128), rand(64, 2, 2, 1, 128)
    got = kf.decode_step(q, new, new, (both[:, 0], both[:, 1]), p.pages, ints([100, 37]))
    want = kf.decode_step(q, new, new, p.cache, p.pages, ints([100, 37]))
    done()
    assert torch.equal(got, want) and torch.equal(both[:, 0], p.k) and torch.equal(both[:, 1], p.v)


def test_thousands_of_sequences():
    lengths = [1 + b % 3 if b % 5 else 0 for b in range(5000)]
    p = Paged(lengths, 1, 128, 16, BF, seed=65)
    q = rand(66, 5000, 1, 1, 128)
    got = kf.decode_attention(q, p.cache, p.pages, ints(lengths))
    done()
    n = torch.tensor(lengths, device="cuda")
    k, v = (x[p.pages.clamp_min(0).long()[:, 0], 0, :3].double() for x in (p.k, p.v))  # [B, 3, D]
    s = torch.einsum("bd,bnd->bn", q[:, 0, 0].double(), k) * 128 ** -0.5
    w = torch.softmax(s.masked_fill(torch.arange(3, device="cuda")[None] >= n[:, None], -math.inf), -1).nan_to_num(0)
    want = torch.einsum("bn,bnd->bd", w, v)
    # the output's rounding, and scores off by 2^-16 of |q||k| (about 11.3 of them): p off by 2^-12 of p at most, values below 6
    assert ((got[:, 0, 0].double() - want).abs() <= want.abs() * U[BF] + 6 * 2.0 ** -11).all()


# ---- rows --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,hkv,page,s", [(128, 2, 16, 1), (128, 8, 48, 40), (256, 3, 16, 33), (256, 1, 128, 200)])
@pytest.mark.parametrize("cache,norm,rope", [("16", True, True), ("16", False, True), ("16", True, False), ("16", False, False),
                                             ("e4m3", True, True), ("e4m3", False, False)])
def test_append(dtype, d, hkv, page, s, cache, norm, rope):
    start, counts = [0, 7, 100, 31, 15], [s, max(0, s - 3), s, 0, 1]
    held = [a + n for a, n in zip(start, counts)]
    p = Paged(held, hkv, d, page, E8 if cache == "e4m3" else dtype, seed=20)
    k, v = (rand(i, 5, s, hkv * d, dtype=dtype).view(5, s, hkv, d).transpose(1, 2) for i in (21, 22))
    gk = weights(23, d, dtype) if norm else None
    cos, sin = tables(max(held), d, dtype, "cuda") if rope else (None, None)
    before = [t.view(torch.uint8).clone() for t in p.cache]
    assert kf.append_rows(p.cache, k, v, p.pages, ints(start), gk, cos, sin, counts=ints(counts)) is not None
    done()
    written = torch.zeros(p.k.shape[0], page, dtype=torch.bool)
    for b in range(5):
        n = counts[b]
        if n == 0:
            continue
        for r in range(start[b], held[b]):
            written[int(p.pages[b, r // page]), r % page] = True
        t = (None, None) if not rope else (cos[start[b]: held[b]], sin[start[b]: held[b]])
        want, off = transform(k[b, :, :n], gk, *t)
        got_k, got_v = p.rows("k", b, held[b])[:, start[b]:], p.rows("v", b, held[b])[:, start[b]:]
        if cache == "16":
            least = 2.0 ** -25 if dtype == FP else 0.0  # half a step of the smallest numbers
            assert ((got_k - want).abs() <= off + (want.abs() + off) * U[dtype] + least).all()
            assert torch.equal(got_v, v[b, :, :n].double())
        else:
            q8, e = quantise(v[b, :, :n].double())
            assert torch.equal(got_v, q8 * two(e)[..., None])
            # the scale is the smallest that holds the row (up to what 32 bits lose of its largest value), each value half a
            # step of e4m3 from its own, or half of its smallest step
            at = p.pages[b, torch.arange(start[b], held[b], device="cuda") // page].long()
            e = p.k_scale.view(torch.uint8)[at, :, torch.arange(start[b], held[b], device="cuda") % page].double().t() - 127
            big = want.abs().amax(-1)
            assert (big <= 448 * two(e) * (1 + 1e-5)).all() and (big >= 224 * two(e) * (1 - 1e-5)).all()
            assert ((got_k - want).abs() <= off + (want.abs() + off) * 2.0 ** -4 + 2.0 ** -10 * two(e)[..., None]).all()
    # nothing else was touched
    for t, was in zip(p.cache, before):
        t, keep = t.view(torch.uint8), (~written).cuda()
        a, c = t.transpose(1, 2)[keep], was.transpose(1, 2)[keep]
        assert torch.equal(a, c)


def test_append_of_extreme_rows():
    # zeros, subnormals, the largest numbers, infinities and NaN into an 8-bit cache
    k = torch.zeros(1, 1, 8, 128, dtype=BF, device="cuda")
    k[0, 0, 1] = 1e-39
    k[0, 0, 2, 5] = 3.3e38
    k[0, 0, 3, 7], k[0, 0, 4, 9] = math.inf, math.nan
    k[0, 0, 5] = 448.0
    k[0, 0, 6, 0], k[0, 0, 6, 1] = 450.0, 1.0
    k[0, 0, 7] = -3.0
    p = Paged([16], 1, 128, 16, E8, seed=24)
    kf.append_rows(p.cache, k, k, p.pages, ints([2]))
    got, same = kf.read_rows(p.cache, p.pages, ints([10]), 10)
    done()
    q8, e = quantise(k[0, 0].double())
    want = q8 * two(e)[..., None]
    for x in (got[0, 0, 2:], same[0, 0, 2:]):
        assert torch.isnan(x[3]).all() and torch.isnan(x[4]).all()
        for r in (0, 1, 2, 5, 6, 7):
            assert torch.equal(x[r].double(), want[r]), r


@pytest.mark.parametrize("cache,dtype", [("16", BF), ("16", FP), ("e4m3", BF), ("e4m3", FP)])
@pytest.mark.parametrize("d,hkv,page,s", [(128, 2, 16, 1), (128, 3, 48, 100), (256, 2, 64, 333)])
def test_read(cache, dtype, d, hkv, page, s):
    lengths = [min(s, 5), 0, s, s + 40, -1, max(1, s - 1)]
    p = Paged(lengths, hkv, d, page, E8 if cache == "e4m3" else dtype, seed=25, strided=True)
    fill_nan_behind(p, lengths)
    got = kf.read_rows(p.cache, p.pages, ints(lengths), s, dtype=dtype)
    flat = [torch.full((6, s, hkv, d), 5.0, dtype=dtype, device="cuda") for _ in range(2)]
    into = kf.read_rows(p.cache, p.pages, ints(lengths), s, k_out=flat[0].transpose(1, 2), v_out=flat[1].transpose(1, 2))
    done()
    for name, x, y in zip("kv", got, into):
        want = torch.zeros(6, hkv, s, d, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lengths):
            if n > 0:
                want[b, :, : min(n, s)] = p.rows(name, b, n)[:, :s]
        assert torch.equal(x, want.to(dtype)) and torch.equal(x, y)


# ---- together ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", ["16", "e4m3"])
@pytest.mark.parametrize("dtype,d,hq,hkv,page", [(BF, 128, 8, 2, 16), (FP, 256, 4, 4, 32), (BF, 128, 20, 1, 48), (FP, 128, 9, 3, 16)])
def test_step_is_append_then_attention(cache, dtype, d, hq, hkv, page):
    lengths = [1, 16, 17, 64, 65, 0, 193, 400, -1, 128]
    cache_dtype = E8 if cache == "e4m3" else dtype
    a, c = (Paged(lengths, hkv, d, page, cache_dtype, seed=26) for _ in range(2))
    q, k, v = (rand(27 + i, 10, 1, h * d, dtype=dtype).view(10, 1, h, d).transpose(1, 2) for i, h in enumerate((hq, hkv, hkv)))
    gq, gk = weights(30, d, dtype), weights(31, d, dtype)
    cos, sin = tables(400, d, dtype, "cuda")
    got = kf.decode_step(q, k, v, a.cache, a.pages, ints(lengths), gq, gk, cos, sin)
    kf.append_rows(c.cache, k, v, c.pages, ints([max(n, 1) - 1 for n in lengths]), gk, cos, sin,
                   counts=ints([int(n > 0) for n in lengths]))
    want = kf.decode_attention(q, c.cache, c.pages, ints(lengths), gq, cos, sin)
    done()
    for x, y in zip(a.cache, c.cache):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert torch.equal(got, want)
    check(got, *attention(a, q, lengths, gq, cos, sin))


@pytest.mark.parametrize("cache", ["16", "e4m3"])
def test_prefill_then_generate(cache):
    """A prompt through optimized_attention, its prepared keys into the cache, then steps; each step's output is that of
    attention over the whole sequence so far."""
    b, s, hq, hkv, d, steps = 3, 75, 8, 2, 128, 20
    q, k, v, gq, gk, cos, sin = [x.cuda() for x in kf.make_inputs(b, s + steps, hq, hkv, d, seed=32)]
    kn = torch.empty_like(k[:, :, :s])
    kf.optimized_attention(*(x[:, :, :s].contiguous() for x in (q, k, v)), gq, gk, cos[:s].contiguous(), sin[:s].contiguous(),
                           causal=True, kn=kn)
    pool = kf.PagedCache.allocate(3 * 6 + 1, 16, hkv, d, E8 if cache == "e4m3" else BF)
    pages = torch.randperm(18, generator=torch.Generator().manual_seed(33)).int().view(3, 6).cuda()
    kf.append_rows(pool, kn, v[:, :, :s], pages, ints([0] * b))
    lengths = ints([s] * b)
    whole = kf.optimized_attention(q, k, v, gq, gk, cos, sin, causal=True)
    for i in range(steps):
        lengths += 1
        t = slice(s + i, s + i + 1)
        got = kf.decode_step(q[:, :, t], k[:, :, t], v[:, :, t], pool, pages, lengths, gq, gk, cos, sin)
        # the prefill rounds q and k a few times more: scores differ by up to 3 u |q||k| scale = 3 * 2^-8 * 11.3 (rows of
        # norm sqrt(128) times a gamma near 1), and an 8-bit key or value by 2^-4 in each component, at random signs
        off = (got.double() - whole[:, :, t].double()).norm() / whole[:, :, t].double().norm()
        assert off < (0.15 if cache == "e4m3" else 3 * 2.0 ** -8 * 11.3), (i, float(off))
    k_back, v_back = kf.read_rows(pool, pages, lengths, s + steps)
    done()
    if cache == "16":
        assert torch.equal(k_back[:, :, :s], kn) and torch.equal(v_back, v)


def test_captured_steps_follow_lengths_and_tables():
    lengths = ints([5, 130, 0, 64])
    most = [200, 700, 100, 300]
    p, fresh = (Paged(most, 2, 128, 16, BF, seed=34) for _ in range(2))
    q, k, v = rand(35, 4, 8, 1, 128), rand(36, 4, 2, 1, 128), rand(37, 4, 2, 1, 128)
    cos, sin = tables(700, 128, BF, "cuda")
    pages = p.pages.clone()
    kf.decode_step(q, k, v, p.cache, pages, lengths, None, None, cos, sin)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kf.decode_step(q, k, v, p.cache, pages, lengths, None, None, cos, sin)
        graphs.append((g, out))
    for new in ([6, 131, 1, 65], [200, 700, 100, 300], [0, 0, 0, 0], [33, 257, 64, 16]):
        lengths.copy_(ints(new))
        pages.copy_(p.pages.flip(1) if new[0] == 33 else p.pages)
        if new[0] == 33:
            pages[:] = p.pages[torch.tensor([0, 1, 2, 3], device="cuda")]
        for g, out in graphs:
            out.fill_(math.nan)
            g.replay()
            torch.cuda.synchronize()
            fresh.k.copy_(p.k)
            fresh.v.copy_(p.v)
            want = kf.decode_step(q, k, v, fresh.cache, pages, ints(new), None, None, cos, sin)
            done()
            assert torch.equal(out, want)
    # two graphs and eager calls at the same time: no workspace is shared
    lengths.copy_(ints(most))
    want = kf.decode_attention(q, p.cache, pages, lengths, None, cos, sin)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, out), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            e = kf.decode_attention(q, fresh.cache, pages, lengths, None, cos, sin)
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], graphs[1][1])
    done()


def test_streams_and_workspace():
    lengths = [2000, 900]
    p = Paged(lengths, 2, 128, 64, BF, seed=38)
    q = rand(39, 2, 8, 1, 128)
    n = ints(lengths)
    want = kf.decode_attention(q, p.cache, p.pages, n)
    ws = torch.empty(kf.decode_workspace_bytes(q, p.cache), dtype=torch.uint8, device="cuda").fill_(255)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = kf.decode_attention(q, p.cache, p.pages, n, workspace=ws)
    st.synchronize()
    done()
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="workspace"):
        kf.decode_attention(q, p.cache, p.pages, n, workspace=ws[:-16])


def test_indexes_outside_are_reported_and_nothing_else_is_touched():
    lengths = [40, 100]
    p = Paged(lengths, 2, 128, 16, BF, seed=40, max_pages=7)
    q, k = rand(41, 2, 4, 1, 128), rand(42, 2, 2, 1, 128)
    cos, sin = tables(100, 128, BF, "cuda")
    n = ints(lengths)
    want = kf.decode_attention(q, p.cache, p.pages, n, None, cos, sin)
    done()

    def bad(code, call):
        before = [t.clone() for t in p.cache]
        call()
        with pytest.raises(kf.KernelStatusError, match=str(code)):
            kf.check_status()
        for t, was in zip(p.cache, before):
            assert torch.equal(t, was)

    for entry in (-1, p.n_pages, 2 ** 31 - 1):
        pages = p.pages.clone()
        pages[1, 6] = pages[0, 2] = entry
        bad(911, lambda: kf.decode_attention(q, p.cache, pages, n, None, cos, sin))
        bad(911, lambda: kf.read_rows(p.cache, pages, n, 100))
        bad(911, lambda: kf.append_rows(p.cache, k, k, pages, ints([39, 99])))
    for too_long in ([113, 3], [2 ** 31 - 1, 2 ** 31 - 1]):
        pages = p.pages.clone().clamp_min(0)
        bad(912, lambda: kf.decode_attention(q, p.cache, pages, ints(too_long)))
        bad(912, lambda: kf.read_rows(p.cache, pages, ints(too_long), 100))
    for start in ([112, -1], [2 ** 31 - 1, -2 ** 31]):
        bad(912, lambda: kf.append_rows(p.cache, k, k, p.pages, ints(start)))
    short = cos[:99].contiguous(), sin[:99].contiguous()
    bad(913, lambda: kf.decode_attention(q, p.cache, p.pages, n, None, *short))
    pages = p.pages.clone()
    pages[0, 2] = -1  # (only sequence 1 would write)
    bad(913, lambda: kf.append_rows(p.cache, k[1:], k[1:], p.pages[1:], ints([99]), None, *short))

    # behind a status nothing is written; afterwards all is as before
    kf.status_word(q.device).fill_(901)
    before = [t.clone() for t in p.cache]
    out = torch.full_like(q, 3.0)
    kf.decode_step(q, k, k, p.cache, p.pages, n, None, None, cos, sin, out=out)
    rows = torch.full((2, 2, 100, 128), 3.0, dtype=BF, device="cuda")
    kf.read_rows(p.cache, p.pages, n, 100, k_out=rows, v_out=rows.clone())
    with pytest.raises(kf.KernelStatusError, match="901"):
        kf.check_status()
    assert (out == 3).all() and (rows == 3).all() and all(torch.equal(t, was) for t, was in zip(p.cache, before))
    assert torch.equal(kf.decode_attention(q, p.cache, p.pages, n, None, cos, sin), want)
    done()


def test_a_cache_that_needs_a_gradient_is_refused():
    p = Paged([5, 9], 2, 128, 16, BF, seed=95)
    q, n = rand(96, 2, 4, 1, 128), ints([5, 9])
    for cache in ((p.k.clone().requires_grad_(), p.v), (p.k, p.v.clone().requires_grad_())):
        for call in (lambda: kf.decode_attention(q, cache, p.pages, n), lambda: kf.read_rows(cache, p.pages, n, 9),
                     lambda: kf.append_rows(cache, q[:, :2], q[:, :2], p.pages, n)):
            with pytest.raises(ValueError, match="forward-only"):
                call()
    done()


def test_offsets_past_32_bits():
    # a pool of more than 2^32 bytes, the sequence in its last pages
    n_pages = (1 << 32) // (64 * 128 * 2) + 40
    k = torch.empty(n_pages, 1, 64, 128, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    p = Paged([600], 1, 128, 64, BF, seed=43, spare=0)
    at = n_pages - 1 - torch.arange(10, device="cuda")
    k[at], v[at] = p.k[p.pages[0].long()], p.v[p.pages[0].long()]
    pages = at.int()[None]
    q, new = rand(44, 1, 4, 1, 128), rand(45, 1, 1, 1, 128)
    got = kf.decode_attention(q, (k, v), pages, ints([600]))
    done()
    check(got, *attention(p, q, [600], None, None, None))
    assert torch.equal(kf.read_rows((k, v), pages, ints([600]), 600)[1][0, 0], p.rows("v", 0, 600)[0].to(BF))
    kf.append_rows((k, v), new, new, pages, ints([601]))
    done()
    assert torch.equal(k[at[9], 0, 25], new[0, 0, 0])


def test_positions_of_a_far_token():
    # the rotation takes the row of the token's own position, also far out
    n = 50001
    p = Paged([n], 1, 128, 128, BF, seed=46)
    q, new, gk = rand(47, 1, 2, 1, 128), rand(48, 1, 1, 1, 128), weights(49, 128, BF)
    cos, sin = tables(n, 128, BF, "cuda")
    got = kf.decode_step(q, new, new, p.cache, p.pages, ints([n]), gk, gk, cos, sin)
    done()
    want, off = transform(new[0, :, 0], gk, cos[n - 1], sin[n - 1])
    assert ((p.rows("k", 0, n)[:, -1] - want).abs() <= off + (want.abs() + off) * U[BF]).all()
    check(got, *attention(p, q, [n], gk, cos, sin))
