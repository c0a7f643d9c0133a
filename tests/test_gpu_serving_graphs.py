"""Captured decode steps: replays follow the page table, and replays and eager calls that run together give what each gives
alone."""
import math

import pytest
import torch

import kernelfuser_b200 as kf
from serving import Paged, tables

pytestmark = pytest.mark.gpu

BF, FP, E8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rand(seed, *shape, dtype=BF):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return torch.randn(*shape, generator=g).to("cuda", dtype)


def done():
    torch.cuda.synchronize()
    kf.check_status()


def moved(p, seed):
    """(the pools' pages in another order, the table that goes with it): the same sequences in other places."""
    order = torch.randperm(p.n_pages, generator=torch.Generator().manual_seed(seed)).cuda()  # page i goes to place order[i]
    new = Paged.__new__(Paged)
    new.__dict__.update(p.__dict__)
    for name in ("k", "v", "k_scale", "v_scale"):
        t = getattr(p, name)
        if t is not None:
            raw = t.view(torch.uint8)
            out = torch.empty_like(raw)
            out[order] = raw
            setattr(new, name, out.view(t.dtype))
    new.pages = torch.where(p.pages >= 0, order[p.pages.clamp_min(0).long()].int(), p.pages)
    return new


@pytest.mark.parametrize("cache,dtype", [("16", BF), ("16", FP), ("e4m3", BF), ("e4m3", FP)])
@pytest.mark.parametrize("lengths,hq,hkv,d", [([5, 130, 0, 64], 8, 2, 128), ([9000, 700, 3], 4, 1, 128), ([6000, 31], 11, 1, 256)])
def test_a_replay_follows_the_table(cache, dtype, lengths, hq, hkv, d):
    cache_dtype = E8 if cache == "e4m3" else dtype
    b = len(lengths)
    p = Paged(lengths, hkv, d, 16, cache_dtype, seed=110)
    q, k, v = rand(111, b, hq, 1, d, dtype=dtype), rand(112, b, hkv, 1, d, dtype=dtype), rand(113, b, hkv, 1, d, dtype=dtype)
    cos, sin = tables(max(lengths), d, dtype, "cuda")
    n = ints(lengths)
    want = kf.decode_step(q, k, v, p.cache, p.pages, n, None, None, cos, sin)
    done()
    # what the graph sees: pools and a table of its own, filled anew before each replay
    own = moved(p, 0)
    pages = p.pages.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kf.decode_step(q, k, v, own.cache, pages, n, None, None, cos, sin)
    for seed in (1, 2, 3):
        other = moved(p, seed)
        assert not torch.equal(other.pages, pages)
        for mine, its in zip(own.cache, other.cache):
            mine.view(torch.uint8).copy_(its.view(torch.uint8))
        newest = [(i, int(other.pages[i, (m - 1) // 16]), (m - 1) % 16) for i, m in enumerate(lengths) if m > 0]
        for _, page, row in newest:  # the step has to write these
            for t in own.cache:
                t.view(torch.uint8)[page, :, row] = 0x7f
        pages.copy_(other.pages)
        out.fill_(math.nan)
        g.replay()
        done()
        assert torch.equal(out, want)
        for mine, its in zip(own.cache, other.cache):
            assert torch.equal(mine.view(torch.uint8), its.view(torch.uint8))


@pytest.mark.parametrize("cache", ["16", "e4m3"])
def test_replays_and_eager_calls_at_the_same_time(cache):
    # two graphs and two eager streams, each with tensors of its own: items that are broken over many CTAs
    lengths = [30000, 700, 9000]
    n = ints(lengths)
    cos, sin = tables(max(lengths), 128, BF, "cuda")
    p = Paged(lengths, 1, 128, 64, E8 if cache == "e4m3" else BF, seed=120)
    sets = [(moved(p, i), rand(121 + i, 3, 8, 1, 128), rand(131 + i, 3, 1, 1, 128)) for i in range(4)]

    def step(s):
        return kf.decode_step(s[1], s[2], s[2], s[0].cache, s[0].pages, n, None, None, cos, sin)

    want = [step(s) for s in sets]
    done()
    assert len({float(w.double().sum()) for w in want}) == 4
    graphs = []
    for s in sets[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(s)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for _ in range(30):
        for g, out in graphs:
            out.fill_(math.nan)
        torch.cuda.synchronize()
        eager = []
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        for s, st in zip(sets[2:], streams[2:]):
            with torch.cuda.stream(st):
                eager.append([step(s) for _ in range(3)])
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert torch.equal(out, w)
        for got, w in zip(eager, want[2:]):
            assert all(torch.equal(x, w) for x in got)
    done()
