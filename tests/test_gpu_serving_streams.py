"""Launches of several streams at a time, however far apart they were enqueued: what they count in is never shared."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import kernelfuser_b200 as kf
from serving import Paged

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def held_apart(call, between, apart):
    """Results of `call` on two streams that start together, `apart` calls of `between` enqueued from the one to the other."""
    gate, first, second = (torch.cuda.Stream() for _ in range(3))
    torch.cuda.synchronize()
    go = torch.cuda.Event()
    with torch.cuda.stream(gate):
        torch.cuda._sleep(200_000_000)  # about a tenth of a second: longer than enqueueing the rest takes
        go.record()
    with torch.cuda.stream(first):
        first.wait_event(go)
        a = call(0)
    with torch.cuda.stream(second):
        for _ in range(apart - 1):
            between()
        second.wait_event(go)
        b = call(1)
    torch.cuda.synchronize()
    kf.check_status()
    return a, b


def test_joins_of_streams_far_apart():
    # items broken over all CTAs: their parts are counted
    lengths = [60000, 9000]
    p = Paged(lengths, 1, 128, 64, BF, seed=100)
    small = Paged([300], 1, 128, 64, BF, seed=101)
    g = torch.Generator().manual_seed(102)
    qs = [torch.randn(2, 4, 1, 128, generator=g).to("cuda", BF) for _ in range(2)]
    q1, n1, n = torch.randn(1, 1, 1, 128, generator=g).to("cuda", BF), ints([300]), ints(lengths)
    want = [kf.decode_attention(q, p.cache, p.pages, n) for q in qs]
    for apart in (1023, 1024, 1025, 2048):
        got = held_apart(lambda i: [kf.decode_attention(qs[i], p.cache, p.pages, n) for _ in range(8)],
                         lambda: kf.decode_attention(q1, small.cache, small.pages, n1), apart)
        for i in range(2):
            assert all(torch.equal(x, want[i]) for x in got[i])
    for _ in range(1100):
        got = kf.decode_attention(qs[0], p.cache, p.pages, n)
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])


@pytest.mark.parametrize("kind", [(2, 1024, 8, 2, 128), (2, 1024, 4, 2, 256), (2, 1024, 3, 1, 256)])
def test_work_counters_of_streams_far_apart(kind):
    def inputs(b, s, hq, hkv, d, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *shape: torch.randn(*shape, generator=g, device="cuda", dtype=BF)
        return r(b, hq, s, d), r(b, hkv, s, d), r(b, hkv, s, d), 1 + 0.1 * r(d), 1 + 0.1 * r(d)

    xs, small = [inputs(*kind, seed=s) for s in (1, 2)], inputs(1, 64, 2, 1, kind[4], seed=3)
    want = [kf.optimized_attention(*x, causal=True, variant=2) for x in xs]
    got = held_apart(lambda i: [kf.optimized_attention(*xs[i], causal=True, variant=3) for _ in range(4)],
                     lambda: kf.optimized_attention(*small, causal=True, variant=3), 1024)
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


MANY_STREAMS = """
import ctypes
import torch
import kernelfuser_b200 as kf
from serving import Paged

rt = ctypes.CDLL('libcudart.so.12')
lengths = [3000, 70]
p = Paged(lengths, 1, 128, 64, torch.bfloat16, seed=103)
q = torch.randn(2, 4, 1, 128, generator=torch.Generator().manual_seed(104)).to('cuda', torch.bfloat16)
n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
want = kf.decode_attention(q, p.cache, p.pages, n)
xs = [torch.randn(2, h, 1024, 128, device='cuda', dtype=torch.bfloat16) for h in (4, 2, 2)]
one = torch.ones(128, device='cuda', dtype=torch.bfloat16)
want_prefill = kf.optimized_attention(*xs, one, one, causal=True, variant=3)
out, ws = torch.empty_like(want), torch.empty(kf.decode_workspace_bytes(q, p.cache), dtype=torch.uint8, device='cuda')
out_prefill, kn = torch.empty_like(xs[0]), torch.empty_like(xs[1])
for i in range(1200):
    h = ctypes.c_void_p()
    assert rt.cudaStreamCreateWithFlags(ctypes.byref(h), 1) == 0
    out.zero_(), ws.fill_(255), out_prefill.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(h.value)):
        kf.decode_attention(q, p.cache, p.pages, n, out=out, workspace=ws)
        kf.optimized_attention(*xs, one, one, causal=True, variant=3, out=out_prefill, kn=kn)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(out_prefill, want_prefill), i
    if i % 2:  # (the handle may come back for another stream)
        assert rt.cudaStreamDestroy(h) == 0
kf.check_status()
"""


def test_more_streams_than_rows():
    # every stream has words to count in; one that finds none left counts in its workspace, or runs a kernel without a counter
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", MANY_STREAMS], cwd=root, env={**os.environ, "PYTHONPATH": f"{root}:{root / 'tests'}"},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
