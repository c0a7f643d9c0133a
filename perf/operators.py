"""The serving operators on a paged key-value cache, as cases for timing: rows appended to a cache, read back from it, the
attention of one new token over it, and the step that does the first and the last together.

A case is a dict of plain values:
  op       "append"  ``append_rows``: a chunk of new K/V rows into a 16-bit cache (K normed and rotated on the way)
           "store"   ``append_rows`` into an e4m3 cache, then ``read_rows`` of all that the sequences hold
           "read"    ``read_rows`` from a 16-bit cache
           "decode"  ``decode_attention``: one query token per sequence against its cached rows
           "step"    ``decode_step``: the new token's K/V appended and its attention, in one call
  B, S     sequences, and the longest one's rows: new rows for "append" and "store", cached rows for the others
  ragged   lengths differ (one is full; with four or more sequences one has a single row and one has none)
  start    rows already cached in front of an appended chunk (of the longest sequence)
  Hq, Hkv, D, page (rows of a page), dtype "bf16" / "fp16", cache "16" (as dtype) / "e4m3", norm, rope
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6
_THETA = {128: 1e6, 256: 1e4}

# 16-bit K and V bytes of the largest listed cases, were all sequences the longest; drawn ones stay below.
_MAX_DECODE_BYTES = 5.0e9
_MAX_ROWS_BYTES = 2.5e8


def _case(op, B, S, Hq, Hkv, D, dtype, cache="16", page=16, ragged=False, start=0, norm=True, rope=True):
    return {"op": op, "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "cache": cache, "page": page,
            "ragged": ragged, "start": start, "norm": norm, "rope": rope}


def listed():
    def named(name, *a, **kw):
        return {"name": name, **_case(*a, **kw)}

    return [
        # a prompt batch's rows go into the cache after the prefill
        named("append_prompts", "append", 8, 2048, 32, 8, 128, "bf16"),
        # one new row for each of many sequences at different positions
        named("append_tokens", "append", 200, 1, 16, 8, 256, "fp16", page=32, ragged=True, start=1500),
        # chunks of ragged prompts into an 8-bit cache, and the whole prefix read back for the next chunk's prefill
        named("store_e4m3", "store", 8, 1000, 32, 8, 128, "bf16", "e4m3", ragged=True, start=1037),
        # cached prompts back to contiguous rows, to move or reuse them
        named("read_prefixes", "read", 16, 2100, 32, 8, 128, "bf16", page=64, ragged=True),
        # one short conversation: latency is what counts
        named("decode_one_short", "decode", 1, 129, 32, 8, 128, "bf16"),
        # one very long document
        named("decode_one_long", "decode", 1, 131072, 32, 8, 128, "bf16", page=64),
        # throughput serving: many long sequences of different lengths
        named("decode_large", "decode", 128, 12000, 32, 8, 128, "bf16", ragged=True),
        # wide heads, fp16, few query heads to a KV head
        named("decode_wide_fp16", "decode", 16, 2047, 16, 8, 256, "fp16", page=48, ragged=True),
        # the same service from an 8-bit cache
        named("decode_e4m3", "decode", 64, 8192, 32, 8, 128, "bf16", "e4m3", ragged=True),
        # one rank's share of a model split by KV head over eight GPUs, 8-bit cache, long sequences
        named("decode_shard_e4m3", "decode", 24, 20000, 8, 1, 128, "fp16", "e4m3", page=128, ragged=True),
        # a whole step of one conversation
        named("step_one", "step", 1, 1000, 32, 8, 128, "bf16"),
        # a whole step of a small ragged batch
        named("step_batch", "step", 32, 1500, 32, 8, 128, "bf16", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "store", "read", "decode", "decode", "decode", "step"])
    D = rng.choice([128, 128, 256])
    # whole models, one rank's share of them, many query heads to a KV head, heads without sharing
    Hq, Hkv = rng.choice([(16, 8), (8, 4), (2, 1), (16, 1)] if D == 256 else
                         [(32, 8), (32, 8), (4, 1), (8, 1), (40, 8), (32, 2), (12, 12), (24, 1)])
    cache = {"append": "16", "store": "e4m3", "read": "16", "step": "16"}.get(op) or rng.choice(["16", "e4m3"])
    page = rng.choice([16, 16, 32, 64, 128, 80])
    c = _case(op, _log(rng, 1, 160), 1, Hq, Hkv, D, rng.choice(["bf16", "fp16"]), cache, page, rng.random() < 0.7,
              0, rng.random() < 0.8, rng.random() < 0.85)
    if op in ("append", "store"):
        c["S"] = 1 if rng.random() < 0.3 else _log(rng, 2, 6000)
        c["start"] = rng.choice([0, _log(rng, 1, 4000)])
        limit = _MAX_ROWS_BYTES
    else:
        c["S"] = _log(rng, 1, 9000 if op != "decode" else 100000)
        limit = _MAX_DECODE_BYTES if op == "decode" else _MAX_ROWS_BYTES
    while (c["S"] + c["start"]) * c["B"] * Hkv * D * 4 > limit:  # K and V in 16 bits, all sequences at the longest
        if c["B"] > 1:
            c["B"] = c["B"] * 3 // 4
        else:
            c["S"], c["start"] = max(1, c["S"] * 3 // 4), c["start"] * 3 // 4
    return c


def _spread(case, longest):
    """Rows of each sequence, from the case alone."""
    B = case["B"]
    if not case["ragged"]:
        return [longest] * B
    low = longest // 4
    rows = [max(1, low + (longest - low) * ((7919 * (i + 1) + 104729 * longest) % 1009) // 1009) for i in range(B)]
    rows[B // 2] = longest
    if B >= 4:
        rows[1], rows[B - 1] = 1, 0  # a sequence that has just begun, and a padding entry of the batch
    return rows


def _rows(case):
    """(rows cached before the call, rows that the call adds, rows that it reads) of each sequence."""
    rows = _spread(case, case["S"])
    if case["op"] in ("append", "store"):
        before = [n if r else 0 for n, r in zip(_spread(case, case["start"]), rows)] if case["start"] else [0] * case["B"]
        return before, rows, [a + b for a, b in zip(before, rows)]
    return rows, [0] * case["B"], rows


def _tables(positions, D):
    """cos and sin of each position, both halves, in 64 bits: far angles need them."""
    dev = torch.device("cuda", torch.cuda.current_device())
    freq = _THETA[D] ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
    angle = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * freq
    angle = torch.cat((angle, angle), -1)
    return angle.cos(), angle.sin()


def prepare(case, seed):
    dtype = _DTYPES[case["dtype"]]
    B, Hq, Hkv, D, page = (case[n] for n in ("B", "Hq", "Hkv", "D", "page"))
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    def heads(rows, h):  # a projection's output [B,S,H*D], as a model views it
        return normal(B, rows, h * D).view(B, rows, h, D).transpose(1, 2)

    before, added, held = _rows(case)
    # the pool: every sequence's pages lie anywhere in it, a few are free; entries without a page are -1
    need = [-(-n // page) for n in held]
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen, device=dev).int()
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    at = 0
    order = order.cpu()
    for b, n in enumerate(need):
        table[b, :n] = order[at: at + n]
        at += n
    state = {"case": case, "pages": table.to(dev)}
    if case["cache"] == "e4m3":
        for n in ("k", "v"):
            state[n + "_pages"] = (normal(total, Hkv, page, D) * 110).clamp_(-448, 448).to(torch.float8_e4m3fn)
            state[n + "_scale"] = torch.randint(119, 122, (total, Hkv, page), generator=gen, device=dev,
                                                dtype=torch.uint8).view(torch.float8_e8m0fnu)
    else:
        state["k_pages"], state["v_pages"] = normal(total, Hkv, page, D), normal(total, Hkv, page, D)
        state["k_scale"] = state["v_scale"] = None
    state["cos"] = state["sin"] = state["gq"] = state["gk"] = None
    if case["rope"]:
        state["cos"], state["sin"] = (t.to(dtype) for t in _tables(max(held), D))
    if case["norm"]:  # the weights of Q and K: scores then spread by a few units
        state["gq"], state["gk"] = ((1.5 + 0.1 * torch.randn(D, generator=gen, device=dev)).to(dtype) for _ in range(2))

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    if case["op"] in ("append", "store"):
        state["k"], state["v"] = heads(case["S"], Hkv), heads(case["S"], Hkv)
        state["start"], state["counts"] = ints(before), ints(added)
    if case["op"] in ("decode", "step"):
        state["q"] = heads(1, Hq)
    if case["op"] == "step":
        state["k"], state["v"] = heads(1, Hkv), heads(1, Hkv)
    state["lengths"], state["longest"] = ints(held), max(held)
    state["cache"] = (state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"])
    return state


# ---- plain form: elementary operations in 32 bits --------------------------------------------------------------------
def _transform(x, gamma, cos, sin):
    x = x.float()
    if gamma is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * gamma.float()
    if cos is not None:
        half = x.shape[-1] // 2
        x = x * cos.float() + torch.cat((-x[..., half:], x[..., :half]), -1) * sin.float()
    return x


def _quantise(x):
    """e4m3 values and the exponent byte of each row's power-of-two scale: the smallest that keeps the row within 448."""
    largest = x.abs().amax(-1)
    m, e = torch.frexp(largest)  # largest = m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    e = (e - 9 + (m > 0.875).int()).clamp(-126, 119)
    e = torch.where(largest > 0, e, torch.full_like(e, -126))
    q = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    return q, torch.where(torch.isfinite(largest), e + 127, torch.full_like(e, 255)).to(torch.uint8)


def _put(pool, scale, at, slot, rows):
    if scale is None:
        pool[at, :, slot] = rows.to(pool.dtype)
    else:
        q, e = _quantise(rows)
        pool.view(torch.uint8)[at, :, slot] = q.view(torch.uint8)
        scale.view(torch.uint8)[at, :, slot] = e


def _plain_append(s, k, v, start, counts):
    """Rows of k and v [B,Hkv,S,D] to positions start + i of the sequences, i < counts."""
    page = s["k_pages"].shape[2]
    b, i = torch.nonzero(torch.arange(k.shape[2], device=k.device)[None] < counts[:, None], as_tuple=True)
    pos = start[b].long() + i
    at, slot = s["pages"][b, pos // page].long(), pos % page
    tables = (None, None) if s["cos"] is None else (s["cos"][pos][:, None], s["sin"][pos][:, None])
    _put(s["k_pages"], s["k_scale"], at, slot, _transform(k[b, :, i], s["gk"], *tables))  # [rows, Hkv, D]
    _put(s["v_pages"], s["v_scale"], at, slot, v[b, :, i].float())


def _cached(s, pool, scale, longest):
    """Rows 0..longest-1 of every sequence in 32 bits, [B, Hkv, longest, D], zero behind its own length."""
    at = s["pages"].clamp_min(0).long()
    x = pool.view(torch.uint8)[at].view(pool.dtype).float() if scale is not None else pool[at].float()
    if scale is not None:
        x = x * scale.view(torch.uint8)[at].view(scale.dtype).float()[..., None]
    x = x.transpose(1, 2).flatten(2, 3)[:, :, :longest]
    return x.masked_fill_(~_held(s, longest)[:, None, :, None], 0)


def _held(s, longest):
    return torch.arange(longest, device=s["pages"].device)[None] < s["lengths"][:, None]


def _plain_read(s, longest):
    dtype = _DTYPES[s["case"]["dtype"]]
    return (_cached(s, s["k_pages"], s["k_scale"], longest).to(dtype), _cached(s, s["v_pages"], s["v_scale"], longest).to(dtype))


def _plain_decode(s, longest):
    q = s["q"][:, :, 0]
    B, Hq, D = q.shape
    Hkv = s["k_pages"].shape[1]
    newest = (s["lengths"] - 1).clamp_min(0).long()
    tables = (None, None) if s["cos"] is None else (s["cos"][newest][:, None], s["sin"][newest][:, None])
    qn = _transform(q, s["gq"], *tables).view(B, Hkv, Hq // Hkv, D) * D ** -0.5
    score = qn @ _cached(s, s["k_pages"], s["k_scale"], longest).transpose(2, 3)
    score.masked_fill_(~_held(s, longest)[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))  # a sequence without rows has no maximum
    p = torch.where((s["lengths"] > 0)[:, None, None, None], p, torch.zeros_like(p))
    o = p @ _cached(s, s["v_pages"], s["v_scale"], longest)
    return (o / p.sum(-1, keepdim=True).clamp_min(1e-30)).reshape(B, Hq, 1, D).to(q.dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        import kernelfuser_b200 as kf
        cache, pages = s["cache"], s["pages"]
        if c["op"] in ("append", "store"):
            kf.append_rows(cache, s["k"], s["v"], pages, s["start"], s["gk"], s["cos"], s["sin"], counts=s["counts"])
            if c["op"] == "store":
                return kf.read_rows(cache, pages, s["lengths"], s["longest"], dtype=s["k"].dtype)
            return s["k_pages"], s["v_pages"]
        if c["op"] == "read":
            return kf.read_rows(cache, pages, s["lengths"], s["longest"])
        if c["op"] == "decode":
            return kf.decode_attention(s["q"], cache, pages, s["lengths"], s["gq"], s["cos"], s["sin"])
        out = kf.decode_step(s["q"], s["k"], s["v"], cache, pages, s["lengths"], s["gq"], s["gk"], s["cos"], s["sin"])
        return out, s["k_pages"], s["v_pages"]
    if c["op"] in ("append", "store"):
        _plain_append(s, s["k"], s["v"], s["start"], s["counts"])
        return (s["k_pages"], s["v_pages"]) if c["op"] == "append" else _plain_read(s, s["longest"])
    if c["op"] == "read":
        return _plain_read(s, s["longest"])
    if c["op"] == "decode":
        return _plain_decode(s, s["longest"])
    newest = s["lengths"] - 1
    _plain_append(s, s["k"], s["v"], newest, (newest >= 0).int())
    return _plain_decode(s, s["longest"]), s["k_pages"], s["v_pages"]


def work(case):
    B, Hq, Hkv, D = (case[n] for n in ("B", "Hq", "Hkv", "D"))
    before, added, held = _rows(case)
    size = 1 if case["cache"] == "e4m3" else 2
    row = 2 * Hkv * (D * size + (1 if size == 1 else 0))  # K and V of one token in the cache
    new = 2 * Hkv * D * 2  # and as the projections give it
    table = 2 * D * 2 if case["rope"] else 0
    weights = D * 2 if case["norm"] else 0
    entries = 4 * sum(-(-n // case["page"]) for n in held) + 4 * B
    if case["op"] in ("append", "store"):
        positions = set()
        for a, n in zip(before, added):
            positions.update(range(a, a + n))
        nbytes = sum(added) * (new + row) + len(positions) * table + weights + entries
        flops = 12 * sum(added) * Hkv * D
        if case["op"] == "store":  # what is read back: the older rows, and the whole result written
            nbytes += sum(before) * row + B * max(held) * new
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "read":
        return {"bytes": sum(held) * row + B * max(held) * new + entries, "flops": 0}
    nbytes = sum(held) * row + B * Hq * D * 2 * 2 + len(set(held)) * table + weights + entries
    flops = 4 * sum(held) * Hq * D + 8 * B * Hq * D
    if case["op"] == "step":  # the newest rows come from the projections and are written besides
        nbytes += sum(1 for n in held if n) * new + weights
    return {"bytes": nbytes, "flops": flops}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def _turn64(x, gamma, cos, sin):
    x = x.double()
    if gamma is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt() * gamma.double()
    if cos is not None:
        a, b = x.chunk(2, -1)
        (ca, cb), (sa, sb) = cos.double().chunk(2, -1), sin.double().chunk(2, -1)
        x = torch.cat((a * ca - b * sa, b * cb + a * sb), -1)
    return x


def _two64(e):
    """2^e exactly, for whole numbers e in a tensor of 64-bit values (a device's pow is off by an ulp for some)."""
    powers = torch.tensor([2.0 ** i for i in range(-160, 161)], dtype=torch.float64, device=e.device)
    return powers[(e + 160).long()]


def _eight64(x):
    """The values that an e4m3 row with its power-of-two scale stands for, by arithmetic in 64 bits."""
    largest = x.abs().amax(-1, keepdim=True)
    unit = torch.ones_like(largest)
    ok = (largest > 0) & torch.isfinite(largest)
    exponent = torch.where(ok, torch.ceil(torch.log2(torch.where(ok, largest, unit) / 448)), -126 * unit).clamp(-126, 119)
    exponent = torch.where(largest > 448 * _two64(exponent), exponent + 1, exponent)  # log2 next to a whole number
    exponent = torch.where((largest <= 224 * _two64(exponent)) & (exponent > -126), exponent - 1, exponent)
    y = x * _two64(-exponent)
    place = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)))  # normal from 2^-6, steps of 2^-9 below
    step = _two64(place - 3)
    return torch.where(torch.isfinite(largest), torch.round(y / step) * step * _two64(exponent), torch.nan)


def exact(case, seed):
    s = prepare(case, seed)
    B, Hq, Hkv, D, page = (case[n] for n in ("B", "Hq", "Hkv", "D", "page"))
    before, added, held = _rows(case)
    table = s["pages"].long()

    def sequence(name, b, n):  # rows 0..n-1 of sequence b, [n, Hkv, D]
        pool, scale = s[name + "_pages"], s[name + "_scale"]
        at = table[b, : (n + page - 1) // page]
        if scale is None:
            x = pool.index_select(0, at).double()
        else:
            x = pool.view(torch.uint8).index_select(0, at).view(torch.float8_e4m3fn).double()
            bits = scale.view(torch.uint8).index_select(0, at).long()
            x = x * _two64(bits - 127)[..., None]
        return x.permute(0, 2, 1, 3).reshape(-1, Hkv, D)[:n]

    def turned(x, gamma, first, n):  # [n, H, D] rows at positions first..
        if s["cos"] is None:
            return _turn64(x, gamma, None, None)
        return _turn64(x, gamma, s["cos"][first: first + n, None], s["sin"][first: first + n, None])

    def fresh(b, first, n):  # the new rows of sequence b as they are kept, before the rounding to 16 bits
        k = turned(s["k"][b, :, :n].transpose(0, 1), s["gk"], first, n)
        v = s["v"][b, :, :n].transpose(0, 1).double()
        return (_eight64(k), _eight64(v)) if case["cache"] == "e4m3" else (k, v)

    if case["op"] in ("append", "step"):
        pools = [s["k_pages"].double(), s["v_pages"].double()]
        kept = {}
        for b in range(B):
            first, n = (before[b], added[b]) if case["op"] == "append" else (held[b] - 1, min(held[b], 1))
            if n == 0:
                continue
            kept[b] = fresh(b, first, n)
            for i in range(first // page, (first + n - 1) // page + 1):
                lo, hi = max(first, i * page), min(first + n, (i + 1) * page)
                for pool, rows in zip(pools, kept[b]):
                    pool[table[b, i], :, lo - i * page: hi - i * page] = rows[lo - first: hi - first].transpose(0, 1)
        if case["op"] == "append":
            return tuple(pools)
    if case["op"] in ("read", "store"):
        out = [torch.zeros(B, Hkv, max(held), D, dtype=torch.float64, device=table.device) for _ in range(2)]
        for b in range(B):
            for x, name in zip(out, "kv"):
                if before[b]:
                    x[b, :, : before[b]] = sequence(name, b, before[b]).transpose(0, 1)
            if added[b]:
                for x, rows in zip(out, fresh(b, before[b], added[b])):
                    x[b, :, before[b]: held[b]] = rows.transpose(0, 1)
        return tuple(out)

    out = torch.zeros(B, Hq, 1, D, dtype=torch.float64, device=table.device)
    for b in range(B):
        n = held[b]
        if n == 0:
            continue
        k, v = sequence("k", b, n), sequence("v", b, n)
        if case["op"] == "step":
            # attention sees the newest key as the cache holds it
            k[n - 1], v[n - 1] = (x[0].to(_DTYPES[case["dtype"]]).double() for x in kept[b])
        q = turned(s["q"][b].transpose(0, 1), s["gq"], n - 1, 1)[0]  # [Hq, D]
        for g in range(Hkv):
            part = slice(g * (Hq // Hkv), (g + 1) * (Hq // Hkv))
            p = torch.softmax(q[part] @ k[:, g].t() * D ** -0.5, -1)
            out[b, part, 0] = p @ v[:, g]
    return out if case["op"] == "decode" else (out, *pools)
