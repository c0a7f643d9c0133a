"""A close bound on what the attention over a paged cache may be off, from the roundings that its kernels make: queries and
probabilities enter the products as two 16-bit numbers (one f16 number for a bf16 call on an e4m3 cache), the rest is 32
bits.  It is small enough that a result without some of its keys is outside."""
import torch

from serving import U, transform

# what is left of a value that enters the products as high (towards zero) + low (to nearest): v in [1, 2) has a high part off by
# less than a step, 2^-7 (bf16) or 2^-10 (f16), and a low part below that, so off by half a step of it
LEFT = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}
SMS = 148

# (lengths, Hq, Hkv, D) of launches whose items are broken over CTAs, or whole and of many steps
LONG = [([70001], 8, 1, 128), ([9000, 1, 0, 5000, 13], 4, 2, 128), ([20000, 64], 2, 1, 256), ([4097] * 3, 16, 1, 256),
        ([6000, 700], 24, 1, 128), ([900] * 150, 24, 1, 128), ([1500] * 150, 16, 1, 256), ([1300] * 300, 2, 1, 256),
        ([2100] * 450, 3, 1, 128), ([900] * 40, 8, 4, 128)]


def steps_of(lengths, hkv, n):
    """Products in a row that a warp of four adds to its output for a sequence of n keys: of 16 keys each, 64 keys a round.  A
    launch of at least 148 CTAs splits its keys, and a CTA has at most a few hundred more than its share."""
    share = sum(max(x, 0) for x in lengths) * hkv / SMS + 512
    return min(n, share) / 64 + 2


def attention_close(paged, q, lengths, gamma, cos, sin, scale=None, only=None):
    """(out, bound) in 64 bits, [B, Hq, 1, D]; `only`: just these sequences (the others are zero)."""
    b, hq, _, d = q.shape
    hkv = paged.k.shape[1]
    out = torch.zeros(b, hq, 1, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    e8 = paged.k_scale is not None
    left = LEFT[torch.float16] if e8 else LEFT[q.dtype]
    if e8 and q.dtype == torch.bfloat16:
        left = U[torch.float16]  # one f16 number
    half = e8 or q.dtype == torch.float16
    scale = d ** -0.5 if scale is None else scale
    for i, n in enumerate(lengths):
        if n <= 0 or (only is not None and i not in only):
            continue
        k, v = (paged.rows(name, i, n).repeat_interleave(hq // hkv, 0) for name in "kv")
        t = (None, None) if cos is None else (cos[n - 1], sin[n - 1])
        qn, q_off = transform(q[i, :, 0], gamma, *t)
        s = torch.einsum("hd,hnd->hn", qn, k) * scale
        p = torch.softmax(s, -1)
        o = torch.einsum("hn,hnd->hd", p, v)
        # Scores.  A 16-step product of 16 terms and the sum so far loses at most 17 units of 2^-24 of the sum of magnitudes, and
        # there are d / 16; f16 has a smallest step of 2^-24 (an e4m3 cache's q' is scaled up to 2^14 first).
        q_left = qn.abs() * (left + (d + 32) * 2.0 ** -24) + q_off
        if half:
            q_left = q_left + (2.0 ** -38 * qn.abs().amax(-1, keepdim=True) if e8 else 2.0 ** -24)
        off = torch.einsum("hd,hnd->hn", q_left, k.abs()) * scale
        # ... and their way through the exponent: three roundings of numbers of up to the largest score, ex2 within 2^-22
        # (an e4m3 cache: with the value rows' exponents in it)
        rows = v.abs().amax(-1)
        far = torch.log2(rows[rows > 0]).abs().amax() + 9 if e8 else 0.0
        off = off + (s.abs().amax(-1, keepdim=True) + far) * 2.0 ** -21 + 2.0 ** -21
        grow = torch.exp(2 * off.amax(-1, keepdim=True))
        moved = torch.einsum("hn,hnd->hd", p * off, (v - o[:, None]).abs())
        # Probabilities: what is left of each, and in f16 its smallest steps (2^-24, twice, where the largest are 2^11 or more),
        # with an e4m3 cache those of the products of probability and value scale (rows whose largest value is 1 .. 448 of it).
        p_left = p * left
        if half:
            largest = (p * rows).amax(-1, keepdim=True) / rows.clamp_min(1e-300) if e8 else p.amax(-1, keepdim=True)
            p_left = p_left + 2.0 ** -34 * largest * (448 if e8 else 1)
        sums = torch.einsum("hn,hnd->hd", p, v.abs())
        # Sums: products in a row, then warps and parts (a few hundred at most), and the sum of the probabilities
        added = sums * ((17 * steps_of(lengths, hkv, n) + 512) * 2.0 ** -24)
        e = (moved + torch.einsum("hn,hnd->hd", p_left, v.abs())) * grow + added
        out[i, :, 0] = o
        bound[i, :, 0] = e + (o.abs() + e) * U[q.dtype] + (2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134)
    return out, bound


def region_values(paged, lengths):
    """Value rows that say where in the sequence they stand: row p of n holds a one in column p * D // n and zeros, so that column c
    of the result is the weight of one D-th of the sequence.  (An e4m3 cache: scale 1.)"""
    d = paged.v.shape[-1]
    for b, n in enumerate(lengths):
        if n <= 0:
            continue
        pages = -(-n // paged.page)
        col = (torch.arange(pages * paged.page, device=paged.v.device) * d // n).clamp_max(d - 1)
        rows = torch.zeros(pages * paged.page, d, device=paged.v.device).scatter_(1, col[:, None], 1.0).to(paged.v.dtype)
        at, rows = paged.pages[b, :pages].long(), rows.view(pages, 1, paged.page, d).expand(-1, paged.v.shape[1], -1, -1)
        if paged.v_scale is None:
            paged.v[at] = rows
        else:
            paged.v.view(torch.uint8)[at] = rows.contiguous().view(torch.uint8)
    if paged.v_scale is not None:
        paged.v_scale.view(torch.uint8).fill_(127)
