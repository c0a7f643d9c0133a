"""What the tests of the serving operators share: random caches, and the operators in 64 bits with bounds on how far a
kernel that rounds where these do may be off (element by element, from the roundings alone)."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative to the value
EPS = 1e-6


def tables(n, d, dtype, device, theta=1e4):
    freq = theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    a = torch.arange(n, dtype=torch.float64)[:, None] * freq
    a = torch.cat((a, a), -1)
    return a.cos().to(device, dtype), a.sin().to(device, dtype)


def two(e):
    """2^e, exactly."""
    return torch.tensor([2.0 ** i for i in range(-200, 201)], dtype=torch.float64, device=e.device)[(e + 200).long()]


def transform(x, gamma, cos, sin):
    """(row in 64 bits, bound on what 32-bit arithmetic loses of it: relative to the terms that are added up)."""
    x = x.double()
    if gamma is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma.double()
    terms = x.abs()
    if cos is not None:
        lo, hi = x.chunk(2, -1)
        c, s = cos.double(), sin.double()
        swapped = torch.cat((-hi, lo), -1)
        x, terms = x * c + swapped * s, terms * c.abs() + swapped.abs() * s.abs()
    # rsqrt and four products or sums, each within two units of 2^-24
    return x, terms * 2.0 ** -20


def quantise(x):
    """e4m3 values and exponent of the row's power of two (at most 119), by arithmetic in 64 bits."""
    big = x.abs().amax(-1)
    e = torch.full(big.shape, -126.0, dtype=torch.float64, device=x.device)
    for k in range(-126, 119):  # the smallest with big <= 448 * 2^e
        e = torch.where(big > 448 * 2.0 ** k, torch.full_like(e, k + 1.0), e)
    y = (x * two(-e)[..., None]).clamp(-448, 448)
    place = torch.frexp(y.abs().clamp_min(2.0 ** -6))[1].double() - 1
    step = two(place - 3)
    return torch.round(y / step) * step, e


class Paged:
    """A pool in random order with a table, its rows as 64-bit tensors, and strides that are not the tight ones."""

    def __init__(self, lengths, hkv, d, page, cache_dtype, seed=0, device="cuda", spare=2, max_pages=None, strided=False,
                 spread=1.0):
        g = torch.Generator(device="cpu").manual_seed(seed)
        need = [max(0, -(-n // page)) for n in lengths]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, generator=g)
        width = max_pages or max(1, max(need))
        table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at: at + n].int()
            at += n
        self.pages = table.to(device)
        self.need, self.page = need, page
        shape = (self.n_pages, hkv, page, d)
        e8 = cache_dtype == torch.float8_e4m3fn

        def pool():
            x = torch.randn(shape, generator=g)
            if e8:
                x = (x * 100).clamp(-448, 448)
            x = (x * spread).to(cache_dtype) if not e8 else x.to(cache_dtype)
            if strided:  # [n_pages, page, Hkv, D] in memory
                raw = x.view(torch.uint8) if e8 else x
                raw = raw.transpose(1, 2).contiguous().to(device).transpose(1, 2)
                return raw.view(cache_dtype) if e8 else raw
            return (x.view(torch.uint8).to(device).view(cache_dtype)) if e8 else x.to(device)

        self.k, self.v = pool(), pool()
        self.k_scale = self.v_scale = None
        if e8:
            self.k_scale, self.v_scale = (torch.randint(118, 123, shape[:3], generator=g, dtype=torch.uint8).to(device)
                                          .view(torch.float8_e8m0fnu) for _ in range(2))

    @property
    def cache(self):
        return (self.k, self.v) if self.k_scale is None else (self.k, self.v, self.k_scale, self.v_scale)

    def rows(self, name, b, n):
        """Rows 0 .. n-1 of sequence b in 64 bits, [Hkv, n, D]."""
        pool, scale = getattr(self, name), getattr(self, name + "_scale")
        at = self.pages[b, : -(-n // self.page)].long()
        if scale is None:
            x = pool[at].double()
        else:
            x = pool.view(torch.uint8)[at].view(torch.float8_e4m3fn).double()
            bits = scale.view(torch.uint8)[at].double()
            x = x * torch.where(bits == 255, torch.nan, two(bits - 127))[..., None]
        return x.transpose(0, 1).flatten(1, 2)[:, :n]


def attention(paged, q, lengths, gamma, cos, sin, scale=None, keys=None):
    """(out, bound) of decode_attention in 64 bits, [B, Hq, 1, D].

    Roundings of a kernel: q' to the products' type (f16 with an 8-bit cache), each probability to that type, the output to
    q's type; the rest in 32 bits.  A score off by d_j moves the output by sum p_j d_j (v_j - out) to first order, at most
    e^(2 max d) times that; a probability off by u p_j moves it by u p_j v_j."""
    b, hq, _, d = q.shape
    out = torch.zeros(b, hq, 1, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    e8 = paged.k_scale is not None
    u_out, u = U[q.dtype], 2.0 ** -11 if e8 else U[q.dtype]
    scale = d ** -0.5 if scale is None else scale
    for i, n in enumerate(lengths):
        if n <= 0:
            continue
        k, v = keys(i, n) if keys else (paged.rows("k", i, n), paged.rows("v", i, n))
        g = hq // k.shape[0]
        k, v = k.repeat_interleave(g, 0), v.repeat_interleave(g, 0)
        t = (None, None) if cos is None else (cos[n - 1], sin[n - 1])
        qn, q_off = transform(q[i, :, 0], gamma, *t)
        s = torch.einsum("hd,hnd->hn", qn, k) * scale
        p = torch.softmax(s, -1)
        o = torch.einsum("hn,hnd->hd", p, v)
        # q's rounding (relative, and the step of the smallest numbers against the row's largest), 32-bit products and sums
        off = torch.einsum("hd,hnd->hn", qn.abs() * (u + 2.0 ** -18) + q_off + 2.0 ** -24 * qn.abs().amax(-1, keepdim=True),
                           k.abs()) * scale + s.abs() * 2.0 ** -20
        grow = torch.exp(2 * off.amax(-1, keepdim=True))
        spread = torch.einsum("hn,hnd->hd", p * off, (v - o[:, None]).abs())
        # (f16 probabilities: below 2^-14 of the largest a step of 2^-24 of it)
        tiny = 2.0 ** -25 if u == 2.0 ** -11 else 0.0
        p_off = p * (u + 2.0 ** -18) + tiny * p.amax(-1, keepdim=True)
        if tiny and e8:  # the step is that of the largest product of probability and value row
            rows = v.abs().amax(-1)
            p_off = p * (u + 2.0 ** -18) + tiny * 2 * (p * rows).amax(-1, keepdim=True) / rows.clamp_min(1e-30)
        e = spread * grow + torch.einsum("hn,hnd->hd", p_off, v.abs()) * grow
        out[i, :, 0], bound[i, :, 0] = o, e + (o.abs() + e) * u_out + 1e-7 * u_out
    return out, bound + (2.0 ** -24 if q.dtype == torch.float16 else 0.0)
