"""A cache held in 4 bits and the attention over it, written out plainly in 64 bits for the tests."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # a rounding is off by at most this, relative to the value
DTYPES = [torch.bfloat16, torch.float16]


def quantise(x, dtype):
    """x float32 [..., D] -> (codes int64 [..., D], step, middle of the 16-bit type [..., D / 64]) by the definition, a float32 operation at a time."""
    g = x.unflatten(-1, (-1, 64))
    lo, hi = g.min(-1).values, g.max(-1).values
    f = torch.tensor(1 / 15, dtype=torch.float32, device=x.device)
    step = (hi * f - lo * f).to(dtype)
    mid = (lo + 8 * step.float()).to(dtype)
    bad = ~torch.isfinite(g).all(-1)
    step[bad], mid[bad] = math.nan, math.nan
    codes = torch.clamp(torch.round((g - mid.float()[..., None]) / step.float()[..., None]) + 8, 0, 15)
    codes[(step == 0) | bad] = 8
    return codes.flatten(-2).long(), step, mid


def values(codes, step, mid):
    """float64 [..., D]."""
    return (mid.double()[..., None] + step.double()[..., None] * (codes.unflatten(-1, (-1, 64)) - 8)).flatten(-2)


def block_bytes(k, v, dtype):
    """Blocks [..., 18 * D] uint8 from (codes [..., 16, D], step, mid [..., 16, D / 64]) of keys and of values."""
    parts = []
    for codes, _, _ in (k, v):
        c = codes.to(torch.uint8)
        parts.append((c[..., ::2] + 16 * c[..., 1::2]).flatten(-2))
    for _, step, mid in (k, v):
        parts.append(torch.stack([step, mid], -1).contiguous().view(torch.uint8).flatten(-3))
    return torch.cat(parts, -1)


class Cache:
    """Random keys and values of some requests in packed pages, in a scattered order, with bytes of 0xff (NaN pairs) wherever no position lies."""

    def __init__(self, lengths, Hkv, D, page, dtype, seed, spread=1.0, offset=1.0, spare=3, width=None, fill=255, size=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n_pages = [-(-n // page) for n in lengths]
        total = sum(n_pages) + spare
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
        self.width = width or max(max(n_pages), 1)
        table = torch.full((len(lengths), self.width), -1, dtype=torch.int32)
        self.plane = torch.full((total, Hkv, page // 16, 18 * D), fill, dtype=torch.uint8, device="cuda")
        self.keys, self.vals, self.mids = [], [], []
        for r, (n, m) in enumerate(zip(lengths, n_pages)):
            mine, order = order[:m], order[m:]
            table[r, :m] = torch.tensor(mine, dtype=torch.int32)
            kv = spread * torch.randn(2, Hkv, m * page, D, device="cuda", generator=g)
            kv = kv + offset * torch.randn(2, Hkv, 1, D, device="cuda", generator=g)
            if size is not None and m:                      # a factor per position
                kv = kv * size(m * page)[:, None]
            c, s, z = quantise(kv, dtype)
            vals = values(c, s, z)
            self.keys.append(vals[0, :, :n]); self.vals.append(vals[1, :, :n])
            self.mids.append(z[1].double().repeat_interleave(64, -1)[:, :n])
            s[:, :, n:], z[:, :, n:] = math.nan, math.nan           # what lies behind the request's end
            cut = lambda t: t.unflatten(1, (m, page // 16, 16)).transpose(0, 1)
            if m:
                self.plane[mine] = block_bytes(*[[cut(t[i]) for t in (c, s, z)] for i in (0, 1)], dtype)
        self.table = table.cuda()
        self.page, self.Hkv, self.D, self.dtype = page, Hkv, D, dtype


def attention(q, keys, vals, mids, pos0, scale, window, dtype, unpacked=False):
    """(out, bound) float64 [n, Hq, D] of q [n, Hq, D] at positions pos0 .. over keys, vals [Hkv, L, D].  bound: how far a kernel may be off.
    The roundings to 16 bits, half a step each: the result; a key's weight times its step (the part of a value beside its middle)
    and the weight itself (the middle), or, where the pages are unpacked first, every key element, every value element and
    the weight.  A key rounded so shifts a score by at most half a step of scale * sum |q||k|, all weights by twice that.  float32 sums
    of a row and D products add 2^-20 of the same sums."""
    n, Hq, D = q.shape
    Hkv, L = keys.shape[:2]
    h = HALF_STEP[dtype]
    G = Hq // Hkv
    qg = q.double().view(n, Hkv, G, D)
    s = torch.einsum("nhgd,hld->hgnl", qg, keys) * scale
    at = pos0 + torch.arange(n, device=q.device)[:, None]
    key = torch.arange(L, device=q.device)[None]
    seen = key <= at
    if window:
        seen = seen & (key > at - window)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    out = torch.einsum("hgnl,hld->nhgd", p, vals)
    size = torch.einsum("nhgd,hld->hgnl", qg.abs(), keys.abs()).masked_fill(~seen, 0) * abs(scale)
    if unpacked:
        weight = p * (2 * h + 2 * (size * (h + 2.0 ** -20)).amax(-1, keepdim=True) + 2.0 ** -20)
        off = torch.einsum("hgnl,hld->nhgd", weight, vals.abs())
    else:
        mids = mids if mids is not None else torch.zeros_like(vals)
        part = (vals - mids).abs() + mids.abs()
        weight = p * (h + 2 * (size * 2.0 ** -20).amax(-1, keepdim=True) + 2.0 ** -20)
        off = torch.einsum("hgnl,hld->nhgd", weight, part)
    bound = off + h * (out.abs() + off) + 1e-7
    return out.reshape(n, Hq, D), bound.reshape(n, Hq, D)


class Step:
    """A step over a `Cache` whose last tokens of each request are the step's own."""

    def __init__(self, cache, new, Hq, seed, window=0, extra_columns=0):
        from ferrum_b200.cache.storage import LayerCache
        from ferrum_b200.engine.batch import StepContext, StepEntry
        from ferrum_b200.parts.attention import PagedAttention
        self.cache, self.new, self.Hq, self.window = cache, list(new), Hq, window
        self.past = [k.shape[1] - n for k, n in zip(cache.keys, self.new)]
        T, R = sum(self.new), len(self.new)
        D, Hkv = cache.D, cache.Hkv
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.qkv = torch.randn(T, (Hq + 2 * Hkv) * D + extra_columns, device="cuda", generator=g).to(cache.dtype)
        self.mixer = PagedAttention(Hq * D, Hq, Hkv, D, None, cache.dtype, window=window)
        self.mixer.set_cache_bits(4)
        self.ctx = StepContext("cuda", T, R, [cache.width])
        self.ctx.fill([StepEntry(r, p, [0] * n) for r, (p, n) in enumerate(zip(self.past, self.new))], [cache.table.tolist()])
        self.view = LayerCache(group=0, plane=cache.plane, page_stride=cache.plane.stride(0), page_size=cache.page, writes=True, state=None)

    def attend(self, fill=float("nan")):
        out = torch.full((self.qkv.shape[0], self.Hq * self.cache.D), fill, dtype=self.cache.dtype, device="cuda")
        self.mixer.attend(self.qkv, out, self.ctx, self.view)
        return out

    def check(self, out, what=""):
        row, D = 0, self.cache.D
        for r, (p, n) in enumerate(zip(self.past, self.new)):
            if n == 0:
                continue
            q = self.qkv[row:row + n, :self.Hq * D].view(n, self.Hq, D)
            few = n * (self.Hq // self.cache.Hkv) <= 16
            want, bound = attention(q, self.cache.keys[r], self.cache.vals[r], self.cache.mids[r], p, self.mixer.scale, self.window,
                                    self.cache.dtype, unpacked=not few)
            got = out[row:row + n].view(n, self.Hq, D).double()
            assert torch.isfinite(got).all(), f"{what} request {r}: not finite"
            over = ((got - want).abs() / bound).max().item()
            assert over <= 1, f"{what} request {r} ({p} + {n}): {over:.2f} of the bound"
            row += n
