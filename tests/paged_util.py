"""A paged e4m3 cache on the CPU and the definitions of what works on it, in 64 bits."""
import math

import torch

from muillm_amd import paged_ops

DEV = "cuda"


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """fp64: the nearest e4m3 number (ties to the even code; |x| <= 464), NaN for infinities and NaN."""
    a = x.double().abs().clamp(min=2.0 ** -6, max=2.0 ** 9)
    unit = torch.exp2(torch.floor(torch.log2(a)) - 3)
    return torch.where(torch.isfinite(x), torch.round(x.double() / unit) * unit, float("nan"))


def exponent(most: float) -> int:
    """Smallest e >= -120 with most <= 448 * 2^e."""
    e = -120
    while most > 448.0 * 2.0 ** e:
        e += 1
    return e


class Cache:
    """Dense twin of a PagedKV: codes fp64 [pages, kv_heads, page, dim], scales fp64 [pages, kv_heads], for keys and values."""

    def __init__(self, n_pages, kv_heads, page, dim, seed=0, filled=True):
        self.page, self.dim, self.kv_heads, self.n_pages = page, dim, kv_heads, n_pages
        g = torch.Generator().manual_seed(seed)
        shape = (n_pages, kv_heads, page, dim)
        self.codes = [e4m3(60.0 * torch.randn(shape, generator=g).clamp(-5, 5)) if filled else torch.zeros(shape, dtype=torch.float64) for _ in range(2)]
        self.scales = [torch.exp2(torch.randint(-9, -4, shape[:2], generator=g).double()) for _ in range(2)]

    def clone(self):
        c = object.__new__(Cache)
        c.__dict__.update(self.__dict__)
        c.codes, c.scales = [x.clone() for x in self.codes], [x.clone() for x in self.scales]
        return c

    def to_gpu(self) -> paged_ops.PagedKV:
        n, h, p, d = self.codes[0].shape
        k, v = (x.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8) for x in self.codes)
        k = k.reshape(n, h, p // 64, 64, d // 64, 64).transpose(3, 4).contiguous()
        v = v.reshape(n, h, p // 64, 4, 4, 4, d).permute(0, 1, 2, 6, 4, 3, 5).contiguous()
        return paged_ops.PagedKV(k.view(torch.float8_e4m3fn).to(DEV), v.view(torch.float8_e4m3fn).to(DEV), *(s.float().to(DEV) for s in self.scales))

    def values(self, which, pages, tokens):
        """fp64 [kv_heads, tokens, dim]."""
        x = self.codes[which][pages] * self.scales[which][pages][..., None, None]
        return x.transpose(0, 1).reshape(self.kv_heads, -1, self.dim)[:, :tokens]

    def same_as(self, kv: paged_ops.PagedKV):
        n, h, p, d = self.codes[0].shape
        k = kv.k.cpu().view(torch.uint8).transpose(3, 4).reshape(n, h, p, d).view(torch.float8_e4m3fn).double()
        v = kv.v.cpu().view(torch.uint8).permute(0, 1, 2, 5, 4, 6, 3).reshape(n, h, p, d).view(torch.float8_e4m3fn).double()
        for name, got, want in (("keys", k, self.codes[0]), ("values", v, self.codes[1]), ("key scales", kv.k_scale.cpu().double(), self.scales[0]),
                                ("value scales", kv.v_scale.cpu().double(), self.scales[1])):
            bad = (got != want) & ~(got.isnan() & want.isnan())
            yield name, bad, got, want


def make_table(lengths, page, n_pages, seed=0, width=None):
    """int32 [requests, width]; the places behind a request's pages hold -7."""
    need = [-(-max(0, n) // page) for n in lengths]
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed))
    assert sum(need) <= n_pages
    t = torch.full((len(lengths), width or max(1, max(need))), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n].int()
        at += n
    return t


def offsets_of(new):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist())


def turn(x, pos, inv_freq, interleaved, factor):
    """fp64 [rows, heads, dim]."""
    x = x.double().clone()
    if inv_freq is None:
        return x
    n = inv_freq.numel()
    c, s = (factor * f(pos.double()[:, None, None] * inv_freq.double()) for f in (torch.cos, torch.sin))
    a, b = (x[..., 0:2 * n:2].clone(), x[..., 1:2 * n:2].clone()) if interleaved else (x[..., :n].clone(), x[..., n:2 * n].clone())
    p, q = a * c - b * s, b * c + a * s
    if interleaved:
        x[..., 0:2 * n:2], x[..., 1:2 * n:2] = p, q
    else:
        x[..., :n], x[..., n:2 * n] = p, q
    return x


def append(cache: Cache, which, x, table, lengths, new):
    """x fp64 [rows, kv_heads, dim] into the cache, token for token."""
    row = 0
    for b, n in enumerate(new):
        start = lengths[b] - n
        touched = {}
        for j in range(n):
            at = start + j
            if at >= 0 and at // cache.page < table.shape[1] and 0 <= int(table[b, at // cache.page]) < cache.n_pages:
                touched.setdefault(at // cache.page, []).append(j)
        for slot, js in touched.items():
            page = int(table[b, slot])
            first = start + js[0] - slot * cache.page
            for h in range(cache.kv_heads):
                y = x[row + js[0]:row + js[-1] + 1, h]
                e = exponent(float(torch.where(torch.isfinite(y), y.abs(), 0.0).max()))
                if first > 0:
                    before = round(math.log2(float(cache.scales[which][page, h])))
                    if e > before:
                        cache.codes[which][page, h, :first] = e4m3(cache.codes[which][page, h, :first] * 2.0 ** (before - e))
                    e = max(e, before)
                cache.scales[which][page, h] = 2.0 ** e
                cache.codes[which][page, h, first:first + len(js)] = e4m3(y * 2.0 ** -e)
        row += n


def attention(cache: Cache, q, table, lengths, new, scale, window=0, keep=0):
    """(out, bound) fp64 [rows, heads, dim]: the definition, and how far a kernel may be from it before it rounds its result.

    A probability goes to the value products in two e4m3 pieces: 2^-4 * 2^-4 of it, and not less than 2^-10 where the largest of its 64 keys is 2^7 or more (2^-17 of that).
    A score's products are exact and added in 32 bits, three times as many as dimensions: 3 dim 2^-24 of the sum of their sizes (nats, so relative to the
    probability), twice that with the sum of the probabilities; four more roundings of 2^-24 at the score itself and at the exponential."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // cache.kv_heads
    row = 0
    for b, n in enumerate(new):
        length = max(0, min(lengths[b], table.shape[1] * cache.page))
        pages = table[b, :-(-length // cache.page)].long()
        real = (pages >= 0) & (pages < cache.n_pages)
        kk, vv = (cache.values(i, pages.clamp(0, cache.n_pages - 1), length) for i in (0, 1))
        have = real.repeat_interleave(cache.page)[:length]
        for j in range(n):
            p = lengths[b] - n + j
            key = torch.arange(length)
            seen = have & (key <= p)
            if window:
                seen &= (key > p - window) | (key < keep)
            if bool(seen.any()):
                at = seen.nonzero()[:, 0]
                for h in range(q.shape[1]):
                    k, v = kk[h // group][at], vv[h // group][at]
                    x = q[row, h].double()
                    s = (k @ x) * scale
                    w = torch.softmax(s, 0)
                    out[row, h] = w @ v
                    d = float(((k.abs() @ x.abs()) * scale).max() * 3 * cache.dim + 8 * s.abs().max() + 8) * 2.0 ** -24
                    tile = torch.zeros(length // 64 + 1, dtype=torch.float64).index_reduce_(0, at // 64, w, "amax")
                    bound[row, h] = ((2.0 ** -8 + 2 * d) * w + 2.0 ** -17 * tile[at // 64]) @ v.abs()
            row += 1
    return out, bound


def check(got, want, bound, what):
    """got (16 bits): within `bound` of want, and half a step of its own type."""
    half = torch.finfo(got.dtype).eps / 2
    got = got.cpu().double()
    assert got.isfinite().all(), f"{what}: not finite"
    allowed = bound + half * (want.abs() + bound) + torch.finfo(torch.float16).tiny * half
    worst = float(((got - want).abs() / allowed.clamp(min=1e-300)).max()) if got.numel() else 0.0
    print(f"{what}: {worst:.3f} of the bound")
    assert worst <= 1.0, f"{what}: {worst} times the bound"
