"""Operators of a server of many requests, as cases to be timed: keys and values appended to a paged 8-bit cache with the position
rotation on the way, attention over that cache, and the choice of the next token from given uniform numbers.

The cache. A layer has pages of `page` tokens (a multiple of 64). Keys are e4m3 codes [pages, kv_heads, page / 64, dim / 64, 64, 64], the last two
token and dimension; values are e4m3 codes [pages, kv_heads, page / 64, dim, 4, 4, 4], the last three g, t, i of token 16 t + 4 g + i of its 64.
Each page and head has one scale for keys and one for values, a power of two, fp32 [pages, kv_heads]; a value is code * scale. A request's pages
stand in its row of `table` (int32 [requests, most pages]); `lengths` (int64) counts its tokens, this call's among them, and `offsets` (int64
[requests + 1]) says which of the call's rows are its new ones (None: one row each).

Appending. scale = 2^e, e the smallest integer >= -120 with max |x| <= 448 * 2^e over the page's appended tokens, at least the one that stands there
where the page holds earlier tokens; their codes are then multiplied by the quotient of the two scales and rounded again.

Sampling, per row. w_i = exp((l_i - max l) / T); tokens in order of falling logits, equal ones by rising index; kept are the first top_k, of
those the ones in front of which less than top_p of the top_k's weight lies, of those the ones with w >= min_p; drawn is the first whose
cumulative weight exceeds u times the kept weight. Results: the token, and its share of the kept weight.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
THETA = 500000.0
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attention(name, dtype, requests, cached, spread=1.0, new=1, new_spread=1.0, heads=32, kv_heads=8, dim=128, page=64, window=0, keep=0):
    """cached: most tokens in front of the new ones of a request; the requests' numbers lie between spread * cached and cached (new: the same)."""
    return dict(op="attention", name=name, dtype=dtype, requests=requests, cached=cached, spread=spread, new=new, new_spread=new_spread, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, window=window, keep=keep)


def _append(name, dtype, requests, cached, spread=1.0, new=1, new_spread=1.0, heads=32, kv_heads=8, dim=128, page=64, rot=128, interleaved=False, factor=1.0):
    return dict(op="append", name=name, dtype=dtype, requests=requests, cached=cached, spread=spread, new=new, new_spread=new_spread, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, rot=rot, interleaved=interleaved, factor=factor)


def _sampling(name, dtype, rows, vocab, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False):
    """mixed: the settings differ from row to row, as a batch of several users' requests has them."""
    return dict(op="sampling", name=name, dtype=dtype, rows=rows, vocab=vocab, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, mixed=mixed)


def listed():
    return [
        # one user's step: a token joins a chat of a thousand
        _append("append one token", "float16", 1, 1000),
        # a served batch's step, requests of all lengths
        _append("append 64 requests", "bfloat16", 64, 4000, spread=0.02),
        # prompts of several users in one call, some behind a cached beginning; interleaved pairs, half of the head rotated, long-context factor
        _append("append prompts", "bfloat16", 5, 333, spread=0.01, new=4111, new_spread=0.1, rot=64, interleaved=True, factor=1.2),
        # one user's step, short chat: latency counts
        _attention("attend one short", "float16", 1, 700),
        # a served batch's step
        _attention("attend 32 requests", "bfloat16", 32, 4095, spread=0.05),
        # a large batch of long requests: the cache's bytes count
        _attention("attend 64 long", "bfloat16", 64, 16383, spread=0.25, page=128),
        # long contexts under a sliding window whose first tokens stay visible, smaller heads
        _attention("attend window", "bfloat16", 16, 32001, spread=0.3, heads=64, kv_heads=8, dim=64, window=4096, keep=4),
        # the next portion of a long prompt, behind what is cached of it
        _attention("prompt portion", "bfloat16", 1, 6144, new=2048),
        # prompts of several users in one call
        _attention("prompts ragged", "float16", 6, 0, new=1501, new_spread=0.03),
        # one user's next token
        _sampling("sample one", "bfloat16", 1, 128256, temperature=0.8, top_p=0.95),
        # a served batch of users with settings of their own
        _sampling("sample 64 mixed", "bfloat16", 64, 128256, temperature=0.9, top_k=50, top_p=0.9, min_p=0.05, mixed=True),
        # a large batch without filters
        _sampling("sample 256 plain", "float16", 256, 32000, temperature=1.1),
    ]


def _spread_over(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "sampling"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "sampling":
        vocab = _spread_over(rng, 2000, 200000)
        rows = _spread_over(rng, 1, min(256, 8_000_000 // vocab))
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, temperature=round(rng.uniform(0.5, 1.5), 3), top_k=rng.choice([0, 0, _spread_over(rng, 1, 2000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.999), 3)]), min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), mixed=rng.random() < 0.5)
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    page = rng.choice([64, 128, 256])
    spread, new_spread = round(rng.uniform(0.02, 1.0), 3), round(rng.uniform(0.02, 1.0), 3)
    c = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, page=page, spread=spread, new_spread=new_spread)
    prompts = rng.random() < 0.4
    if op == "append":
        new = _spread_over(rng, 2, 5000) if prompts else 1
        requests = _spread_over(rng, 1, min(64, max(1, 16000 // new)))
        return dict(c, requests=requests, cached=_spread_over(rng, 1, 8000) - 1, new=new, rot=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                    factor=rng.choice([1.0, 1.0, round(rng.uniform(0.8, 1.4), 3)]))
    window = rng.choice([0, 0, _spread_over(rng, 100, 8000)])
    keep = rng.choice([0, _spread_over(rng, 1, 100)]) if window else 0
    if prompts:
        new = _spread_over(rng, 2, 2000)
        cached = _spread_over(rng, 1, 8000) - 1
        requests = _spread_over(rng, 1, max(1, min(16, 200_000_000 // (heads * new * (cached + new)))))
    else:
        new = rng.choice([1, 1, 1, 2, 5])
        cached = _spread_over(rng, 30, 30000)
        requests = _spread_over(rng, 1, max(1, min(64, 500_000_000 // (kv_heads * dim * cached))))
    return dict(c, requests=requests, cached=cached, new=new, window=window, keep=keep)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _numbers(most, spread, count):
    """`count` whole numbers between spread * most and most, the first of them `most`: the same for every seed."""
    return [most] + [int(round(most * spread ** math.modf(i * 0.6180339887498949)[0])) for i in range(1, count)]


def _counts(c):
    cached = _numbers(c["cached"], c["spread"], c["requests"])
    new = [max(1, n) for n in _numbers(c["new"], c["new_spread"], c["requests"])]
    return cached, new


def _power_of_two(e):
    """2^e in 32 bits, e whole."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise_pages(x):
    """Codes and scales [pages, heads] of x [pages, heads, tokens, dim]."""
    m, e = torch.frexp(x.abs().amax((-2, -1)))
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-120)
    s = _power_of_two(e)
    return (x / s[..., None, None]).to(torch.float8_e4m3fn), s


def _to_pages_k(codes):
    n, h, p, d = codes.shape
    return codes.view(torch.uint8).reshape(n, h, p // 64, 64, d // 64, 64).permute(0, 1, 2, 4, 3, 5).contiguous().view(torch.float8_e4m3fn)


def _to_pages_v(codes):
    n, h, p, d = codes.shape
    return codes.view(torch.uint8).reshape(n, h, p // 64, 4, 4, 4, d).permute(0, 1, 2, 6, 4, 3, 5).contiguous().view(torch.float8_e4m3fn)  # t, g, i -> g, t, i


def _from_pages_k(k):
    """uint8 [pages, heads, page, dim]."""
    n, h, tiles, blocks = k.shape[:4]
    return k.view(torch.uint8).permute(0, 1, 2, 4, 3, 5).reshape(n, h, tiles * 64, blocks * 64)


def _from_pages_v(v):
    n, h, tiles, d = v.shape[:4]
    return v.view(torch.uint8).permute(0, 1, 2, 5, 4, 6, 3).reshape(n, h, tiles * 64, d)


def _make_pages(gen, pages, heads, page, dim, to_pages, gain):
    """Keys and values as trained models have them: channels of different sizes, pages of different loudness."""
    codes, scales = [], []
    step = max(1, (1 << 27) // (heads * page * dim))
    for at in range(0, pages, step):
        x = torch.randn((min(step, pages - at), heads, page, dim), generator=gen, device=DEVICE)
        x *= gain * torch.exp(0.3 * torch.randn((x.shape[0], heads, 1, 1), generator=gen, device=DEVICE))
        q, s = _quantise_pages(x)
        codes.append(to_pages(q))
        scales.append(s)
    return torch.cat([c.view(torch.uint8) for c in codes]).view(torch.float8_e4m3fn), torch.cat(scales)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[c["dtype"]]
    if c["op"] == "sampling":
        rows, vocab = c["rows"], c["vocab"]
        x = 2.0 * torch.randn((rows, vocab), generator=gen, device=DEVICE)
        likely = torch.randint(0, vocab, (rows, 40), generator=gen, device=DEVICE)
        x.scatter_reduce_(1, likely, 6.0 + 6.0 * torch.rand((rows, 40), generator=gen, device=DEVICE), "amax")
        s = dict(op=c["op"], logits=x.to(dtype), u=torch.rand((rows,), generator=gen, device=DEVICE))
        near = torch.arange(rows, device=DEVICE) if c["mixed"] else torch.zeros((rows,), dtype=torch.int64, device=DEVICE)
        s["temperature"] = c["temperature"] * (1.0 + 0.05 * (near % 5)).float()
        s["top_k"] = torch.where(near % 4 == 3, 0, c["top_k"] + near % 7 * (c["top_k"] > 0)).to(torch.int32)
        s["top_p"] = torch.where(near % 3 == 2, 1.0, c["top_p"]).float()
        s["min_p"] = torch.where(near % 5 == 4, 0.0, c["min_p"]).float()
        return s
    cached, new = _counts(c)
    lengths = [a + b for a, b in zip(cached, new)]
    page, heads, kv_heads, dim = c["page"], c["heads"], c["kv_heads"], c["dim"]
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.zeros((len(need), max(need)), dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    gain = torch.exp(0.4 * torch.randn((kv_heads, 1, dim), generator=gen, device=DEVICE))
    k, k_scale = _make_pages(gen, pages, kv_heads, page, dim, _to_pages_k, gain)
    v, v_scale = _make_pages(gen, pages, kv_heads, page, dim, _to_pages_v, 1.0)
    s = dict(op=c["op"], k=k, v=v, k_scale=k_scale, v_scale=v_scale, table=table, lengths=torch.tensor(lengths, device=DEVICE),
             most_new=max(new), longest=max(lengths), page=page)
    s["offsets"] = None if max(new) == 1 else torch.tensor([0] + list(np.cumsum(new)), device=DEVICE)
    rows = sum(new)
    if c["op"] == "append":
        # one projection's output, q | k | v, as a decoder layer has it
        proj = torch.randn((rows, (heads + 2 * kv_heads) * dim), generator=gen, device=DEVICE).to(dtype)
        q, nk, nv = proj.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
        s |= dict(q=q.view(rows, heads, dim), nk=nk.view(rows, kv_heads, dim), nv=nv.view(rows, kv_heads, dim))
        s["inv_freq"] = torch.tensor([THETA ** (-2.0 * i / c["rot"]) for i in range(c["rot"] // 2)], dtype=torch.float64, device=DEVICE)
        s |= dict(interleaved=c["interleaved"], factor=c["factor"])
    else:
        s["q"] = (1.5 * torch.randn((rows, heads, dim), generator=gen, device=DEVICE)).to(dtype)
        s |= dict(window=c["window"], keep=c["keep"], scale=dim ** -0.5)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _run_own(s):
    from muillm_amd import muillm_ext, paged_ops

    if s["op"] == "sampling":
        return muillm_ext.mui_sample_filtered(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    kv = paged_ops.PagedKV(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if s["op"] == "append":
        q = paged_ops.paged_append(s["q"], s["nk"], s["nv"], kv, s["table"], s["lengths"], s["offsets"], inv_freq=s["inv_freq"], interleaved=s["interleaved"],
                                   rope_scale=s["factor"], max_tokens=s["most_new"])
        return [q, s["k"], s["v"], s["k_scale"], s["v_scale"]]
    return paged_ops.paged_attention(s["q"], kv, s["table"], s["lengths"], s["offsets"], scale=s["scale"], window=s["window"], keep_first=s["keep"],
                                     max_tokens=s["most_new"], max_length=s["longest"])


def _new_rows(s, rows):
    """(request, position) of each of the call's rows; numbers of new tokens."""
    b = s["table"].shape[0]
    n = torch.arange(rows, device=DEVICE)
    offsets = torch.arange(b + 1, device=DEVICE) if s["offsets"] is None else s["offsets"]
    new = offsets[1:] - offsets[:-1]
    request = torch.searchsorted(offsets[1:].contiguous(), n, right=True)
    return request, s["lengths"][request] - new[request] + n - offsets[request], new


def _rotate(x, pos, s):
    """x [rows, heads, dim] in 32 bits with its first dimensions rotated by the rows' positions; angles in 64 bits."""
    half = s["inv_freq"].numel()
    a = pos.double()[:, None] * s["inv_freq"]
    cos, sin = (s["factor"] * f(a).float()[:, None, :] for f in (torch.cos, torch.sin))
    x = x.float()
    if s["interleaved"]:
        p, q = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((p * cos - q * sin, q * cos + p * sin), -1).flatten(-2)
    else:
        p, q = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((p * cos - q * sin, q * cos + p * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _append_plain(x, codes, scales, from_pages, to_pages, s):
    """x [rows, heads, dim] in 32 bits to its places in codes and scales."""
    page = s["page"]
    request, pos, new = _new_rows(s, x.shape[0])
    first = s["lengths"] - new
    spans = (s["most_new"] + page - 2) // page + 1
    slot = first[:, None] // page + torch.arange(spans, device=DEVICE)          # the pages that a request's new tokens lie in
    real = slot * page < s["lengths"][:, None]
    number = (real.flatten().cumsum(0) - 1).view(real.shape)
    pages = s["table"].gather(1, slot.clamp(max=s["table"].shape[1] - 1)).long()[real]
    old = (first[:, None] - slot * page).clamp(min=0)[real]                     # earlier tokens of each of those pages
    mine = number[request, pos // page - first[request] // page]                # the one that each row lies in
    most = torch.zeros((pages.numel(), x.shape[1]), device=DEVICE).index_reduce_(0, mine, x.abs().amax(-1), "amax")
    m, e = torch.frexp(most)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-120)
    before = torch.frexp(scales[pages])[1] - 1
    e = torch.where(old[:, None] > 0, torch.maximum(e, before), e)
    held = from_pages(codes.view(torch.uint8)[pages])
    moved = (held.view(torch.float8_e4m3fn).float() * _power_of_two((before - e).clamp(min=-126))[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    earlier = torch.arange(page, device=DEVICE) < old[:, None]
    held = torch.where(earlier[:, None, :, None] & (e > before)[..., None, None], moved, held)
    held[mine, :, pos % page] = (x * _power_of_two(-e)[mine][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes.view(torch.uint8)[pages] = to_pages(held.view(torch.float8_e4m3fn)).view(torch.uint8)
    scales[pages] = _power_of_two(e)


def _attend_plain(s):
    q, table, page = s["q"], s["table"], s["page"]
    rows, heads, dim = q.shape
    kv_heads, b = s["k"].shape[1], table.shape[0]
    request, pos, new = _new_rows(s, rows)
    at = pos - (s["lengths"] - new)[request]
    # keys and values of all requests, [requests, kv heads, tokens, dim] in 32 bits
    k, v = ((from_pages(x.view(torch.uint8)[table.flatten()]).view(torch.float8_e4m3fn).float() * scale[table.flatten()][..., None, None])
            .unflatten(0, table.shape).transpose(1, 2).flatten(2, 3)
            for x, scale, from_pages in ((s["k"], s["k_scale"], _from_pages_k), (s["v"], s["v_scale"], _from_pages_v)))
    grid = torch.zeros((b, s["most_new"], heads, dim), device=DEVICE)
    grid[request, at] = q.float()
    grid = grid.unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4)               # [requests, kv heads, group, new, dim]
    score = torch.matmul(grid.flatten(2, 3), k.transpose(-1, -2)).mul_(s["scale"]).unflatten(2, grid.shape[2:4])
    key = torch.arange(k.shape[2], device=DEVICE)
    here = (s["lengths"] - new)[:, None] + torch.arange(s["most_new"], device=DEVICE)
    seen = (key <= here[..., None]) & (key < s["lengths"][:, None, None])
    if s["window"]:
        seen &= (key > here[..., None] - s["window"]) | (key < s["keep"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = score.sub_(torch.where(top.isfinite(), top, 0.0)).exp_()
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.flatten(2, 3), v).unflatten(2, grid.shape[2:4])
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [requests, new, heads, dim]
    return out[request, at].to(q.dtype)


def _sample_plain(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    w = torch.exp((x - x.amax(-1, keepdim=True)) / s["temperature"].double()[:, None])
    order = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True).indices
    w = w.gather(1, order)
    sums = w.cumsum(-1)
    place = torch.arange(vocab, device=DEVICE)
    top_k = s["top_k"].long()[:, None]
    keep = (place < top_k) | (top_k <= 0)
    limit = s["top_p"].double()[:, None] * (w * keep).sum(-1, keepdim=True)
    keep &= ((sums - w) < limit) | (s["top_p"][:, None] >= 1) | (place == 0)
    keep &= (w >= s["min_p"].double()[:, None]) | (place == 0)
    count = keep.long().cumprod(-1).sum(-1, keepdim=True)
    kept = sums.gather(1, count - 1)
    pick = torch.minimum((sums <= s["u"].double()[:, None] * kept).sum(-1, keepdim=True), count - 1)
    return order.gather(1, pick)[:, 0], (w.gather(1, pick) / kept).float()[:, 0]


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "sampling":
        return _sample_plain(s)
    if s["op"] == "attention":
        return _attend_plain(s)
    pos = _new_rows(s, s["q"].shape[0])[1]
    _append_plain(_rotate(s["nk"], pos, s), s["k"], s["k_scale"], _from_pages_k, _to_pages_k, s)
    _append_plain(s["nv"].float(), s["v"], s["v_scale"], _from_pages_v, _to_pages_v, s)
    return [_rotate(s["q"], pos, s).to(s["q"].dtype), s["k"], s["v"], s["k_scale"], s["v_scale"]]


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def _seen(c, first, new):
    """(keys that any of a request's new tokens sees, pairs of a token and a key that it sees)."""
    w, keep = c["window"], c["keep"]
    if not w:
        return first + new, new * first + new * (new + 1) // 2
    low = max(0, first + 1 - w)
    keys = first + new - low + min(low, keep)
    return keys, sum(min(p + 1, w) + max(0, min(p + 1 - w, keep)) for p in range(first, first + new))


def work(case):
    c = case
    if c["op"] == "sampling":
        n = c["rows"] * c["vocab"]
        return {"bytes": 2 * n + 36 * c["rows"], "flops": 4 * n}
    cached, new = _counts(c)
    rows = sum(new)
    if c["op"] == "append":
        wide = (2 * c["heads"] + 2 * c["kv_heads"]) * c["dim"] * 2 + 2 * c["kv_heads"] * c["dim"]
        return {"bytes": rows * wide, "flops": rows * (3 * (c["heads"] + c["kv_heads"]) * c["rot"] + 3 * 2 * c["kv_heads"] * c["dim"])}
    keys, pairs = (sum(x) for x in zip(*(_seen(c, a, b) for a, b in zip(cached, new))))
    return {"bytes": 2 * keys * c["kv_heads"] * c["dim"] + 2 * rows * c["heads"] * c["dim"] * 2, "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _two_to(p):
    """2^p in 64 bits, p whole."""
    return ((p.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(x):
    """The nearest of the numbers +-n * 2^(p - 3), n < 16, p >= -6; ties to even n."""
    power = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    power = torch.where(_two_to(power + 1) <= x.abs(), power + 1, power)
    power = torch.where(_two_to(power) > x.abs(), torch.clamp(power - 1, min=-6.0), power)
    unit = _two_to(power - 3)
    return torch.round(x / unit) * unit


def _token_values(codes, tile_of, token):
    """codes of one token of a page's head, as an index: keys [tile, block, token, dim], values [tile, dim, g, t, i]."""
    tile, at = divmod(token, 64)
    return codes[tile, :, at, :].reshape(-1) if tile_of == "k" else codes[tile, :, at // 4 % 4, at // 16, at % 4]


def _exact_append(c, s):
    starts = [0] + list(np.cumsum(_counts(c)[1]))
    cached, new = _counts(c)
    freq = s["inv_freq"].double()
    half = freq.numel()

    def turned(x, pos):
        y = x.double().clone()
        ca, sa = c["factor"] * torch.cos(pos[:, None, None] * freq), c["factor"] * torch.sin(pos[:, None, None] * freq)
        i = torch.arange(half, device=DEVICE)
        i, j = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
        a, b = x.double()[..., i], x.double()[..., j]
        y[..., i], y[..., j] = a * ca - b * sa, b * ca + a * sa
        return y

    q = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    out = {n: s[n].double() for n in ("k", "v", "k_scale", "v_scale")}
    page = c["page"]
    for b in range(c["requests"]):
        rows = slice(starts[b], starts[b + 1])
        pos = torch.arange(cached[b], cached[b] + new[b], device=DEVICE, dtype=torch.float64)
        q[rows] = turned(s["q"][rows], pos)
        for n, x in (("k", turned(s["nk"][rows], pos)), ("v", s["nv"][rows].double())):
            for slot in range(cached[b] // page, (cached[b] + new[b] - 1) // page + 1):
                p = int(s["table"][b, slot])
                low, high = max(cached[b], slot * page), min(cached[b] + new[b], (slot + 1) * page)
                y = x[low - cached[b]:high - cached[b]]
                e = torch.ceil(torch.log2((y.abs().amax((0, 2)) / 448).clamp(min=2.0 ** -120)))
                e = torch.where(448.0 * _two_to(e - 1) >= y.abs().amax((0, 2)), e - 1, e).clamp(min=-120.0)
                scale = _two_to(e)
                if low > slot * page:
                    scale = torch.maximum(scale, out[n + "_scale"][p])
                    for h in range(c["kv_heads"]):
                        ratio = out[n + "_scale"][p, h] / scale[h]
                        if ratio < 1:
                            for t in range(low - slot * page):
                                moved = _round_e4m3(_token_values(out[n][p, h], n, t) * ratio)
                                _put(out[n][p, h], n, t, moved)
                out[n + "_scale"][p] = scale
                codes = _round_e4m3(y / scale[:, None])
                t = torch.arange(low, high, device=DEVICE) % page
                if n == "k":
                    out[n][p][:, t // 64, :, t % 64, :] = codes.unflatten(2, (-1, 64))
                else:
                    out[n][p][:, t // 64, :, t // 4 % 4, t % 64 // 16, t % 4] = codes
    return [q, out["k"], out["v"], out["k_scale"], out["v_scale"]]


def _put(codes, kind, token, values):
    tile, at = divmod(token, 64)
    if kind == "k":
        codes[tile, :, at, :] = values.view(-1, 64)
    else:
        codes[tile, :, at // 4 % 4, at // 16, at % 4] = values


def _exact_attention(c, s):
    cached, new = _counts(c)
    if sum(a * b + b * b for a, b in zip(cached, new)) * c["heads"] * c["dim"] > 4e11:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    group, at, page, dim = c["heads"] // c["kv_heads"], 0, c["page"], c["dim"]
    token = torch.arange(page, device=DEVICE)
    for b in range(c["requests"]):
        n = cached[b] + new[b]
        pages = s["table"][b, :-(-n // page)].long()
        key = torch.arange(n, device=DEVICE)
        here = torch.arange(cached[b], n, device=DEVICE)[:, None]
        seen = key <= here
        if c["window"]:
            seen = seen & ((here - key < c["window"]) | (key < c["keep"]))
        kd, vd = s["k"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double(), s["v"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
        for h in range(c["kv_heads"]):
            kh = kd[:, h][:, token // 64, :, token % 64, :].permute(1, 0, 2, 3).reshape(pages.numel(), page, dim) * s["k_scale"][pages, h].double()[:, None, None]
            vh = vd[:, h][:, token // 64, :, token // 4 % 4, token % 64 // 16, token % 4].permute(1, 0, 2) * s["v_scale"][pages, h].double()[:, None, None]
            kh, vh = kh.reshape(-1, dim)[:n], vh.reshape(-1, dim)[:n]
            for g in range(h * group, (h + 1) * group):
                x = (s["q"][at:at + new[b], g].double() @ kh.T) * s["scale"]
                w = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
                out[at:at + new[b], g] = w @ vh
        at += new[b]
    return out


def _exact_sampling(s):
    x = s["logits"].double().cpu().numpy()
    u, t, k, p, m = (s[n].double().cpu().numpy() for n in ("u", "temperature", "top_k", "top_p", "min_p"))
    token, share = np.zeros(len(x), np.int64), np.zeros(len(x))
    for r, row in enumerate(x):
        order = np.argsort(-row, kind="stable")
        w = np.exp((row[order] - row[order[0]]) / t[r])
        n = int(k[r]) if 0 < k[r] < len(w) else len(w)
        if p[r] < 1:
            n = min(n, max(1, int(np.searchsorted(np.concatenate(([0.0], np.cumsum(w[:n])[:-1])), p[r] * w[:n].sum()))))
        n = max(1, min(n, int((w >= m[r]).sum())))
        total = np.cumsum(w[:n])
        i = min(int(np.searchsorted(total, u[r] * total[-1], side="right")), n - 1)
        token[r], share[r] = order[i], w[i] / total[-1]
    return token, share


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sampling":
        return _exact_sampling(s)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attention(case, s)
