"""How exact attention over a paged cache is. Sums of products are 32-bit ones, whatever the keys have in common, and probabilities carry more bits than the outputs do."""
import pytest
import torch

from muillm_amd import paged_ops

from .paged_util import DEV, Cache, make_table, offsets_of
from .test_paged_gpu import ATTEND, gpu

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def definition(cache, q, table, lengths, new, scale, rounding):
    """(out, bound) fp64 [rows, heads, dim]. rounding: a probability's, relative to it.

    A score is a sum of dim products that are exact, in 32 bits and any order: dim 2^-24 of the sum of their sizes; its unit, the product with it and the exponential: 8 more of 2^-24 of the
    score's size, and of 1 for the exponential itself. It counts twice, in the probability and in their sum. Below 2^-28 of the largest (fp16's smallest normal number beside 2^14) a
    probability's bits go. Values' sums: the products of 64 keys and the tiles, 2^-24 each of the sizes' sum, which grows no longer than there are keys."""
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    group, row = q.shape[1] // cache.kv_heads, 0
    for b, n in enumerate(new):
        k, v = (cache.values(i, table[b, :-(-lengths[b] // cache.page)].long(), lengths[b]).repeat_interleave(group, 0) for i in (0, 1))
        x = q[row:row + n].double().transpose(0, 1)
        s = x @ k.transpose(1, 2) * scale
        size = x.abs() @ k.abs().transpose(1, 2) * scale
        hidden = torch.arange(lengths[b]) > torch.arange(lengths[b] - n, lengths[b])[:, None]
        w = torch.softmax(s.masked_fill(hidden, -torch.inf), -1)
        d = 2.0 ** -24 * (cache.dim * size.masked_fill(hidden, 0.0).amax(-1, keepdim=True) + 8 * s.masked_fill(hidden, 0.0).abs().amax(-1, keepdim=True) + 8)
        off = (rounding + 2 * d) * w + 2.0 ** -28 * w.amax(-1, keepdim=True) * ~hidden + 2.0 ** -24 * min(lengths[b], 64 + lengths[b] // 64) * w
        out[row:row + n], bound[row:row + n] = ((y @ z).transpose(0, 1) for y, z in ((w, v), (off, v.abs())))
        row += n
    return out, bound


def hold(dtype, dim, page, lengths, new, common, rounding, seed=0, change=None, **kw):
    """common: what a channel that all keys have alike adds to every score."""
    kv_heads, heads, scale = 2, 8, dim ** -0.5
    cache = Cache(2 + sum(-(-n // page) for n in lengths), kv_heads, page, dim, seed)
    cache.scales[0][:] = 2.0 ** -6
    table = make_table(lengths, page, cache.n_pages, seed)
    q = (1.5 * torch.randn((sum(new), heads, dim), generator=torch.Generator().manual_seed(seed + 1)))
    if common:
        cache.codes[0][..., 5] = 448.0
        q[..., 5] = common / (7.0 * scale)
    q = q.to(dtype)
    if change:
        change(cache, table)
    want, bound = definition(cache, q, table, lengths, new, scale, rounding)
    t, ln, off = gpu(table, torch.tensor(lengths), offsets_of(new) if max(new) > 1 else None)
    got = paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), t, ln, off, **kw).cpu().double()
    allowed = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + torch.finfo(F16).tiny * torch.finfo(dtype).eps / 2
    worst = float(((got - want).abs() / allowed).max())
    print(f"{worst:.3f} of the bound")
    assert worst <= 1.0


@pytest.mark.parametrize("common", [0.0, 60.0, 300.0])
@pytest.mark.parametrize("dtype,dim,page", ATTEND)
@pytest.mark.parametrize("lengths", [[2, 5, 60, 64, 130, 700], [3000, 8, 1900]], ids=str)
def test_single_tokens(dtype, dim, page, lengths, common):
    """Probabilities go into the products in two fp16 pieces."""
    hold(dtype, dim, page, lengths, [1] * len(lengths), common, 2.0 ** -22)


@pytest.mark.parametrize("common", [0.0, 60.0, 300.0])
@pytest.mark.parametrize("dtype,dim,page", ATTEND)
@pytest.mark.parametrize("lengths,new", [([300, 180], [300, 150]), ([2600, 90], [60, 90])], ids=str)
def test_prompts(dtype, dim, page, lengths, new, common):
    """Probabilities go into the products in fp16: of bf16 queries in one piece, of fp16 ones in two."""
    hold(dtype, dim, page, lengths, new, common, 2.0 ** -11 if dtype is BF16 else 2.0 ** -22)


@pytest.mark.parametrize("apart", [30, 60, 80])
@pytest.mark.parametrize("dtype,dim,page", [(F16, 128, 64), (BF16, 128, 64), (BF16, 256, 64)])
@pytest.mark.parametrize("lengths,new", [([500], [1]), ([500], [300]), ([2600], [60])], ids=str)
def test_quiet_pages_beside_loud_ones(lengths, new, dtype, dim, page, apart):
    """A page's scale stays where a token that has been taken back has left it: values of the others keep all their bits."""
    def change(cache, table):
        for i in (0, 2, 3, 5):
            cache.scales[1][int(table[0, i])] = 2.0 ** (apart - 8)
            cache.codes[1][int(table[0, i])] = 0.0
        for i in (1, 4, 6, 7):
            cache.scales[1][int(table[0, i])] = 2.0 ** -8
    hold(dtype, dim, page, lengths, new, 0.0, 2.0 ** -11 if dtype is BF16 and new[0] > 1 else 2.0 ** -22, change=change)


@pytest.mark.parametrize("dtype,dim,page", [(F16, 128, 64), (BF16, 128, 64), (BF16, 64, 64), (F16, 256, 64)])
@pytest.mark.parametrize("lengths,new", [([300, 90], [1, 1]), ([300, 90], [150, 90]), ([2600, 90], [1, 1])], ids=str)
@pytest.mark.parametrize("power", [-126, -125, -124, -123, -121, 100, 112])
def test_value_scales_at_the_ends(power, lengths, new, dtype, dim, page):
    """Any power of two is a scale: fp16 outputs of the smallest are zeros, bf16 ones the same bits as at 1, but for the power."""
    cache = Cache(2 + sum(-(-n // page) for n in lengths), 2, page, dim, 7)
    table = make_table(lengths, page, cache.n_pages, 7)
    q = torch.randn((sum(new), 4, dim), generator=torch.Generator().manual_seed(3)).to(dtype)
    t, ln, off = gpu(table, torch.tensor(lengths), offsets_of(new))
    outs = []
    for e in (0, power):
        cache.scales[1][:] = 2.0 ** e
        outs.append(paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), t, ln, off, max_tokens=max(new)).cpu())
    if dtype is F16:
        assert bool((outs[1] == 0).all()) if power < 0 else bool(outs[1].isinf().any())
    else:
        want = (outs[0].double() * 2.0 ** power).to(dtype)
        normal = outs[0].double().abs() * 2.0 ** power >= 2.0 ** -126
        assert float(normal.float().mean()) > 0.5 and torch.equal(outs[1][normal], want[normal])
        assert bool((outs[1].double()[~normal].abs() <= 2.0 ** -126).all())


@pytest.mark.parametrize("dim,page", [(64, 64), (128, 64), (256, 128)])
@pytest.mark.parametrize("lengths,new", [([1, 70, 700], [1, 1, 1]), ([40, 70, 300], [40, 30, 300]), ([2600, 3], [1, 1])], ids=str)
@pytest.mark.parametrize("size", [-1e29, -1e31, -1e35, 1e35])
def test_scores_at_the_ends_of_32_bits(dim, page, lengths, new, size):
    """All of a token's scores are the same large number: its keys weigh the same."""
    cache = Cache(2 + sum(-(-n // page) for n in lengths), 1, page, dim, 8)
    cache.codes[0][:] = 0.0
    cache.codes[0][..., 3] = 256.0
    cache.scales[0][:] = 2.0 ** 40
    table = make_table(lengths, page, cache.n_pages, 8)
    q = torch.zeros((sum(new), 2, dim))
    q[..., 3] = size / 2.0 ** 48
    q = q.to(BF16)
    t, ln, off = gpu(table, torch.tensor(lengths), offsets_of(new) if max(new) > 1 else None)
    got = paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), t, ln, off, scale=1.0).cpu().double()
    even = cache.clone()
    even.codes[0][:] = 0.0
    want, bound = definition(even, torch.zeros_like(q), table, lengths, new, 1.0, 2.0 ** -11)
    allowed = bound + torch.finfo(BF16).eps / 2 * (want.abs() + bound)
    assert bool(((got - want).abs() <= allowed).all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lengths,new", [([128], [1]), ([2624], [1]), ([128], [64]), ([2624], [64])], ids=str)
def test_very_large_scores_of_pages_of_different_scales(dim, lengths, new):
    """2^111 beside 2^110: the larger one has all the weight, whatever the pages' scales are."""
    cache = Cache(lengths[0] // 64 + 2, 1, 64, dim, 9)
    cache.codes[0][:] = 0.0
    table = make_table(lengths, 64, cache.n_pages, 9)
    first, second = int(table[0, 0]), int(table[0, 1])
    cache.scales[0][:] = 2.0 ** 46
    cache.scales[0][first], cache.codes[0][first, :, 7, 3] = 2.0 ** 50, 2.0
    cache.codes[0][second, :, 5, 3] = 16.0
    q = torch.zeros((sum(new), 2, dim))
    q[..., 3] = 2.0 ** 60
    t, ln, off = gpu(table, torch.tensor(lengths), offsets_of(new) if max(new) > 1 else None)
    got = paged_ops.paged_attention(q.to(BF16).to(DEV), cache.to_gpu(), t, ln, off, scale=1.0).cpu().double()
    want = cache.values(1, table[0].long(), lengths[0])[0, 7]
    assert bool(((got - want).abs() <= torch.finfo(BF16).eps / 2 * want.abs() * (1 + 2.0 ** -10)).all())
