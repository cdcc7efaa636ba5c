"""The codes that an append writes, each for itself: a turned key may be the neighbouring code only where its value lies on the border between the two; everything else is equal."""
import pytest
import torch

from muillm_amd import paged_ops

from .paged_util import DEV, Cache, append, make_table, offsets_of, turn
from .test_paged_gpu import ONE, PROMPTS, frequencies, gpu

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

FORMS = [(F16, 128, 64, 128, False), (BF16, 128, 128, 64, True), (BF16, 64, 256, 64, False), (F16, 256, 64, 64, False), (BF16, 256, 256, 256, True), (F16, 64, 64, 0, False),
         (F16, 128, 256, 16, True)]


def places(cache, table, lengths, new):
    """(row, page, place in it) of each token of the call."""
    row = 0
    for n, count, pages in zip(lengths, new, table.tolist()):
        for at in range(n - count, n):
            yield row, pages[at // cache.page], at % cache.page
            row += 1


def hold(dtype, dim, page, rot, interleaved, lengths, new, factor=1.25, kv_heads=2, seed=0, positions=None):
    cache = Cache(3 + sum(-(-n // page) for n in lengths), kv_heads, page, dim, seed)
    table = make_table(lengths, page, cache.n_pages, seed)
    g = torch.Generator().manual_seed(seed + 1)
    k, v = (torch.randn((sum(new), kv_heads, dim), generator=g).to(dtype) for _ in range(2))
    freq, kv = frequencies(rot), cache.to_gpu()
    t, ln, off, fr, ps = gpu(table, torch.tensor(lengths), offsets_of(new) if max(new) > 1 else None, freq, positions)
    paged_ops.paged_append(None, k.to(DEV), v.to(DEV), kv, t, ln, off, inv_freq=fr, positions=ps, interleaved=interleaved, rope_scale=factor)
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lengths, new)]) if positions is None else positions
    want, turned = cache.clone(), turn(k.double(), pos, freq, interleaved, factor)
    append(want, 0, turned, table, lengths, new)
    append(want, 1, v.double(), table, lengths, new)
    # Two products and their sum, each rounded to 32 bits, and a cosine and a sine off by 2^-23 each, times the factor: 6 * 2^-24 of the pair's sizes. 0 where nothing turns.
    size = torch.zeros_like(turned)
    if rot:
        a = k.double().abs()
        pairs = a[..., :rot].unflatten(-1, (-1, 2)).sum(-1) if interleaved else a[..., :rot // 2] + a[..., rot // 2:rot]
        size[..., :rot] = pairs.repeat_interleave(2, -1) if interleaved else pairs.repeat(1, 1, 2)
    value, error = (torch.full(want.codes[0].shape, x, dtype=torch.float64) for x in (float("nan"), 0.0))
    for row, p, at in places(cache, table, lengths, new):
        value[p, :, at] = turned[row] / want.scales[0][p][:, None]
        error[p, :, at] = 6 * 2.0 ** -24 * factor * size[row] / want.scales[0][p][:, None]
    wrong = 0
    for name, bad, got, ref in want.same_as(kv):
        if name == "keys":
            border = (value - (got + ref) / 2).abs() <= error  # (false where nothing was turned, or appended at all)
            step = torch.exp2(torch.floor(torch.log2(torch.maximum(got.abs(), ref.abs()).clamp(min=2.0 ** -6))) - 3)
            wrong = int(bad.sum())
            bad = bad & ~(border & (error > 0) & ((got - ref).abs() <= step))
        assert not bool(bad.any()), f"{name}: {int(bad.sum())} differ"
    # (a code's step is 2^-3 to 2^-4 of its value: an error of 2^-20 crosses a border once in some ten thousand values)
    assert wrong <= 1 + sum(new) * kv_heads * rot // 1000


@pytest.mark.parametrize("lengths", ONE, ids=str)
@pytest.mark.parametrize("dtype,dim,page,rot,interleaved", FORMS)
def test_one_token_each(lengths, dtype, dim, page, rot, interleaved):
    hold(dtype, dim, page, rot, interleaved, lengths, [1] * len(lengths))


@pytest.mark.parametrize("lengths,new", PROMPTS, ids=str)
@pytest.mark.parametrize("dtype,dim,page,rot,interleaved", FORMS)
def test_several_tokens_each(lengths, new, dtype, dim, page, rot, interleaved):
    hold(dtype, dim, page, rot, interleaved, lengths, new)


@pytest.mark.parametrize("new", [[1] * 6, [6]], ids=str)
def test_far_positions(new):
    # (an angle's two products in 64 bits are off by 2^-52 of it: 2^-26 at the last of these)
    positions = torch.tensor([0, 1 << 20, 3, (1 << 24) + 1, 131071, (1 << 26) - 1])
    hold(F16, 128, 64, 128, False, [9] * 6 if len(new) == 6 else [9], new, positions=positions)
