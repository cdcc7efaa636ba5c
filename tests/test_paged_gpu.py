"""Appending to and attending over a paged e4m3 cache against the definitions in 64 bits."""
import pytest
import torch

from muillm_amd import paged_ops

from .paged_util import DEV, Cache, append, attention, check, make_table, offsets_of, turn

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def frequencies(rot):
    return torch.tensor([10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64) if rot else None


def gpu(*tensors):
    return [None if t is None else t.to(DEV) for t in tensors]


def run_append(dtype, lengths, new, heads, kv_heads, dim, page, rot, interleaved=False, factor=1.0, table=None, cache=None, seed=0, use_offsets=None, positions=None,
               loud=1.0, most=None, with_q=True, values=None):
    n_pages = 3 + sum(-(-max(0, n) // page) for n in lengths)
    cache = cache or Cache(n_pages, kv_heads, page, dim, seed)
    table = make_table(lengths, page, cache.n_pages, seed) if table is None else table
    g = torch.Generator().manual_seed(seed + 1)
    rows = sum(new)
    proj = (torch.randn((rows, (heads + 2 * kv_heads) * dim), generator=g) * loud).to(dtype)
    if values is not None:
        values(proj)
    freq = frequencies(rot)
    offsets = offsets_of(new) if (max(new) != 1 or min(new) != 1 or use_offsets) else None
    dev = proj.to(DEV)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in dev.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    kv = cache.to_gpu()
    t, ln, off, fr, ps = gpu(table, torch.tensor(lengths), offsets, freq, positions)
    out = paged_ops.paged_append(q if with_q else None, k, v, kv, t, ln, off, inv_freq=fr, positions=ps, interleaved=interleaved, rope_scale=factor, max_tokens=most)
    torch.cuda.synchronize()
    want = cache.clone()
    at = torch.cat([torch.arange(n - m, n) for n, m in zip(lengths, new)])
    at = at if positions is None else positions
    cq, ck, cv = (x.unflatten(1, (-1, dim)).double() for x in proj.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    append(want, 0, turn(ck, at, freq, interleaved, factor), table, lengths, new)
    append(want, 1, cv, table, lengths, new)
    return out, turn(cq, at, freq, interleaved, factor), kv, want, torch.cat([ck.abs().flatten(), torch.zeros(1)]).max()


def same_cache(kv, want, turned):
    """Values are exact. Keys are turned in 32 bits before they are rounded: one in a thousand may be the neighbouring code where they lie on a border, and no more than that
    (their distance to it is about 2^-24 * 3 of the pair's size, a code's step 2^-3 of the value and the pair seldom over 2^7 times the value)."""
    for name, bad, got, ref in want.same_as(kv):
        if name != "keys" or not turned:
            assert not bool(bad.any()), f"{name}: {int(bad.sum())} differ"
            continue
        n = int(bad.sum())
        assert n <= 1 + bad.numel() // 1000, f"{name}: {n} differ"
        step = torch.exp2(torch.floor(torch.log2(ref.abs().clamp(min=2.0 ** -6))) - 3)
        assert bool(((got - ref).abs()[bad] <= step[bad]).all()), "keys: more than a step"


def close_queries(out, want, dtype, most):
    # products and their sum in 32 bits, cosine and sine off by two units each: 6 * 2^-24 of the pair; then half a step
    half = torch.finfo(dtype).eps / 2
    err = (out.cpu().double() - want).abs()
    assert bool((err <= half * want.abs() * (1 + 1e-3) + 6 * 2.0 ** -24 * 2 * most + torch.finfo(dtype).tiny * half).all()), float(err.max())


ONE = [[1], [64], [65], [1000], [1, 64, 65, 130, 7], [256, 257, 255]]


@pytest.mark.parametrize("lengths", ONE, ids=str)
@pytest.mark.parametrize("dtype,dim,page,rot,interleaved", [(F16, 128, 64, 128, False), (BF16, 128, 128, 64, True), (BF16, 64, 256, 64, False), (F16, 256, 64, 64, False),
                                                            (BF16, 256, 256, 256, True), (F16, 64, 64, 0, False), (F16, 128, 256, 16, True)])
def test_one_token_each(lengths, dtype, dim, page, rot, interleaved):
    out, want_q, kv, want, _ = run_append(dtype, lengths, [1] * len(lengths), 6, 2, dim, page, rot, interleaved, 1.25)
    same_cache(kv, want, rot > 0)
    close_queries(out, want_q, dtype, 1.25 * 6)


PROMPTS = [([5], [5]), ([64], [64]), ([65], [65]), ([300], [300]), ([130, 3, 77, 200], [66, 3, 1, 200]), ([90, 128, 129], [27, 65, 2]), ([513, 40], [449, 17])]


@pytest.mark.parametrize("lengths,new", PROMPTS, ids=str)
@pytest.mark.parametrize("dtype,dim,page,rot,interleaved", [(F16, 128, 64, 128, False), (BF16, 128, 128, 64, True), (BF16, 64, 256, 64, False), (F16, 256, 64, 64, False),
                                                            (BF16, 256, 256, 256, True), (F16, 64, 64, 0, False), (F16, 128, 256, 32, False)])
def test_several_tokens_each(lengths, new, dtype, dim, page, rot, interleaved):
    out, want_q, kv, want, _ = run_append(dtype, lengths, new, 3, 3, dim, page, rot, interleaved)
    same_cache(kv, want, rot > 0)
    close_queries(out, want_q, dtype, 6)


@pytest.mark.parametrize("loud", [2.0 ** -20, 2.0 ** -4, 1.0, 30.0, 3000.0])
@pytest.mark.parametrize("lengths,new", [([70, 3, 64], [1, 1, 1]), ([100, 70, 190], [30, 5, 100])], ids=str)
def test_scales_rise_and_never_fall_under_earlier_tokens(lengths, new, loud):
    out, want_q, kv, want, _ = run_append(BF16, lengths, new, 2, 2, 128, 64, 0, loud=loud)
    same_cache(kv, want, False)


def test_zeros_infinities_and_nan():
    def values(proj):
        proj[0, 256:] = 0
        proj[1, 300], proj[1, 400], proj[1, 620] = float("inf"), float("nan"), float("-inf")
    for lengths, new in (([65, 66], [1, 1]), ([66], [2]), ([2], [2])):
        out, want_q, kv, want, _ = run_append(F16, lengths, new, 2, 2, 128, 64, 0, values=values)
        same_cache(kv, want, False)


def test_empty_requests_and_rows_behind_the_last():
    lengths, new = [70, 0, 64, 130], [3, 0, 0, 2]
    cache = Cache(8, 2, 64, 128, 3)
    out, want_q, kv, want, _ = run_append(F16, lengths, new, 4, 2, 128, 64, 128, cache=cache)
    same_cache(kv, want, True)
    # two rows more than the requests have: neither the cache nor their queries change
    table, g = make_table(lengths, 64, 8, 0), torch.Generator().manual_seed(5)
    x = torch.randn((7, 2, 128), generator=g).to(F16)
    q = torch.randn((7, 4, 128), generator=g).to(F16)
    before = torch.full((7, 4, 128), 3.0, dtype=F16, device=DEV)
    kv = cache.to_gpu()
    paged_ops.paged_append(q.to(DEV), x.to(DEV), x.to(DEV), kv, table.to(DEV), torch.tensor(lengths).to(DEV), offsets_of(new).to(DEV), max_tokens=4, out=before)
    want = cache.clone()
    append(want, 0, x.double(), table, lengths, new)
    append(want, 1, x.double(), table, lengths, new)
    same_cache(kv, want, False)
    assert torch.equal(before[:5].cpu(), q[:5]) and bool((before[5:] == 3.0).all())


@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1], [2, 3, 1, 5, 2]], ids=str)
def test_places_that_are_none(new):
    """Entries that are no page, lengths beyond the table and below the new tokens: those tokens are left out, the others are there."""
    lengths = [70, 65, 129, 1 if max(new) > 1 else 0, 500]
    cache = Cache(9, 2, 64, 128, 3)
    table = torch.tensor([[0, 1], [2, -1], [3, 4], [5, 6], [7, 8]], dtype=torch.int32)
    table[2, 0] = 1 << 30
    out, want_q, kv, want, _ = run_append(F16, lengths, new, 4, 2, 128, 64, 64, cache=cache, table=table, use_offsets=max(new) > 1)
    same_cache(kv, want, True)
    close_queries(out, want_q, F16, 6)


def test_positions_of_the_callers_and_far_ones():
    positions = torch.tensor([0, 1, 1 << 20, 7, (1 << 24) + 1])
    for new in ([1] * 5, [5]):
        lengths = [9] * 5 if len(new) == 5 else [9]
        out, want_q, kv, want, _ = run_append(F16, lengths, new, 4, 2, 128, 64, 128, positions=positions)
        same_cache(kv, want, True)
        close_queries(out, want_q, F16, 6)


def test_without_queries_and_the_bound_on_new_tokens():
    for lengths, new, most in (([90, 10], [1, 1], None), ([90, 10], [26, 4], 26), ([90, 10], [26, 4], 64), ([300, 10], [300, 4], None)):
        out, _, kv, want, _ = run_append(BF16, lengths, new, 2, 2, 64, 64, 64, with_q=False, most=most)
        assert out is None
        same_cache(kv, want, True)


# ---------------------------------------------------------------------------------------------------------------------
ATTEND = [(F16, 128, 64), (BF16, 128, 128), (F16, 64, 256), (BF16, 64, 64), (F16, 256, 128), (BF16, 256, 64)]


def run_attention(dtype, dim, page, lengths, new, heads, kv_heads, window=0, keep=0, scale=None, table=None, cache=None, seed=0, loud=1.5, **kw):
    n_pages = 2 + sum(-(-max(0, n) // page) for n in lengths)
    cache = cache or Cache(n_pages, kv_heads, page, dim, seed)
    table = make_table(lengths, page, cache.n_pages, seed) if table is None else table
    q = (torch.randn((sum(new), heads, dim), generator=torch.Generator().manual_seed(seed + 9)) * loud).to(dtype)
    offsets = offsets_of(new) if (max(new) != 1 or min(new) != 1) else None
    t, ln, off = gpu(table, torch.tensor(lengths), offsets)
    got = paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), t, ln, off, scale=scale, window=window, keep_first=keep, **kw)
    torch.cuda.synchronize()
    want, bound = attention(cache, q, table, lengths, new, dim ** -0.5 if scale is None else scale, window, keep)
    check(got, want, bound, f"{dtype} {lengths} {new} {heads}/{kv_heads} x {dim}")


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (7, 1), (16, 1), (40, 2), (3, 1)])
@pytest.mark.parametrize("dtype,dim,page", ATTEND)
def test_one_query_each(dtype, dim, page, heads, kv_heads):
    run_attention(dtype, dim, page, [1, 2, 63, 64, 65, 200, 0, 700], [1] * 8, heads, kv_heads)


@pytest.mark.parametrize("dtype,dim,page", ATTEND)
@pytest.mark.parametrize("length", [1500, 5000])
def test_one_query_over_many_keys(dtype, dim, page, length):
    run_attention(dtype, dim, page, [length, 17], [1, 1], 4, 2)


@pytest.mark.parametrize("lengths,new", [([2], [2]), ([70], [5]), ([64, 65], [64, 1]), ([200, 31, 0, 5], [120, 31, 0, 5]), ([300, 129], [4, 129])], ids=str)
@pytest.mark.parametrize("dtype,dim,page", ATTEND)
def test_several_queries_each(dtype, dim, page, lengths, new):
    run_attention(dtype, dim, page, lengths, new, 6, 2)


@pytest.mark.parametrize("window,keep", [(1, 0), (1, 1), (5, 3), (64, 0), (64, 4), (100, 70), (1000, 9), (63, 64), (130, 129)])
@pytest.mark.parametrize("lengths,new", [([1, 70, 300, 128], [1, 1, 1, 1]), ([1, 70, 300, 128], [1, 30, 100, 128])], ids=str)
def test_windows_and_first_tokens(lengths, new, window, keep):
    run_attention(BF16, 128, 64, lengths, new, 4, 2, window, keep)
    run_attention(F16, 64, 128, lengths, new, 4, 1, window, keep)


@pytest.mark.parametrize("loud,scale", [(0.01, None), (20.0, None), (1.0, 1.0), (1.0, 1e-4)])
def test_flat_and_sharp_scores(loud, scale):
    run_attention(F16, 128, 64, [300, 90], [1, 30], 4, 2, loud=loud, scale=scale)
    run_attention(BF16, 64, 64, [300, 90], [1, 30], 4, 2, loud=loud, scale=scale)


def test_a_sink_beside_many_light_keys():
    """The first key holds most of the weight, thousands share the rest: each weighs less than 2^-18 of it, together they are a third."""
    cache = Cache(66, 1, 64, 64, 1)
    cache.scales[0][:] = 2.0 ** -6
    cache.codes[0][:] = 0.0
    lengths = [4160]
    table = make_table(lengths, 64, 66, 0)
    first = int(table[0, 0])
    cache.codes[0][first, 0, 0, 0] = 448.0   # score 448 / 64 * q
    q = torch.zeros((1, 2, 64), dtype=F16)
    q[..., 0] = 13.0
    cache.codes[1][first, 0, 0] = 0.0
    want, bound = attention(cache, q, table, lengths, [1], 0.1)
    assert 0.2 < float(torch.exp(torch.tensor(0.1 * 7 * 13)) / 4160) < 3
    got = paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), table.to(DEV), torch.tensor(lengths).to(DEV), scale=0.1)
    check(got, want, bound, "sink")
    q[..., 0] = 24.0
    want, bound = attention(cache, q, table, lengths, [1], 0.1)
    got = paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), table.to(DEV), torch.tensor(lengths).to(DEV), scale=0.1)
    check(got, want, bound, "far sink")


@pytest.mark.parametrize("new", [[1, 1], [40, 65]], ids=str)
def test_what_is_hidden_does_not_count(new):
    """NaN codes behind the length, in front of the window and, for the earlier of several queries, in later tokens."""
    for dtype, dim, page in ATTEND:
        lengths = [100, 165]
        cache = Cache(7, 2, page, dim, 4)
        table = make_table(lengths, page, 7, 0)
        for b, n in enumerate(lengths):
            for i in (0, 1):
                last = int(table[b, (n - 1) // page])
                cache.codes[i][last, :, (n - 1) % page + 1:] = float("nan")
                cache.codes[i][int(table[b, 0]), :, 3] = float("nan")          # in front of the window
        for i in range(7):
            if i not in table.tolist()[0] + table.tolist()[1]:
                cache.codes[0][i] = cache.codes[1][i] = float("nan")
        q = torch.randn((sum(new), 4, dim), generator=torch.Generator().manual_seed(1)).to(dtype)
        want, bound = attention(cache, q, table, lengths, new, 0.1, 20, 2)
        off = offsets_of(new) if max(new) > 1 else None
        t, ln, off = gpu(table, torch.tensor(lengths), off)
        got = paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), t, ln, off, scale=0.1, window=20, keep_first=2)
        seen = want.isfinite() & bound.isfinite()
        assert bool(seen.any())
        assert bool((got.cpu().isfinite() == want.isfinite()).all())
        check(torch.where(seen, got.cpu(), torch.zeros((), dtype=dtype)), torch.where(seen, want, 0.0), torch.where(seen, bound, 0.0), "hidden NaN")


@pytest.mark.parametrize("dtype,dim,page", ATTEND)
def test_a_nan_that_is_seen_is_a_nan(dtype, dim, page):
    """Of the later queries alone, in its dimension alone (values); everywhere for those that see it (keys)."""
    lengths, new = [100], [60]
    table = make_table(lengths, page, 4, 0)
    q = torch.randn((60, 2, dim), generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    at = 70  # query 30 is the first that sees it
    for which in (0, 1):
        cache = Cache(4, 1, page, dim, 4)
        cache.codes[which][int(table[0, at // page]), 0, at % page, 5] = float("nan")
        got = paged_ops.paged_attention(q, cache.to_gpu(), table.to(DEV), torch.tensor(lengths).to(DEV), offsets_of(new).to(DEV)).cpu()
        nan = got.isnan()
        assert not bool(nan[:30].any())
        if which:
            assert bool(nan[30:, :, 5].all()) and int(nan.sum()) == 30 * 2
        else:
            assert bool(nan[30:].all())


def test_entries_that_are_no_page_do_not_count():
    cache = Cache(6, 1, 64, 128, 2)
    table = torch.tensor([[0, -1, 2], [3, 1 << 30, 5], [-5, -5, -5]], dtype=torch.int32)
    run_attention(F16, 128, 64, [150, 190, 100], [1, 1, 1], 4, 1, table=table, cache=cache)
    run_attention(BF16, 128, 64, [150, 192, 100], [30, 70, 100], 4, 1, table=table, cache=cache)
    run_attention(BF16, 128, 64, [150, 500, 100], [1, 1, 1], 4, 1, table=table, cache=cache)  # a length beyond the table


def test_rows_behind_the_last_request_stay():
    cache = Cache(4, 1, 64, 128, 2)
    lengths, new = [70, 20], [3, 2]
    table = make_table(lengths, 64, 4, 0)
    q = torch.randn((9, 2, 128), generator=torch.Generator().manual_seed(1)).to(F16)
    out = torch.full((9, 2, 128), 5.0, dtype=F16, device=DEV)
    paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), table.to(DEV), torch.tensor(lengths).to(DEV), offsets_of(new).to(DEV), out=out)
    want, bound = attention(cache, q[:5], table, lengths, new, 128 ** -0.5)
    check(out[:5], want, bound, "first rows")
    assert bool((out[5:] == 5.0).all())


def test_strided_queries_and_wide_tables():
    cache = Cache(6, 2, 64, 128, 2)
    lengths = [200, 90]
    table = make_table(lengths, 64, 6, 0, width=40)
    wide = torch.randn((2, 10, 128), generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    q = wide[:, 2:10:2]
    t = torch.full((2, 100), 3, dtype=torch.int32, device=DEV)
    t[:, :40] = table.to(DEV)
    got = paged_ops.paged_attention(q, cache.to_gpu(), t[:, :40], torch.tensor(lengths).to(DEV), max_length=200)
    want, bound = attention(cache, q.cpu(), table, lengths, [1, 1], 128 ** -0.5)
    check(got, want, bound, "strided")
