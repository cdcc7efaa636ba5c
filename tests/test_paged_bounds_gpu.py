"""What a call's bounds leave out is the rows beyond them, and nothing of the requests that keep to them."""
import pytest
import torch

from muillm_amd import paged_ops

from .paged_util import DEV, Cache, attention, check, make_table, offsets_of
from .test_paged_gpu import gpu

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

BEYOND = [  # requests' lengths and new tokens, max_tokens, heads, KV heads
    ([100 + 7 * i for i in range(40)], [8] * 17 + [64] + [8] * 22, 8, 32, 8),                  # short caches, a workgroup a unit
    ([90 + i for i in range(100)], [8] * 99 + [90], 8, 16, 4),
    ([100 + 7 * i for i in range(40)], [30] * 17 + [90] + [30] * 22, 30, 16, 4),               # prompts, a block of columns each
    ([90 + i for i in range(100)], [20] * 99 + [90], 20, 8, 2),                                # more requests than a wave has lanes
    ([9000, 9100, 12800], [32, 100, 32], 32, 8, 2),                                            # keys divided and joined
    ([9000, 9100, 12800], [4, 40, 4], 4, 8, 2),                                                # dealt out and joined
    ([100, 200, 150], [2, 30, 2], 2, 8, 2),                                                    # a workgroup a unit
]


@pytest.mark.parametrize("dtype,dim", [(F16, 128), (BF16, 64), (BF16, 256)])
@pytest.mark.parametrize("lengths,new,most,heads,kv_heads", BEYOND, ids=range(len(BEYOND)))
def test_a_request_beyond_the_bound_on_new_tokens(dtype, dim, lengths, new, most, heads, kv_heads):
    """Its first tokens and everybody else's have their results, each row behind those its result or what stood there."""
    cache = Cache(2 + sum(-(-n // 64) for n in lengths), kv_heads, 64, dim, 1)
    table = make_table(lengths, 64, cache.n_pages, 1)
    q = torch.randn((sum(new), heads, dim), generator=torch.Generator().manual_seed(2)).to(dtype)
    t, ln, off = gpu(table, torch.tensor(lengths), offsets_of(new))
    out = torch.full(q.shape, 7.0, dtype=dtype, device=DEV)
    junk = torch.full((1 << 24,), float("nan"), device=DEV)  # (what a workspace may hold)
    del junk
    paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), t, ln, off, max_tokens=most, out=out)
    torch.cuda.synchronize()
    want, bound = attention(cache, q, table, lengths, new, dim ** -0.5)
    out = out.cpu()
    inside = torch.cat([torch.arange(n) < most for n in new])
    left = ~inside & (out == 7.0).flatten(1).all(1)
    check(out[~left], want[~left], bound[~left], f"{int(inside.sum())} rows within the bound, {int((~inside & ~left).sum())} beyond")
