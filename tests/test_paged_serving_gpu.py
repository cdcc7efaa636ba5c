"""The paged cache's operators and the sampling as a server uses them: one after another, captured and replayed, on other streams; and the ends of their ranges."""
import pytest
import torch

from muillm_amd import muillm_ext, paged_ops

from .paged_util import DEV, Cache, append, attention, check, make_table, offsets_of, turn
from .test_paged_gpu import ATTEND, frequencies, gpu, run_attention, same_cache
from .test_sample_filtered_gpu import pick, run

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


class Server:
    """Token ids to queries, keys and values by tables; a request's logits are its attention's numbers in another order."""

    HEADS, KV, DIM, PAGE, VOCAB = 4, 2, 64, 64, 256

    def __init__(self, dtype, n_pages, seed=0):
        g = torch.Generator().manual_seed(seed)
        width = (self.HEADS + 2 * self.KV) * self.DIM
        self.embedding = (2.0 * torch.randn((self.VOCAB, width), generator=g)).to(dtype)
        self.order = torch.randperm(self.VOCAB, generator=g)
        self.freq = frequencies(self.DIM)
        self.dev = [x.to(DEV) for x in (self.embedding, self.order, self.freq)]
        self.kv = paged_ops.PagedKV.empty(n_pages, self.KV, self.PAGE, self.DIM, DEV)

    def parts(self, x):
        return (y.unflatten(1, (-1, self.DIM)) for y in x.split([self.HEADS * self.DIM, self.KV * self.DIM, self.KV * self.DIM], 1))

    def attend(self, ids, table, lengths, offsets=None, **kw):
        q, k, v = self.parts(self.dev[0].index_select(0, ids))
        q = paged_ops.paged_append(q, k, v, self.kv, table, lengths, offsets, inv_freq=self.dev[2], **kw)
        return q, paged_ops.paged_attention(q, self.kv, table, lengths, offsets, **kw)

    def sample(self, out, last, u):
        logits = out.flatten(1).index_select(0, last).index_select(1, self.dev[1]) * 4
        return logits, muillm_ext.mui_sample_filtered(logits, u, temperature=0.8, top_k=100, top_p=0.9, min_p=0.01)[0]


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompts_then_single_tokens(dtype):
    """Each stage against its definition on what the stage before it gave; the cache's codes are followed from the first token on."""
    prompts, steps = [70, 3, 129, 1], 4
    server = Server(dtype, 14)
    want = Cache(14, server.KV, server.PAGE, server.DIM, filled=False)
    want.scales = [torch.ones_like(s) for s in want.scales]
    table = make_table([n + steps for n in prompts], server.PAGE, 14, 1)
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, server.VOCAB, (sum(prompts),), generator=g).to(DEV)
    lengths, new = list(prompts), list(prompts)
    for step in range(steps):
        off = offsets_of(new)
        u = torch.rand(len(prompts), generator=g)
        t, ln = gpu(table, torch.tensor(lengths))
        q, out = server.attend(ids, t, ln, off.to(DEV) if step == 0 else None)
        last = off[1:] - 1
        logits, token = server.sample(out, last.to(DEV), u.to(DEV))
        torch.cuda.synchronize()
        at = torch.cat([torch.arange(n - m, n) for n, m in zip(lengths, new)])
        cq, ck, cv = server.parts(server.embedding[ids.cpu()].double())
        append(want, 0, turn(ck, at, server.freq, False, 1.0), table, lengths, new)
        append(want, 1, cv, table, lengths, new)
        same_cache(server.kv, want, True)
        # (a key on a border may have the neighbouring code: the attention is held against the codes that are there)
        for name, bad, got, _ in list(want.same_as(server.kv))[:1]:
            want.codes[0] = torch.where(bad, got, want.codes[0])
        ref, bound = attention(want, q.cpu(), table, lengths, new, server.DIM ** -0.5)
        check(out, ref, bound, f"step {step}")
        for b in range(len(prompts)):
            assert int(token[b]) == pick(logits[b].cpu(), float(u[b]), torch.tensor(0.8).item(), 100, torch.tensor(0.9).item(), torch.tensor(0.01).item())[0]
        ids, new = token, [1] * len(prompts)
        lengths = [n + 1 for n in lengths]


def test_captured_steps_follow_the_eager_ones():
    """Two graphs of the same server, replayed in turn with eager work between, against a server that runs eagerly: the same bits at every step. Lengths of 1 to 1300 keys."""
    steps, starts = 6, [1300, 1, 64, 700]
    prompts = torch.randint(0, Server.VOCAB, (sum(starts),), generator=torch.Generator().manual_seed(1)).to(DEV)
    table = make_table([n + steps + 2 for n in starts], Server.PAGE, 40, 1).to(DEV)
    numbers = torch.rand((steps, len(starts)), generator=torch.Generator().manual_seed(3)).to(DEV)
    rows = torch.arange(len(starts), device=DEV)

    def start():
        s = Server(BF16, 40)
        s.attend(prompts, table, torch.tensor(starts, device=DEV), offsets_of(starts).to(DEV))
        return s, torch.tensor(starts, device=DEV), torch.arange(len(starts), device=DEV), torch.zeros((1,), dtype=torch.int64, device=DEV)

    def one(s, lengths, ids, at):
        lengths.add_(1)
        _, out = s.attend(ids, table, lengths)
        _, token = s.sample(out, rows, numbers.index_select(0, at)[0])
        ids.copy_(token)
        at.add_(1)
        return out

    eager = start()
    want = [(one(*eager).clone(), eager[2].clone()) for _ in range(steps)]
    server = start()
    saved = [x.clone() for x in (*(getattr(server[0].kv, n).view(torch.uint8) if n in "kv" else getattr(server[0].kv, n) for n in ("k", "v", "k_scale", "v_scale")), *server[1:])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(*server)  # (warm)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = one(*server)
        graphs.append((g, out))
    kv = server[0].kv
    for dst, src in zip((kv.k.view(torch.uint8), kv.v.view(torch.uint8), kv.k_scale, kv.v_scale, *server[1:]), saved):
        dst.copy_(src)
    for i in range(steps):
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i][0]) and torch.equal(server[2], want[i][1]), f"step {i}"
        one(*start())  # eager work between the replays
    assert all(torch.equal(getattr(kv, n).view(torch.uint8), getattr(eager[0].kv, n).view(torch.uint8)) for n in ("k", "v"))


def test_two_streams_at_once():
    """Calls in flight together have nothing in common but the library."""
    def make(seed):
        s = Server(F16, 90, seed)
        lengths = torch.tensor([2000, 1500], device=DEV)
        t = make_table([2000, 1500], s.PAGE, 90, seed).to(DEV)
        g = torch.Generator().manual_seed(seed)
        ids = torch.randint(0, s.VOCAB, (3500,), generator=g).to(DEV)
        return s, ids, t, lengths, offsets_of([2000, 1500]).to(DEV), torch.tensor([1999, 3499], device=DEV), torch.rand(2, generator=g).to(DEV)

    def work(s, ids, t, lengths, off, last, u):
        _, out = s.attend(ids, t, lengths, off)
        _, token = s.sample(out, last, u)
        _, single = s.attend(token, t, lengths)
        return out, token, single

    want = [work(*make(seed)) for seed in (1, 2)]
    made = [make(seed) for seed in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = []
    for s, m in zip(streams, made):
        with torch.cuda.stream(s):
            got.append(work(*m))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_drafted_tokens_taken_back():
    """Five tokens are appended, three of them taken back by the lengths alone, and others appended in their place: a page's scale stays where the discarded ones left it."""
    cache = Cache(6, 2, 64, 128, 3)
    table = make_table([70, 133], 64, 6, 0)
    g = torch.Generator().manual_seed(1)
    kv, want = cache.to_gpu(), cache.clone()
    for lengths, new, loud in (([66, 132], [5, 5], 40.0), ([65, 130], [2, 1], 1.0), ([66, 131], [1, 1], 3.0)):
        x = (loud * torch.randn((sum(new), 2, 128), generator=g)).to(BF16)
        off = None if new == [1, 1] else offsets_of(new)
        t, ln, off, dev = gpu(table, torch.tensor(lengths), off, x)
        paged_ops.paged_append(None, dev, dev, kv, t, ln, off)
        append(want, 0, x.double(), table, lengths, new)
        append(want, 1, x.double(), table, lengths, new)
        same_cache(kv, want, False)


def test_queries_turned_in_place():
    for new in ([1, 1, 1], [40, 3, 90]):
        lengths = [50, 60, 90]
        g = torch.Generator().manual_seed(1)
        q, x = (torch.randn((sum(new), h, 128), generator=g).to(F16).to(DEV) for h in (9, 2))
        t, ln, off, fr = gpu(make_table(lengths, 64, 6, 0), torch.tensor(lengths), None if max(new) == 1 else offsets_of(new), frequencies(128))
        kv = Cache(6, 2, 64, 128, 3).to_gpu()
        want = paged_ops.paged_append(q, x, x, kv, t, ln, off, inv_freq=fr)
        assert paged_ops.paged_append(q, x, x, kv, t, ln, off, inv_freq=fr, out=q) is q
        assert torch.equal(q, want)


# --------------------------------------------------------------------------------------------------------------------- the ends of the ranges
@pytest.mark.parametrize("dtype,dim,page", ATTEND)
def test_queries_and_keys_of_zeros(dtype, dim, page):
    """Padding: a page of zeros has the smallest scale there is. Every key that is seen weighs the same."""
    for lengths, new in (([70, 5, 1500], [1, 1, 1]), ([70, 5, 200], [40, 5, 130])):
        cache = Cache(2 + sum(-(-n // page) for n in lengths), 1, page, dim, 1)
        cache.codes[0][:] = 0.0
        cache.scales[0][:] = 2.0 ** -120
        run_attention(dtype, dim, page, lengths, new, 4, 1, cache=cache, loud=0.0)
        run_attention(dtype, dim, page, lengths, new, 4, 1, cache=cache, loud=1.0, window=20, keep=3)


def far_scores(dtype, dim, page, loud, seed):
    """Queries and keys so large that a 32-bit score has no places left behind the point: one key holds all the weight."""
    lengths = [300, 90, 1400]
    for new in ([1, 1, 1], [64, 90, 70]):
        cache = Cache(2 + sum(-(-n // page) for n in lengths), 1, page, dim, seed)
        cache.scales[0][:] = 2.0 ** -6 * loud
        table = make_table(lengths, page, cache.n_pages, seed)
        q = (torch.randn((sum(new), 2, dim), generator=torch.Generator().manual_seed(seed)) * 40 * loud).to(dtype)
        off = offsets_of(new) if max(new) > 1 else None
        t, ln, off = gpu(table, torch.tensor(lengths), off)
        got = paged_ops.paged_attention(q.to(DEV), cache.to_gpu(), t, ln, off, scale=1.0).cpu().double()
        assert bool(got.isfinite().all())
        row = decided = 0
        for b, n in enumerate(new):
            k, v = (cache.values(i, table[b, :-(-lengths[b] // page)].long(), lengths[b])[0] for i in (0, 1))
            for j in range(n):
                p = lengths[b] - n + j
                for h in range(2):
                    s = k[:p + 1] @ q[row, h].double()
                    best, at = s.topk(min(2, p + 1))
                    size = float((k[:p + 1].abs() @ q[row, h].double().abs()).max())
                    if p and float(best[0] - best[1]) < 8 * dim * 2.0 ** -24 * size + 60:
                        continue  # (within the roundings of two 32-bit sums of 3 dim products and of what they are multiplied by, or worth a probability)
                    decided += 1
                    w = v[at[0]]
                    assert bool(((got[row, h] - w).abs() <= w.abs() * (2.0 ** -8 + torch.finfo(dtype).eps / 2)).all()), f"row {row}, head {h}"
                row += 1
        assert decided > row  # of two heads each


@pytest.mark.parametrize("loud", [2.0 ** 5, 2.0 ** 8])
@pytest.mark.parametrize("dtype,dim,page", ATTEND)
def test_far_scores(dtype, dim, page, loud):
    far_scores(dtype, dim, page, loud, 3)


@pytest.mark.parametrize("loud", [2.0 ** 20, 2.0 ** 40])
@pytest.mark.parametrize("dim,page", [(64, 64), (128, 64), (256, 128)])
def test_very_far_scores(dim, page, loud):
    far_scores(BF16, dim, page, loud, 4)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_and_small_values(dim):
    """Powers of two go through to the last bit."""
    for lengths, new in (([300, 90], [1, 1]), ([300, 90], [100, 90]), ([1400, 90], [1, 1])):
        cache = Cache(26, 2, 64, dim, 5)
        table = make_table(lengths, 64, 26, 0)
        q = torch.randn((sum(new), 4, dim), generator=torch.Generator().manual_seed(1)).to(BF16)
        args = gpu(table, torch.tensor(lengths), offsets_of(new))
        outs = []
        for e in (0, 85, -80):
            scaled = cache.clone()
            scaled.scales[1] *= 2.0 ** e
            outs.append(paged_ops.paged_attention(q.to(DEV), scaled.to_gpu(), *args, max_tokens=max(new)).cpu().double() * 2.0 ** -e)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_pages_of_very_different_scales():
    """fp16's values are held relative to the loudest page so far: one 2^20 times as loud as those before it, and behind it."""
    for order in ([-22, -22, -2, -22, -22], [-2, -22, -22, -22, -2], [-22, -18, -14, -10, -6]):
        for lengths, new in (([300], [1]), ([300], [200])):
            cache = Cache(5, 1, 64, 128, 6)
            table = torch.arange(5, dtype=torch.int32)[None]
            cache.scales[1][:, 0] = torch.exp2(torch.tensor(order).double())
            for dtype in (F16, BF16):
                run_attention(dtype, 128, 64, lengths, new, 4, 1, cache=cache, table=table)


def test_more_requests_than_are_dealt_out():
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 40, (1100,), generator=g).tolist()
    lengths[0], lengths[700], lengths[1099] = 1500, 200, 1100
    run_attention(BF16, 64, 64, lengths, [1] * 1100, 2, 1)


@pytest.mark.parametrize("n", [1023, 1024])
def test_as_many_requests_as_are_dealt_out(n):
    lengths = [1 + (7 * i) % 30 for i in range(n)]
    lengths[5], lengths[n - 1] = 1500, 1300
    run_attention(F16, 64, 64, lengths, [1] * n, 2, 1)


@pytest.mark.parametrize("dtype,dim,page", ATTEND)
def test_long_caches_of_several_and_no_tokens(dtype, dim, page):
    lengths, new = [2500, 40, 0, 1300, 1100, 3], [3, 0, 0, 7, 1, 2]
    run_attention(dtype, dim, page, lengths, new, 10, 2, max_tokens=7)
    run_attention(dtype, dim, page, lengths, new, 10, 2, max_tokens=7, max_length=2500, window=1200, keep=70)


@pytest.mark.parametrize("dtype,dim,page", ATTEND)
def test_prompts_behind_long_caches(dtype, dim, page):
    """Few blocks of columns and many keys: the keys are divided and joined."""
    run_attention(dtype, dim, page, [2700, 1, 600], [30, 1, 4], 8, 2)
    run_attention(dtype, dim, page, [2700, 1, 600], [30, 1, 4], 8, 2, window=900, keep=65)


def test_bounds_far_above_what_there_is():
    for lengths, new in (([200, 90], [1, 1]), ([200, 90], [30, 90])):
        for kw in (dict(max_tokens=0x7fffffff), dict(max_length=0x7fffffff), dict(max_tokens=1 << 40, max_length=1 << 40), dict(window=1 << 40, keep=1 << 33)):
            run_attention(F16, 128, 64, lengths, new, 4, 2, **kw)


def test_caches_of_more_than_32_bits():
    """Pages whose bytes begin behind 2^31 and 2^32 hold the same as the first ones do."""
    page, heads, dim = 256, 8, 128
    n = (1 << 32) // (page * heads * dim) + 8
    kv, small = paged_ops.PagedKV.empty(n, heads, page, dim, DEV), paged_ops.PagedKV.empty(8, heads, page, dim, DEV)
    near = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    far = torch.tensor([[n - 1, n // 2 + 1, n - 3], [n // 2 + 3, n - 2, 5]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    for lengths, new in (([700, 520], [700, 520]), ([701, 521], [1, 1]), ([731, 524], [30, 3])):
        x = torch.randn((sum(new), heads, dim), generator=g).to(BF16).to(DEV)
        off = None if max(new) == 1 else offsets_of(new)
        ln, off = gpu(torch.tensor(lengths), off)
        outs = []
        for c, t in ((small, near), (kv, far)):
            q = paged_ops.paged_append(x, x, -x, c, t.to(DEV), ln, off)
            outs.append(paged_ops.paged_attention(q, c, t.to(DEV), ln, off))
        assert torch.equal(*outs)
        for a, b in zip(near.flatten().tolist(), far.flatten().tolist()):
            assert torch.equal(small.k[a].view(torch.uint8), kv.k[b].view(torch.uint8)) and torch.equal(small.v[a].view(torch.uint8), kv.v[b].view(torch.uint8))


def test_refusals_of_tensors():
    kv = paged_ops.PagedKV.empty(4, 2, 64, 128, DEV)
    x = torch.zeros((2, 2, 128), dtype=F16, device=DEV)
    t, ln = torch.zeros((2, 2), dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int64, device=DEV)
    freq = torch.ones(64, dtype=torch.float64, device=DEV)
    good = dict(q=x, k=x, v=x, table=t, lengths=ln, offsets=None, inv_freq=freq)
    for change in (dict(k=x.float()), dict(v=x.to(BF16)), dict(q=x.to(BF16)), dict(k=x[:, :1]), dict(k=x[:, :, :64]), dict(v=x[:1]), dict(k=x.transpose(1, 2)), dict(table=t.long()),
                   dict(table=t.t()[:, :1]), dict(lengths=ln.int()), dict(lengths=ln[:1]), dict(offsets=ln), dict(inv_freq=freq.float()), dict(inv_freq=freq[:63]),
                   dict(inv_freq=torch.ones(72, dtype=torch.float64, device=DEV)), dict(positions=ln.int()), dict(positions=ln[:1]), dict(max_tokens=0), dict(lengths=ln.cpu()),
                   dict(table=t.cpu()), dict(q=x.cpu()), dict(out=x[:1]), dict(out=x.float()),
                   dict(k=torch.zeros(2 * 2 * 132, dtype=F16, device=DEV).view(2, 2, 132)[..., 4:]), dict(k=torch.zeros((2, 2, 130), dtype=F16, device=DEV)[..., :128])):
        with pytest.raises(RuntimeError):
            paged_ops.paged_append(kv=kv, **{**good, **change})
    wide = torch.zeros((3, 2, 128), dtype=F16, device=DEV)
    good = dict(q=x, table=t, lengths=ln, offsets=None)
    for change in (dict(q=x[:, :1]), dict(q=x.float()), dict(q=wide), dict(scale=0.0), dict(scale=-1.0), dict(window=-1), dict(keep_first=-1), dict(max_tokens=-3), dict(out=x),
                   dict(q=wide[:2], out=wide[1:]), dict(q=wide[1:], out=wide[:2]), dict(out=x.to(BF16)), dict(q=x[:, :, :64])):
        with pytest.raises(RuntimeError):
            paged_ops.paged_attention(kv=kv, **{**good, **change})
    with pytest.raises(RuntimeError):
        paged_ops.paged_append(wide[:2], x, x, kv, t, ln, out=wide[1:])
    assert paged_ops.paged_attention(wide[:2], kv, t, ln, out=wide[:2].clone()).shape == (2, 2, 128)


def test_no_rows():
    kv = paged_ops.PagedKV.empty(4, 2, 64, 128, DEV)
    x = torch.zeros((0, 2, 128), dtype=F16, device=DEV)
    t, ln = torch.zeros((2, 2), dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int64, device=DEV)
    off = torch.zeros(3, dtype=torch.int64, device=DEV)
    assert paged_ops.paged_append(x, x, x, kv, t, ln, off).shape == paged_ops.paged_attention(x, kv, t, ln, off).shape == (0, 2, 128)
    assert paged_ops.paged_append(None, x, x, kv, t, ln, off) is None


def test_sampling_refusals_and_rows_that_share():
    logits, u = torch.randn((3, 50), generator=torch.Generator().manual_seed(1)).to(F16), torch.tensor([0.1, 0.5, 0.9])
    dev, number = logits.to(DEV), u.to(DEV)
    for kw in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=-0.5), dict(min_p=-0.1), dict(min_p=1.5), dict(temperature=float("nan")), dict(top_p=float("nan"))):
        with pytest.raises(ValueError):
            muillm_ext.mui_sample_filtered(dev, number, **kw)
    for kw in (dict(temperature=number.double()), dict(top_k=number), dict(top_p=number[:2]), dict(min_p=u)):
        with pytest.raises(RuntimeError):
            muillm_ext.mui_sample_filtered(dev, number, **kw)
    for bad in (u, number[:2], number.double(), 0.5):
        with pytest.raises(RuntimeError):
            muillm_ext.mui_sample_filtered(dev, bad)
    with pytest.raises(ValueError):
        muillm_ext.mui_sample_filtered(dev.float(), number)
    run(logits, u, k=1 << 40)
    run(logits, u, k=(1 << 32) + 1)
    one = dev[:1].expand(3, -1)
    token, _ = muillm_ext.mui_sample_filtered(one, number)
    assert token.tolist() == [pick(logits[0], float(x), 1.0, 0, 1.0, 0.0)[0] for x in u]
    turned = dev.t().contiguous().t()
    assert torch.equal(muillm_ext.mui_sample_filtered(turned, number)[0], muillm_ext.mui_sample_filtered(dev, number)[0])


@pytest.mark.parametrize("dtype,dim,page", [(F16, 128, 64), (BF16, 64, 128), (BF16, 256, 64)])
def test_prompts_of_many_requests(dtype, dim, page):
    """More than one wave's lanes of requests, some without tokens, some behind cached ones: every block is found once."""
    g = torch.Generator().manual_seed(3)
    new = torch.randint(0, 12, (150,), generator=g).tolist()
    new[7], new[63], new[64], new[149] = 90, 70, 0, 65
    lengths = [n + int(torch.randint(0, 50, (1,), generator=g)) for n in new]
    lengths[10] += 700
    run_attention(dtype, dim, page, lengths, new, 7, 1)
    run_attention(dtype, dim, page, lengths, new, 8, 2, max_tokens=90)
    run_attention(dtype, dim, page, lengths[:3] + [2000], [0, 0, 1, 300], 8, 1)


@pytest.mark.parametrize("dtype,dim,page", [(F16, 128, 64), (BF16, 64, 128), (BF16, 256, 64)])
@pytest.mark.parametrize("requests,length,tokens", [(1, 300, 300), (1, 900, 33), (1, 2100, 17), (3, 1100, 9), (20, 130, 9), (2, 3000, 40)])
def test_between_single_tokens_and_prompts(dtype, dim, page, requests, length, tokens):
    """Either kernel, with and without a workgroup per block, around the sizes at which the other is taken."""
    lengths = [max(tokens, length - 37 * b) for b in range(requests)]
    run_attention(dtype, dim, page, lengths, [max(1, tokens - b) for b in range(requests)], 4, 2)
    run_attention(dtype, dim, page, lengths, [tokens] + [0] * (requests - 1), 6, 1, window=100, keep=3)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [9, 40, 3, 70]], ids=str)
def test_lengths_that_are_none(new):
    """Fewer tokens than are new, lengths beyond the table and any number that 64 bits hold: no token at a place that is none, and the requests beside them as ever."""
    for window, keep in ((0, 0), (50, 5)):
        for dtype, dim, page in ATTEND:
            cache = Cache(9, 2, page, dim, 3)
            table = torch.tensor([[0, 1], [2, 3], [4, 5], [6, 7]], dtype=torch.int32)
            if max(new) > 1:
                run_attention(dtype, dim, page, [5, 100, 1, 90], new, 4, 2, window, keep, table=table, cache=cache)
            good = [90, 100, 80, 128]
            want = None
            for bad in (90, 1 << 62, -(1 << 63), (1 << 63) - 1, -7, 1 << 36, 1 << 32):
                lengths = [good[0], bad, good[2], good[3]]
                q = torch.randn((sum(new), 4, dim), generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
                x = q[:, :2].contiguous()
                off = None if max(new) == 1 else offsets_of(new).to(DEV)
                kv = cache.to_gpu()
                ln = torch.tensor(lengths).to(DEV)
                paged_ops.paged_append(None, x, x, kv, table.to(DEV), ln, off)
                out = paged_ops.paged_attention(q, kv, table.to(DEV), ln, off, window=window, keep_first=keep).cpu()
                rows = [r for b in (0, 2, 3) for r in range(sum(new[:b]), sum(new[:b + 1]))]
                pages = [0, 1, 4, 5, 6, 7, 8]
                got = (out[rows], kv.k.view(torch.uint8)[pages].cpu(), kv.v.view(torch.uint8)[pages].cpu())
                want = want or got
                assert all(torch.equal(a, b) for a, b in zip(got, want)), bad
                if bad > 1000 or bad < 0:  # nothing of it was written
                    untouched = cache.to_gpu()
                    assert torch.equal(kv.k.view(torch.uint8)[2:4], untouched.k.view(torch.uint8)[2:4])


@pytest.mark.parametrize("dtype,rows,vocab", [(BF16, 3, 70001), (F16, 2, 131072), (BF16, 70, 66000), (F16, 5, 8000)])
def test_captured_sampling_of_one_and_two_launches(dtype, rows, vocab):
    """Replays on other logits and numbers, eager calls between them: each the eager call's tokens and probabilities."""
    g = torch.Generator().manual_seed(2)
    given = [((2 * torch.randn((rows, vocab), generator=g)).to(dtype).to(DEV), torch.rand(rows, generator=g).to(DEV)) for _ in range(4)]
    kw = dict(temperature=0.9, top_k=3000, top_p=0.95, min_p=1e-4)
    want = [muillm_ext.mui_sample_filtered(x, u, **kw) for x, u in given]
    logits, numbers = given[0][0].clone(), given[0][1].clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = muillm_ext.mui_sample_filtered(logits, numbers, **kw)
        graphs.append((graph, out))
    for i in range(8):
        graph, out = graphs[i % 2]
        logits.copy_(given[i % 4][0])
        numbers.copy_(given[i % 4][1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[i % 4][0]) and torch.equal(out[1], want[i % 4][1]), f"replay {i}"
        again = muillm_ext.mui_sample_filtered(given[(i + 1) % 4][0], given[(i + 1) % 4][1], **kw)
        assert torch.equal(again[0], want[(i + 1) % 4][0])


def test_captured_prompts_and_joined_results():
    """Prompts whose keys are divided, and single tokens of long caches, replayed as the device's lengths change."""
    page, heads, kv_heads, dim = 128, 8, 2, 128
    cache = Cache(44, kv_heads, page, dim, 1)
    kv = cache.to_gpu()
    table = make_table([2600, 2700], page, 44, 0).to(DEV)
    g = torch.Generator().manual_seed(1)
    q = torch.randn((48, heads, dim), generator=g).to(BF16).to(DEV)
    off = torch.tensor([0, 40, 48], device=DEV)
    lengths = torch.tensor([2000, 1500], device=DEV)

    def calls():
        return (paged_ops.paged_attention(q, kv, table, lengths, off, max_tokens=40), paged_ops.paged_attention(q[:2], kv, table, lengths))

    calls()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for n in ([2000, 1500], [2600, 8], [41, 2700], [500, 900], [2000, 1500]):
        lengths.copy_(torch.tensor(n))
        graph.replay()
        torch.cuda.synchronize()
        again = calls()
        assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1]), n
        want, bound = attention(cache, q[:2].cpu(), table.cpu(), n, [1, 1], dim ** -0.5)
        check(out[1], want, bound, str(n))


@pytest.mark.parametrize("dtype,dim", [(F16, 128), (BF16, 64)])
def test_longer_prompts_of_many_requests(dtype, dim):
    """More than 64 requests on the kernel for prompts, and more than are dealt out, most of them with one new token."""
    g = torch.Generator().manual_seed(5)
    new = torch.randint(20, 60, (80,), generator=g).tolist()
    new[3], new[63], new[64], new[79] = 0, 1, 120, 0
    lengths = [n + int(torch.randint(0, 300, (1,), generator=g)) for n in new]
    run_attention(dtype, dim, 64, lengths, new, 8, 1)
    new = [1] * 1100
    new[5], new[600], new[700], new[1099] = 40, 0, 33, 17
    lengths = [n + i % 7 for i, n in enumerate(new)]
    run_attention(dtype, dim, 64, lengths, new, 8, 1, max_tokens=40)
