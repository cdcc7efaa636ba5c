"""Tokens from given random numbers against the definition in 64 bits: whole numbers are equal."""
import math

import pytest
import torch

from muillm_amd import muillm_ext

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


def pick(row, u, t, k, p, m):
    """(token, probability) by the definition, one row in 64 bits."""
    x = [float("-inf") if math.isnan(v) else v + 0.0 for v in row.double().tolist()]
    order = sorted((i for i in range(len(x)) if x[i] > float("-inf")), key=lambda i: (-x[i], i))
    if not order:
        return 0, 0.0
    top = x[order[0]]
    if t <= 0:
        return order[0], 1.0
    w = [1.0 if x[i] == top else 0.0 if top == float("inf") else math.exp((x[i] - top) / t) for i in order]
    n = k if 0 < k < len(w) else len(w)
    if p < 1:
        limit, before, kept = p * math.fsum(w[:n]), 0.0, 0
        while kept < n and before < limit:
            before += w[kept]
            kept += 1
        n = kept
    n = max(1, min(n, sum(v >= m for v in w)))
    total = math.fsum(w[:n])
    run, i = 0.0, 0
    while True:
        run += w[i]
        if run > u * total or i == n - 1:
            return order[i], w[i] / total
        i += 1


def run(logits, u, t=1.0, k=0, p=1.0, m=0.0, stride=None):
    rows = logits.shape[0]
    dev = logits.to(DEV)
    if stride:
        wide = torch.full((rows, stride), 50.0, dtype=logits.dtype, device=DEV)
        wide[:, :logits.shape[1]] = dev
        dev = wide[:, :logits.shape[1]]
    given = [x.to(DEV) if isinstance(x, torch.Tensor) else x for x in (t, k, p, m)]
    token, share = muillm_ext.mui_sample_filtered(dev, u.to(DEV), temperature=given[0], top_k=given[1], top_p=given[2], min_p=given[3])
    torch.cuda.synchronize()
    at = lambda x, r: x[r].item() if isinstance(x, torch.Tensor) else torch.tensor(x, dtype=torch.float32).item() if isinstance(x, float) else x  # noqa: E731
    for r in range(rows):
        want, prob = pick(logits[r], float(u[r]), at(t, r), at(k, r), at(p, r), at(m, r))
        assert int(token[r]) == want, f"row {r}: {int(token[r])}, expected {want}"
        assert abs(float(share[r]) - prob) <= 2.0 ** -24 * prob * 1.001 + 1e-40, f"row {r}: {float(share[r])}, expected {prob}"


def noise(rows, vocab, dtype, seed=0, loud=2.0):
    g = torch.Generator().manual_seed(seed)
    return (loud * torch.randn((rows, vocab), generator=g)).to(dtype), torch.rand(rows, generator=g)


SETTINGS = [dict(), dict(t=0.7), dict(k=1), dict(k=40), dict(p=0.9), dict(m=0.1), dict(t=1.3, k=50, p=0.8, m=0.02), dict(k=5000, p=0.99), dict(t=0.0), dict(p=0.0), dict(m=1.0),
            dict(t=100.0, p=0.5), dict(t=0.01), dict(p=0.9999, m=1e-4)]


@pytest.mark.parametrize("setting", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype,vocab", [(F16, 1), (BF16, 2), (BF16, 500), (F16, 1000), (BF16, 8200), (F16, 32001)])
def test_filters(dtype, vocab, setting):
    logits, u = noise(5, vocab, dtype)
    run(logits, u, **setting)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_settings_of_each_row(dtype):
    logits, u = noise(12, 3001, dtype, 3)
    g = torch.Generator().manual_seed(4)
    t = torch.rand(12, generator=g) * 2
    t[3] = 0.0
    k = torch.randint(0, 60, (12,), generator=g).to(torch.int32)
    k[5], k[6] = 0, -3
    p = torch.rand(12, generator=g)
    p[7], p[8] = 1.0, 2.0
    m = torch.rand(12, generator=g) * 0.2
    run(logits, u, t, k, p, m)
    run(logits, u, t, 7, p, 0.0)
    run(logits, u, 0.9, k, 0.7, m, stride=3011)


@pytest.mark.parametrize("vocab", [65528, 65529, 131100, 200003])
def test_many_values_and_parts(vocab):
    """More tokens than 16 bits count, in one value and in many."""
    logits, u = noise(2, vocab, BF16, 1)
    run(logits, u, p=0.95)
    logits[:] = 1.5
    run(logits, torch.tensor([0.0, 0.999]))
    run(logits, torch.tensor([0.5, 0.25]), p=0.5)
    run(logits, torch.tensor([0.5, 0.999]), k=vocab - 3)


def test_ties_go_to_the_lowest_index():
    for dtype in (F16, BF16):
        logits = torch.zeros((4, 1000), dtype=dtype)
        logits[:, 100:900:7] = 2.0
        logits[1, 500] = -0.0
        run(logits, torch.tensor([0.0, 0.3, 0.7, 0.99]), k=50)
        run(logits, torch.tensor([0.0, 0.3, 0.7, 0.99]), p=0.5)
        run(logits, torch.tensor([0.0, 0.3, 0.9, 0.99]))
        run(logits, torch.tensor([0.0, 0.3, 0.9, 0.99]), t=0.0)
        run(torch.where(torch.arange(1000) % 2 == 0, 0.0, -0.0).to(dtype).expand(4, -1).contiguous(), torch.tensor([0.0, 0.3, 0.9, 0.99]))


def test_infinities_and_nan():
    for dtype in (F16, BF16):
        logits, u = noise(8, 700, dtype, 2)
        inf, nan = float("inf"), float("nan")
        logits[0, ::2] = -inf
        logits[1, 5:] = nan
        logits[2, :] = -inf
        logits[3, :] = nan
        logits[4, 17], logits[4, 400] = inf, inf
        logits[5, 1:] = -inf
        logits[6, ::3] = nan
        logits[6, 1::3] = -inf
        for setting in (dict(), dict(k=3), dict(p=0.6), dict(m=0.05), dict(t=0.0), dict(t=0.3, k=300, p=0.9), dict(t=inf)):
            run(logits, u, **setting)


def test_random_numbers_at_the_ends():
    logits, _ = noise(6, 2000, BF16, 7)
    u = torch.tensor([0.0, 2.0 ** -30, 0.5, 1 - 2.0 ** -24, 1.0, 7.0])
    for setting in (dict(), dict(k=10), dict(p=0.7), dict(m=0.2)):
        run(logits, u, **setting)
    token, _ = muillm_ext.mui_sample_filtered(logits.to(DEV), torch.full((6,), float("nan"), device=DEV))
    assert torch.equal(token.cpu(), logits.float().argmax(-1))


def test_far_apart_logits():
    for dtype in (F16, BF16):
        logits = torch.linspace(-60000.0, 60000.0, 4001).to(dtype).expand(3, -1).contiguous()
        run(logits, torch.tensor([0.0, 0.5, 0.999]), t=1.0)
        run(logits, torch.tensor([0.0, 0.5, 0.999]), t=20000.0, p=0.9)
        run(1e-6 * logits, torch.tensor([0.0, 0.5, 0.999]), k=2000)


def test_odd_strides_and_no_rows():
    logits, u = noise(3, 1001, F16, 9)
    run(logits, u, p=0.9, stride=1003)
    run(logits, u, p=0.9, stride=1008)
    token, share = muillm_ext.mui_sample_filtered(torch.empty((0, 5), dtype=F16, device=DEV), torch.empty(0, device=DEV))
    assert token.shape == share.shape == (0,)


def test_draws_follow_the_weights():
    """Even random numbers: each token comes up in its share of them, give or take one."""
    row = torch.tensor([0.0, 1.0, 2.0, 0.5, -1.0, 2.0]).to(F16)
    n = 2048
    u = (torch.arange(n) + 0.5) / n
    token, share = muillm_ext.mui_sample_filtered(row.expand(n, -1).contiguous().to(DEV), u.to(DEV))
    w = torch.softmax(row.double(), 0)
    seen = torch.bincount(token.cpu(), minlength=6).double()
    assert bool(((seen - n * w).abs() <= 1.0).all())
    assert torch.allclose(share.cpu().double(), w[token.cpu()], rtol=2.0 ** -23, atol=0)


@pytest.mark.parametrize("dtype,vocab", [(F16, 9), (BF16, 1003), (F16, 47723), (BF16, 65521), (BF16, 70003)])
def test_rows_that_begin_anywhere(dtype, vocab):
    """Rows an odd number of logits apart, in a tensor that begins at any of eight places: each token at the ends of its row is found."""
    logits, u = noise(9, vocab, dtype, 5)
    for shift in (0, 1, 5):
        wide = torch.full((9 * (vocab + 2) + 16,), 60.0, dtype=dtype, device=DEV)
        at = wide[shift:shift + 9 * (vocab + 2)].view(9, vocab + 2)[:, :vocab]
        at.copy_(logits)
        token, _ = muillm_ext.mui_sample_filtered(at, u.to(DEV), temperature=0.9, top_p=0.95)
        for r in range(9):
            assert int(token[r]) == pick(logits[r], float(u[r]), torch.tensor(0.9).item(), 0, torch.tensor(0.95).item(), 0.0)[0]
        for place in (0, 1, 7, 8, vocab - 8, vocab - 2, vocab - 1):
            if 0 <= place < vocab:
                one = logits.clone()
                one[:, place] = 50.0
                at.copy_(one)
                assert muillm_ext.mui_sample_filtered(at, u.to(DEV), top_k=1)[0].tolist() == [place] * 9
