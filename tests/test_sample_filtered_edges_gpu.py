"""Settings beyond the usual ones, and the paths that long rows take, against the definition."""
import pytest
import torch

from muillm_amd import muillm_ext

from .test_sample_filtered_gpu import DEV, noise, run

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("least", [1.0, 1.0000001, 1.5, float("inf")])
@pytest.mark.parametrize("dtype,vocab", [(F16, 100), (BF16, 3000), (BF16, 70001)])
def test_min_p_of_one_and_more(dtype, vocab, least):
    """Up to 1 the tokens tied with the largest stay, beyond it the first of them alone."""
    logits, _ = noise(4, vocab, dtype, 3)
    for row in range(4):
        logits[row, 5 + row::17] = 9.0
    u = torch.tensor([0.0, 0.4, 0.8, 0.999])
    m = torch.full((4,), least)
    run(logits, u, m=m)
    run(logits, u, m=m, k=3)
    run(logits, u, m=m, p=0.5, t=0.7)
    run(logits, u, m=m, t=0.0)
    m[1::2] = 0.1
    run(logits, u, m=m)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("vocab", [40000, 40001, 65528, 65529, 131072, 200003])
def test_long_rows(dtype, vocab):
    """In one launch (fp16 up to 65528 logits), in two with two parts and with more; counts that 16 bits hold just so, and such that they do not."""
    logits, u = noise(2, vocab, dtype, 1)
    run(logits, u, p=0.95)
    run(logits, u, k=700, m=0.01)
    logits[:] = 1.5
    run(logits, torch.tensor([0.0, 0.999]))
    run(logits, torch.tensor([0.5, 0.25]), p=0.5)
    run(logits, torch.tensor([0.5, 0.999]), k=vocab - 3)


@pytest.mark.parametrize("dtype,vocab", [(BF16, 65521), (BF16, 65528), (F16, 65528), (BF16, 65529)])
def test_a_batch_of_long_rows_of_equal_logits(dtype, vocab):
    """64 rows: one launch up to 65528 logits of either type, all of them in one count. Token i is drawn where i <= u * vocab < i + 1."""
    logits = torch.full((64, vocab), -2.0, dtype=dtype, device=DEV)
    at = torch.linspace(0, vocab - 1, 64).round().long()
    u = ((at.double() + 0.5) / vocab).float()
    token, share = muillm_ext.mui_sample_filtered(logits, u.to(DEV))
    assert torch.equal(token.cpu(), (u.double() * vocab).floor().long())
    assert torch.allclose(share.cpu().double(), torch.full((64,), 1.0 / vocab, dtype=torch.float64), rtol=2.0 ** -23, atol=0)
