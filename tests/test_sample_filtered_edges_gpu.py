"""Settings beyond the usual ones, and the paths that long rows take, against the definition."""
import pytest
import torch

from .test_sample_filtered_gpu import noise, run

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
