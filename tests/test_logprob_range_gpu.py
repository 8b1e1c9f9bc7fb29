"""Token log-probabilities over the whole range of the logits, against the formulas in 64 bits with the bounds of
test_logprob_gpu."""
import pytest
import torch

from test_logprob_gpu import check, logits, tokens_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('V', [44, 300, 5000, 20011])
@pytest.mark.parametrize('temperature', [10.0, 1e6])
def test_logits_further_apart_than_the_largest_number(dtype, V, temperature):
    """Their difference over the temperature is a number again."""
    x = logits((4, V), V, dtype)
    x[0, 1], x[0, V // 2] = 3e38, -3e38
    x[1, V - 1], x[1, 2] = torch.finfo(dtype).max, torch.finfo(dtype).min
    x[2] = torch.linspace(-3e38, 3e38, V, dtype=torch.float64)        # (in 32 bits its own step overflows)
    tk = tokens_for((4,), V, 5)
    tk[0], tk[1], tk[2] = V // 2, 2, 0
    check(x, tk, temperature)
