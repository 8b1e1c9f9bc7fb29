"""Token sampling of few long rows, which several workgroups share, next to rows of the same length that are not split."""
import pytest
import torch

from test_sample_gpu import check, dev, logits, uniform
from vqa_amd import _lib

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def test_which_rows_are_split():
    need = _lib.load().vqa_sample_workspace
    for rows, V in ((1, 34304), (8, 45056), (32, 81920), (64, 131072)):
        assert need(rows, V) > 0 and need(rows, V - 1) == 0 and need(65, V) == 0


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,V', [(48, 107003), (64, 131072)])
def test_every_row_its_own_parameters(dtype, rows, V):
    g = torch.Generator().manual_seed(V)
    pick = lambda: torch.rand(rows, generator=g)                       # noqa: E731
    check(logits(rows, V, V, dtype), pick(), temperature=(pick() * 2).masked_fill(pick() < 0.2, 0.0),
          top_k=torch.randint(0, V + 5, (rows,), generator=g, dtype=torch.int32).masked_fill(pick() < 0.3, 0),
          top_p=(pick() * 1.2).clamp(max=1.0), min_p=(pick() * 0.3 - 0.1).clamp(min=0.0))


@pytest.mark.parametrize('V', [45056, 65536, 100003])
def test_split_and_whole_rows_agree(V):
    from vqa_amd.sampling import sample
    x = logits(300, V, V, torch.float32)
    u = uniform(300, V).to(dev())
    for params in (dict(top_p=0.9), dict(top_k=30), dict(top_k=1900), dict(temperature=0.5)):
        want = sample(x, u, return_log_probs=True, **params)
        for n in (1, 8):
            got = sample(x[:n], u[:n], return_log_probs=True, **params)
            assert torch.equal(got[0], want[0][:n])
            assert ((got[1] - want[1][:n]).abs() <= want[1][:n].abs() * 2.0 ** -23).all()
