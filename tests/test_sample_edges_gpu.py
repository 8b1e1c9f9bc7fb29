"""Token sampling where the weights run out: numbers at and above 1, weights of 0."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# a wave a row, a list of all tokens, and bins: of 256, 512 and 1024 threads, with and without a guess of the range, split rows
SIZES = [(5, 44), (5, 64), (5, 65), (5, 100), (5, 128), (5, 300), (5, 9001), (300, 3000), (300, 20000), (5, 70000)]


def dev():
    return torch.device('cuda:0')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,V', SIZES)
def test_infinite_logits_share_all_the_weight(dtype, rows, V):
    """Also for numbers that no generator of [0, 1) gives: 1 and above draw the last token that weighs anything."""
    from vqa_amd.sampling import sample
    x = torch.randn(rows, V, generator=torch.Generator().manual_seed(V)).to(dtype).to(dev())
    x[:, 3] = x[:, V // 2] = x[:, V - 4] = math.inf
    for u, want in ((0.0, 3), (0.5, V // 2), (1 - 2.0 ** -24, V - 4), (1.0, V - 4), (7.0, V - 4), (math.inf, V - 4)):
        for params in (dict(), dict(temperature=0.3), dict(top_p=0.99), dict(min_p=0.1)):
            tk, lp = sample(x, torch.full((rows,), u, device=dev()), return_log_probs=True, **params)
            assert (tk == want).all(), (u, params, tk[:4])
            assert ((lp + math.log(3)).abs() <= math.log(3) * 2.0 ** -24 + 1e-12).all()


@pytest.mark.parametrize('rows,V', SIZES)
def test_weights_of_zero_are_never_drawn(rows, V):
    """Logits so far down that exp is 0 in 64 bits, in front of and behind the few that count, far above what the row's front
    shows."""
    from vqa_amd.sampling import sample
    x = torch.full((rows, V), -5000.0)
    x[:, : V // 3] = -2000 - torch.rand(V // 3, generator=torch.Generator().manual_seed(V))
    last = V - 2
    x[:, V - 9], x[:, last] = 0.25, 0.0
    x = x.to(dev())
    for u, want in ((0.0, V - 9), (0.999, last), (1.0, last), (math.inf, last)):
        for params in (dict(), dict(top_p=0.999), dict(top_k=V - 1), dict(top_k=30, temperature=0.8)):
            tk, lp = sample(x, torch.full((rows,), u, device=dev()), return_log_probs=True, **params)
            assert (tk == want).all(), (u, params, tk[:4])
            assert torch.isfinite(lp).all() and (lp > -1.0).all()


@pytest.mark.parametrize('dtype', [torch.int8, torch.uint8, torch.int16, torch.uint16, torch.uint32, torch.int64, torch.uint64])
def test_top_k_in_every_integer_type(dtype):
    from vqa_amd.sampling import sample
    x = torch.randn(40, 300, generator=torch.Generator().manual_seed(1)).to(dev())
    u = torch.rand(40, generator=torch.Generator().manual_seed(2)).to(dev())
    k = torch.arange(40)
    assert torch.equal(sample(x, u, top_k=k.to(dtype).to(dev())), sample(x, u, top_k=k.to(torch.int32).to(dev())))
    if dtype in (torch.int64, torch.uint64):
        k = torch.full((40,), 2 ** 32 + 3).to(dtype).to(dev())
        assert torch.equal(sample(x, u, top_k=k), sample(x, u))
