"""Dropout (vqa_amd.dropout over vqa_dropout) against the generator's definition in numpy.  Results are exact: the product
x * scale in fp32 and one rounding to the type are what torch does with the same numbers."""
import math

import numpy as np
import pytest
import torch

from philox_oracle import bits16

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def dev():
    return torch.device('cuda:0')


def expect(x, thr, seed, offset=0):
    keep = torch.from_numpy(bits16(x.numel(), seed, offset) >= thr).view(x.shape).to(x.device)
    scale = torch.tensor(65536.0 / (65536 - thr) if thr < 65536 else 0.0, dtype=torch.float32, device=x.device)
    return torch.where(keep, (x.float() * scale).to(x.dtype), torch.zeros((), dtype=x.dtype, device=x.device))


def data(shape, seed, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n', [1, 7, 8, 9, 255, 2047, 2049, 100003])
@pytest.mark.parametrize('p', [0.1, 0.5])
def test_forward_and_backward(dtype, n, p):
    from vqa_amd.dropout import dropout, threshold
    x = data((n,), n, dtype).requires_grad_(True)
    dy = data((n,), n + 1, dtype)
    seed, offset = 0x123456789ABCDEF + n, 2 ** 32 - 3          # the counter's low word runs over
    y = dropout(x, p, seed, offset)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(y.detach(), expect(x.detach(), threshold(p), seed, offset))
    assert torch.equal(dx, expect(dy, threshold(p), seed, offset))


def test_many_elements_and_the_counter_running_over():
    from vqa_amd.dropout import dropout, threshold
    n = 2 ** 25 + 2 ** 14 + 5
    x = torch.ones(n, dtype=torch.bfloat16, device=dev())
    y = dropout(x, 0.25, 3, 2 ** 64 - 2)                        # and the counter itself runs over
    a = 2 ** 25 - 64                                            # a multiple of 8
    want = expect(x[a:], threshold(0.25), 3, 2 ** 64 - 2 + a // 8)
    assert torch.equal(y[a:], want)
    assert abs(y.float().count_nonzero().item() / n - 0.75) <= 6 * math.sqrt(0.25 * 0.75 / n)


def test_every_probability_extreme_and_what_is_dropped_is_zero():
    from vqa_amd.dropout import dropout
    x = data((4096,), 1, torch.float32)
    x[::2] = math.nan
    x[1::4] = -math.inf
    assert torch.equal(dropout(x, 0.0, 1).isnan(), x.isnan())
    assert torch.equal(dropout(x, 1.0, 1), torch.zeros_like(x))
    y = dropout(x, 0.5, 1)
    keep = torch.from_numpy(bits16(4096, 1, 0) >= 32768).to(dev())
    assert torch.equal(y.isnan(), x.isnan() & keep) and (y[~keep] == 0).all()
    assert not torch.signbit(y[~keep]).any()


def test_strides_alignment_and_broadcast():
    """The mask goes by the row-major index, whatever the strides; a view that starts at an odd element is read in place."""
    from vqa_amd.dropout import dropout, threshold
    base = data((40, 33), 2, torch.bfloat16)
    for v in (base.t(), base[:, 1:20], base.view(-1)[3:1001], base[::2], base[:1].expand(5, 33)):
        assert torch.equal(dropout(v, 0.3, 9), expect(v.contiguous(), threshold(0.3), 9))
    x = data((1, 33), 3, torch.float32).requires_grad_(True)
    (dx,) = torch.autograd.grad(dropout(x.expand(4, 33), 0.5, 2).sum(), x)
    keep = torch.from_numpy(bits16(4 * 33, 2, 0) >= 32768).view(4, 33).to(dev())
    assert torch.equal(dx, 2.0 * keep.sum(0, keepdim=True).float())
    dy = data((33, 40), 4, torch.bfloat16).t()                  # a gradient in another order than x
    xx = base.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(dropout(xx, 0.3, 9), xx, dy)
    assert torch.equal(dx, expect(dy.contiguous(), threshold(0.3), 9))
    e = torch.zeros(0, 5, device=dev(), requires_grad=True)
    assert torch.autograd.grad(dropout(e, 0.3, 9).sum(), e)[0].shape == (0, 5)


def test_in_place_entry():
    from vqa_amd import ops
    x = data((1003,), 5, torch.float16)
    want = expect(x, 20000, 5, 7)
    ops.dropout(x, x, 20000, 5, 7)
    assert torch.equal(x, want)


def test_module_counts_and_follows_training_mode():
    from vqa_amd.dropout import Dropout, threshold
    drop = Dropout(0.2, seed=-5)
    x = data((100,), 6, torch.float32)
    assert torch.equal(drop(x), expect(x, threshold(0.2), -5, 0))
    assert torch.equal(drop(x), expect(x, threshold(0.2), -5, 13)) and drop.offset == 26
    drop.eval()
    assert drop(x) is x and drop.offset == 26


def test_seed_tensor_in_a_captured_graph():
    from vqa_amd.dropout import Dropout, dropout, threshold
    x, dy = data((777,), 7, torch.bfloat16), data((777,), 8, torch.bfloat16)
    leaf = x.clone().requires_grad_(True)
    state = torch.tensor([11, 5], dtype=torch.int64, device=dev())

    def step():
        y = dropout(leaf, 0.4, state)
        (dx,) = torch.autograd.grad(y, leaf, dy)
        state[1:].add_(98)
        return y.detach(), dx
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    state.copy_(torch.tensor([11, 5]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = step()
        with pytest.raises(RuntimeError, match='counts on the host'):
            Dropout(0.5)(leaf)
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, expect(x, threshold(0.4), 11, 5 + 98 * k))
        assert torch.equal(dx, expect(dy, threshold(0.4), 11, 5 + 98 * k))
    assert state.tolist() == [11, 5 + 3 * 98]


def test_advancing_the_seed_tensor_before_backward_is_refused():
    from vqa_amd.dropout import dropout
    x = data((50,), 1, torch.float32).requires_grad_(True)
    state = torch.tensor([1, 0], dtype=torch.int64, device=dev())
    y = dropout(x, 0.5, state)
    state[1:].add_(7)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_a_second_derivative_is_refused():
    from vqa_amd.dropout import dropout
    from vqa_amd.loss import token_log_probs
    x = data((4, 50), 1, torch.float32).requires_grad_(True)
    tk = torch.zeros(4, dtype=torch.int64, device=dev())
    for y in (dropout(x, 0.5, 1), token_log_probs(x, tk)):
        dy = torch.ones_like(y).requires_grad_(True)
        (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
        with pytest.raises(RuntimeError, match='once_differentiable'):
            dx.sum().backward()
