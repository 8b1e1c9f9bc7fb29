"""The Dropout module on the GPU where its forward pass runs twice."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('reentrant', [True, False])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
def test_a_recomputed_module_takes_the_same_mask(dtype, reentrant):
    from vqa_amd.dropout import Dropout
    torch.manual_seed(5)
    drop = Dropout(0.5)                                        # kept elements are doubled: all products here are exact
    w = (torch.randint(1, 8, (33, 70)) * 0.25).to('cuda:0', dtype).requires_grad_(True)
    x = (torch.randint(1, 8, (33, 70)) * 0.25).to('cuda:0', dtype).requires_grad_(True)
    out = checkpoint(lambda t: drop(t) * w, x, use_reentrant=reentrant)
    other = drop(x.detach())                                   # (another call in between)
    out.sum().backward()
    mask = (out != 0).to(dtype) * 2
    assert not torch.equal(mask, (other != 0).to(dtype) * 2)
    assert torch.equal(out, x * w * mask)
    assert torch.equal(x.grad, w * mask) and torch.equal(w.grad, x * mask)


def test_an_executor_with_hidden_dropout_refuses_to_be_recomputed(vocab):
    from test_policy_gpu import batch, executor
    net = executor(vocab)
    x, prog, _ = batch(vocab, 5)
    x.requires_grad_(True)
    net.hidden_dropout = 0.5
    out = checkpoint(net, x, prog, use_reentrant=True)
    with pytest.raises(RuntimeError, match='recomputed'):
        out.sum().backward()
    assert net.dropout_offset == 5 * 256 // 8
    net.hidden_dropout = 0.0
    (want,) = torch.autograd.grad(net(x, prog).sum(), x)
    checkpoint(net, x, prog, use_reentrant=True).sum().backward()
    assert torch.equal(x.grad, want)
