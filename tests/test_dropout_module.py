"""The Dropout module's random numbers: which seed and counters each call takes.  The kernels' place is taken by the generator's
definition on the CPU, so none of it needs a GPU."""
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from philox_oracle import bits16
from vqa_amd import dropout, ops


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    def apply(x, y, threshold, seed, offset, state=None):
        if state is not None:
            seed, offset = state.tolist()
        keep = torch.from_numpy(bits16(x.numel(), seed, offset) >= threshold).view(x.shape)
        y.copy_(torch.where(keep, x * (65536.0 / (65536 - threshold)), 0.0))
    monkeypatch.setattr(ops, '_need_cuda', lambda *t: None)
    monkeypatch.setattr(ops, 'dropout', apply)
    monkeypatch.setattr(ops, 'dropout_backward', apply)


def test_modules_without_a_seed_draw_masks_of_their_own():
    x = torch.ones(512)
    a, b = dropout.Dropout(0.5), dropout.Dropout(0.5)
    torch.manual_seed(3)
    ya, yb, yc = a(x), b(x), a(x)
    # two independent masks agree in 256 of 512 elements, give or take 11.3: 8 deviations
    for u, v in ((ya, yb), (ya, yc), (yb, yc)):
        assert 166 <= (u == v).sum() <= 346
    torch.manual_seed(3)                                       # torch's generator decides them
    assert torch.equal(a(x), ya) and torch.equal(b(x), yb)
    assert 'seed' not in repr(a) and 'seed=4' in repr(dropout.Dropout(0.5, 4))


def test_ranks_draw_masks_of_their_own(monkeypatch):
    x, drop = torch.ones(512), dropout.Dropout(0.5)
    got = []
    monkeypatch.setattr(torch.distributed, 'is_initialized', lambda: True)
    for rank in range(2):
        monkeypatch.setattr(torch.distributed, 'get_rank', lambda: rank)
        torch.manual_seed(3)
        got.append(drop(x))
    assert 166 <= (got[0] == got[1]).sum() <= 346


@pytest.mark.parametrize('reentrant', [True, False])
def test_a_recomputed_module_takes_the_same_mask(reentrant):
    """Activation recomputation runs the forward pass again inside the backward one, with the generator's old state."""
    torch.manual_seed(5)
    drop = dropout.Dropout(0.5)
    w = torch.rand(64, requires_grad=True)
    x = (torch.rand(64) + 1).requires_grad_(True)
    out = checkpoint(lambda t: drop(t) * w, x, use_reentrant=reentrant)
    drop(x.detach())                                           # (another call in between)
    out.sum().backward()
    dropped = out.detach() / (x * w).detach()                  # 0 or 2
    assert torch.allclose(x.grad, dropped * w.detach(), rtol=1e-6) and torch.allclose(w.grad, dropped * x.detach(), rtol=1e-6)


@pytest.mark.parametrize('reentrant', [True, False])
def test_a_counting_module_refuses_to_be_recomputed(reentrant):
    """Its second pass would take the next counters, another mask: wrong gradients."""
    drop = dropout.Dropout(0.5, seed=7)
    w = torch.rand(64, requires_grad=True)
    x = torch.rand(64).requires_grad_(True)
    out = checkpoint(lambda t: drop(t) * w, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match='recomputed'):
        out.sum().backward()
    assert drop.offset == 8
    drop.eval()
    checkpoint(lambda t: drop(t) * w, x, use_reentrant=reentrant).sum().backward()
    assert torch.equal(w.grad, x.detach()) and torch.equal(x.grad, w.detach())


@pytest.mark.parametrize('reentrant', [True, False])
def test_hidden_dropout_refuses_to_be_recomputed(vocab, reentrant):
    from vqa_amd.module_net import ModuleNet
    net = ModuleNet(False, vocab, feature_dim=(128, 14, 14), classifier_proj_dim=128, classifier_fc_layers=(256, 128))
    net.hidden_dropout = 0.25
    got = []

    def stand_in(x):
        got.append(net._start_dropout(5))
        return x * x
    x = torch.rand(8).requires_grad_(True)
    out = checkpoint(stand_in, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match='recomputed'):
        out.sum().backward()
    assert len(got) == 1 and net.dropout_offset == 160 + 80
    net.eval()                                                 # without dropout nothing is refused
    checkpoint(stand_in, x, use_reentrant=reentrant).sum().backward()
    assert got[1:] == [None, None] and torch.equal(x.grad, 2 * x.detach())


def test_two_threads_that_call_one_module_take_different_counters(monkeypatch):
    drop, took, both = dropout.Dropout(0.5, seed=7), [], threading.Barrier(2, timeout=20)

    def apply(x, y, threshold, seed, offset, state=None):
        both.wait()                                            # both calls are on their way
        took.append(offset)
        y.zero_()
    monkeypatch.setattr(ops, 'dropout', apply)
    threads = [threading.Thread(target=drop, args=(torch.ones(64),)) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(took) == [0, 8] and drop.offset == 16
