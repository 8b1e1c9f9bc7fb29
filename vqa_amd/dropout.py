"""Dropout from a counter-based generator: the mask is a function of (seed, offset, element index), computed in the forward
and again in the backward pass, and never stored.

    y = vqa_amd.dropout.dropout(x, 0.1, seed, offset)          # the caller's own counter
    drop = vqa_amd.dropout.Dropout(0.1)                        # or a module; y = drop(x)

Element i (row-major) is dropped with probability p, rounded to a multiple of 2^-16; the others are multiplied by
1 / (1 - p) for that rounded p.  Dropped elements become 0 whatever they were.  A call uses the counters offset to
offset + ceil(numel / 8) - 1: calls whose ranges do not meet have independent masks, the same range gives the same mask.
bf16, fp16 or fp32 on the GPU; there is no CPU path.
"""
import threading

import torch
from torch.autograd.function import once_differentiable

from . import ops


def blocks(numel):
    """Counters that a call on `numel` elements uses."""
    return (numel + 7) // 8


def threshold(p):
    """p in units of 2^-16, as the kernel takes it."""
    p = float(p)
    if not 0 <= p <= 1:
        raise ValueError('dropout probability must be in [0, 1]')
    return int(p * 65536 + 0.5)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, thr, seed, offset, state):
        x = x.contiguous()
        y = torch.empty_like(x)
        ops.dropout(x, y, thr, seed, offset, state)
        ctx.args = thr, seed & 2 ** 64 - 1, offset & 2 ** 64 - 1
        ctx.save_for_backward(state)          # (changed before backward, it would give another mask: autograd refuses that)
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_dropout_grad_once if torch.is_grad_enabled() else _dropout_grad)(ctx, dy)


def _dropout_grad(ctx, dy):
    # (as little as can be: what runs in autograd's thread takes three times as long as in the caller's)
    (state,) = ctx.saved_tensors
    if state is not None and state.get_device() != dy.get_device():
        ops._same_device(dy, state)           # (raises: a saved-tensor hook has left it elsewhere)
    dy = dy.contiguous()
    dx = torch.empty_like(dy)
    ops.dropout_backward(dy, dx, *ctx.args, state)
    return dx, None, None, None, None


_dropout_grad_once = once_differentiable(_dropout_grad)


def dropout(x, p, seed, offset=0):
    """x with a share p of its elements set to 0 and the others multiplied by 1 / (1 - p).  `seed`, `offset`: integers, taken
    modulo 2^64.  Or `seed` is an int64 tensor {seed, offset} on x's device, read by the kernels when they run: a captured
    graph that advances it draws a new mask on every replay (advance it after the backward pass, not between)."""
    if x.dtype not in ops.ROW_DTYPES:
        raise ValueError('x must be bf16, fp16 or fp32')
    thr = threshold(p)
    ops._need_cuda(x)
    state = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.shape != (2,) or not seed.is_contiguous() or seed.device != x.device or offset != 0:
            raise ValueError('a seed tensor must be int64 [2] (seed, offset) on the device of x, without another offset')
        seed, state = 0, seed
    return _Dropout.apply(x, thr, int(seed), int(offset), state)


def data_rank():
    """This process's number among the data-parallel ranks, 0 outside of a process group."""
    on = torch.distributed.is_available() and torch.distributed.is_initialized()
    return torch.distributed.get_rank() if on else 0


def in_backward():
    """Whether this thread is inside a backward pass: a forward pass there is an earlier one that is recomputed."""
    return torch._C._current_graph_task_id() >= 0


_counting = threading.Lock()              # (of the module's, not of an instance: instances are copied and pickled)


class Dropout(torch.nn.Module):
    """Dropout as a module.  Without a seed every training call draws its own from torch's generator on the host (and adds the
    data-parallel rank): modules, calls and ranks have independent masks, torch.manual_seed decides them, a run that restores
    torch.get_rng_state() repeats none, and activation recomputation, which restores that state as well, gets the mask of the
    first pass.

    With a seed the module counts: every training call takes the next range of counters of that seed, from `offset` on.  Modules
    or ranks of the same seed and offset have the same masks, and `offset` is not in the state dict: whoever resumes such a run
    saves it and sets it again.  A counting module cannot be recomputed (the second pass would count on) and raises."""

    def __init__(self, p=0.5, seed=None):
        super().__init__()
        threshold(p)
        self.p, self.seed, self.offset = float(p), None if seed is None else int(seed), 0

    def forward(self, x):
        if not self.training or self.p == 0:
            return x
        if x.is_cuda and torch.cuda.is_current_stream_capturing():
            # the random numbers would be constants of the graph: the same mask on every replay
            raise RuntimeError('vqa_amd.dropout.Dropout draws or counts on the host: in a captured graph call '
                               'vqa_amd.dropout.dropout with a {seed, offset} tensor')
        if self.seed is None:
            return dropout(x, self.p, torch.empty((), dtype=torch.int64, device='cpu').random_().item() + data_rank())
        if in_backward():
            raise RuntimeError('vqa_amd.dropout.Dropout with a seed counts its calls: recomputed in the backward pass it would '
                               'have another mask; leave the seed out, or call vqa_amd.dropout.dropout with an offset')
        with _counting:
            at = self.offset
            self.offset = at + blocks(x.numel())
        return dropout(x, self.p, self.seed, at)

    def extra_repr(self):
        return 'p=%g' % self.p if self.seed is None else 'p=%g, seed=%d' % (self.p, self.seed)
