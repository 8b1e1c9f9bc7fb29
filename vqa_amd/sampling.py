"""Program tokens drawn on the device: one step of the sampler (Seq2Seq.reinforce_sample, LSTM_Model.py:205-235) for a batch of
logits, with given random numbers, so that the programs never leave the device:

    for t in range(T):
        logits = generator.step(...)                                   # [N, V]
        vqa_amd.sampling.sample(logits, torch.rand(N, device='cuda'), top_p=0.95, out=programs[:, t])
    net.schedule_on_device = True
    scores = net(feats, programs)

Definition.  The tokens of a row stand in descending order of their logits, equal ones by index, with weights
exp((x - max) / temperature).  Kept are at most top_k of them, those whose weight is at least min_p, and of these the tokens in
front of which less than top_p of the weight stands.  Drawn is the first kept token up to which more than u of the kept weight
stands.  The same logits and numbers give the same token on every run.
"""
import torch

from . import ops


_RANGES = dict(temperature=(0.0, 1e30), top_k=(0, 2 ** 31 - 1), top_p=(0.0, 1.0), min_p=(0.0, 1.0))


def _per_row(name, v, rows, device):
    """A number (checked), or a tensor with one value per row in the type the kernel reads.  (Values in a tensor are not looked
    at here: that would wait for the device.  The kernel has an answer for each.)"""
    if isinstance(v, torch.Tensor):
        kind = torch.int32 if name == 'top_k' else torch.float32
        if (v.shape != (rows,) or v.device != device or v.is_floating_point() != kind.is_floating_point or v.dtype == torch.bool or
                v.is_complex()):
            raise ValueError('%s must be a number or a tensor of %d %s on the device of the logits' %
                             (name, rows, 'integers' if name == 'top_k' else 'floating numbers'))
        if v.dtype in (torch.int64, torch.uint64, torch.uint32):
            v = v.to(torch.int64).clamp(0, _RANGES[name][1])       # (2^63 and more become negative, then 0: off, as it should)
        return v.detach().to(kind).contiguous()
    lo, hi = _RANGES[name]
    v = int(v) if name == 'top_k' else float(v)
    if not lo <= v <= hi:
        raise ValueError('%s must be in [%g, %g]' % (name, lo, hi))
    return v


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, return_log_probs=False):
    """int64 tokens [N] drawn from logits [N, V] (bf16, fp16 or fp32) with the uniform numbers u [N] in [0, 1), fp32.

    temperature (0: the first token of the order), top_k (0: off), top_p (1: off) and min_p (0: off) are numbers or tensors
    with one value per row.  `out`: an int64 tensor [N] of any stride to write to, e.g. a column of the programs.
    `return_log_probs`: also the fp32 log-probability of each token among the kept ones, the distribution it was drawn from.
    -inf masks a token out and NaN counts as -inf; a row with nothing to draw gets -1 and -inf.  Not differentiable: see
    vqa_amd.loss.token_log_probs."""
    if logits.dim() != 2 or logits.dtype not in ops.ROW_DTYPES or logits.size(1) < 1:
        raise ValueError('logits must be [N, V] in bf16, fp16 or fp32')
    rows, V = logits.shape
    if u.shape != (rows,) or u.dtype != torch.float32:
        raise ValueError('u must be fp32 [%d]' % rows)
    if out is not None and (out.shape != (rows,) or out.dtype != torch.int64 or (rows > 1 and out.stride(0) == 0)):
        raise ValueError('out must be int64 [%d]' % rows)
    ops._need_cuda(logits, u, out)
    x = logits if V == 1 or logits.stride(1) == 1 else logits.detach().contiguous()
    dev = x.device
    params = [_per_row('temperature', temperature, rows, dev), _per_row('top_k', top_k, rows, dev),
              _per_row('top_p', top_p, rows, dev), _per_row('min_p', min_p, rows, dev)]
    token = torch.empty(rows, dtype=torch.int64, device=dev) if out is None else out
    logp = torch.empty(rows, dtype=torch.float32, device=dev) if return_log_probs else None
    if rows:
        ops.sample(x, x.stride(0), rows, V, u if u.is_contiguous() else u.contiguous(), token, token.stride(0), logp, *params)
        if out is not None:                   # as every write in place: tokens that a backward pass still needs are missed then
            torch.autograd.graph.increment_version(out)
    return (token, logp) if return_log_probs else token
