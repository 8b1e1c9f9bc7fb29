"""Cross-entropy for the executor's logits in two small launches (torch.nn.CrossEntropyLoss of
Train_model.py:185,312 takes seven: log-softmax, gather, mean, and their gradients).

    loss_fn = vqa_amd.loss.CrossEntropyLoss()
    loss_fn(scores, answers).backward()

Mean reduction over the batch, no class weights, no label smoothing, targets int64 in [0, num_answers):
the reference's call.  The forward kernel also writes d(loss)/d(logits); backward multiplies it by the
incoming gradient.  fp32 logits on the GPU only: there is no CPU path.

Log-probability and entropy of sampled program tokens, differentiable: the score of a policy gradient
(Seq2Seq.reinforce_backward, LSTM_Model.py:261-278), for any vocabulary, in bf16, fp16 or fp32.

    lp, ent = vqa_amd.loss.token_log_probs(logits, programs, ignore_index=0, entropy=True)   # [N, T] each
    (-(reward[:, None] * lp).sum() - 0.01 * ent.sum()).backward()
"""
import torch
from torch.autograd.function import once_differentiable

from . import ops


class _Xent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target):
        if not logits.is_cuda or logits.dim() != 2 or logits.dtype != torch.float32:
            raise ValueError('logits must be a 2-D fp32 tensor on the GPU')
        if target.dim() != 1 or target.size(0) != logits.size(0):
            raise ValueError('targets must be [N]')
        lg = logits.detach().contiguous()
        tg = target.detach().to(device=logits.device, dtype=torch.int64).contiguous()
        loss = torch.empty((), dtype=torch.float32, device=logits.device)
        d = torch.empty_like(lg)
        ops.xent(lg, tg, loss, d)
        ctx.save_for_backward(d)
        return loss

    @staticmethod
    def backward(ctx, grad):
        (d,) = ctx.saved_tensors
        return d * grad, None


def cross_entropy(logits, target):
    return _Xent.apply(logits, target)


class CrossEntropyLoss(torch.nn.Module):
    def forward(self, logits, target):
        return _Xent.apply(logits, target)


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, ignore, want_entropy):
        ctx.set_materialize_grads(False)
        x, *layout = ops.row_layout(logits)
        tk = tokens.contiguous()
        lp = torch.empty(tokens.shape, dtype=torch.float32, device=x.device)
        ent = torch.empty_like(lp) if want_entropy else None
        stats = torch.empty(layout[0], 4, dtype=torch.float32, device=x.device)
        if layout[0]:
            ops.token_logp(x, layout, tk, lp, ent, stats, x.size(-1), temperature, ignore)
        # (the caller's own tensor where it was read in place: autograd then notices a change before backward)
        ctx.save_for_backward(x, tk, stats)
        ctx.args = x.stride(), layout, logits.shape, temperature, ignore
        return (lp, ent) if want_entropy else lp

    @staticmethod
    def backward(ctx, g, h=None):
        return (_log_probs_grad_once if torch.is_grad_enabled() else _log_probs_grad)(ctx, g, h)


def _log_probs_grad(ctx, g, h):
    # (as little as can be: what runs in autograd's thread takes three times as long as in the caller's)
    if g is None and h is None:
        return None, None, None, None, None
    x, tk, stats = ctx.saved_tensors
    if not x.get_device() == tk.get_device() == stats.get_device():
        ops._same_device(x, tk, stats)        # (raises: a saved-tensor hook has left some elsewhere)
    strides, layout, shape, temperature, ignore = ctx.args
    if x.stride() != strides:                 # (a saved-tensor hook has laid it out anew, be it at the same address)
        x, *layout = ops.row_layout(x)
    dx = torch.empty(shape, dtype=x.dtype, device=x.device)
    if layout[0]:
        ops.token_logp_backward(x, layout, tk.contiguous(), stats.contiguous(), g if g is None else g.contiguous(),
                                h if h is None else h.contiguous(), dx, shape[-1], temperature, ignore)
    return dx, None, None, None, None


_log_probs_grad_once = once_differentiable(_log_probs_grad)


def token_log_probs(logits, tokens, temperature=1.0, ignore_index=None, entropy=False):
    """log softmax(logits / temperature) at `tokens`, fp32 of the tokens' shape; with `entropy` a pair of that and the
    entropy of each row's distribution.  Both are differentiable with respect to the logits (once).

    logits [..., V]: bf16, fp16 or fp32 on the GPU, rows at up to two strides are read in place (a slice over time steps);
    tokens [...]: int64.  A token equal to `ignore_index` or outside [0, V) (padding behind a program's end) gives 0 and no
    gradient.  -inf masks a token out; a row with nothing else gives -inf, entropy 0 and no gradient."""
    if logits.dtype not in ops.ROW_DTYPES or logits.dim() < 1 or logits.size(-1) < 1:
        raise ValueError('logits must be [..., V] in bf16, fp16 or fp32')
    if tokens.dtype != torch.int64 or tokens.shape != logits.shape[:-1]:
        raise ValueError('tokens must be int64 of shape %s' % (tuple(logits.shape[:-1]),))
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError('temperature must be in [1e-6, 1e6]')
    ops._same_device(logits, tokens)
    ignore = -1 if ignore_index is None or not 0 <= ignore_index < logits.size(-1) else int(ignore_index)
    return _TokenLogProbs.apply(logits, tokens, temperature, ignore, bool(entropy))
