"""The operators of the program policy where the framework uses them: dropout on the executor's hidden layers, and a whole
cycle of sampling programs on the device, scoring them, and training the generator and the executor on the outcome."""
import numpy as np
import pytest
import torch

from philox_oracle import bits16

pytestmark = pytest.mark.gpu


def dev():
    return torch.device('cuda:0')


def rel(a, b):
    return ((a.detach().double().cpu() - b.detach().double().cpu()).norm() / b.detach().double().norm().cpu().clamp_min(1e-30)).item()


def executor(vocab, fcs=(256,), precision='bf16', seed=11):
    from vqa_amd import synth
    from vqa_amd.module_net import ModuleNet
    dims = dict(feature_dim=(128, 14, 14), module_dim=128, classifier_proj_dim=128, classifier_fc_layers=fcs)
    net = ModuleNet(False, vocab, **dims)
    net.load_state_dict(synth.synth_state_dict(seed, vocab, **dims))
    net.to(dev()).train()
    net.precision = precision
    net.keep_state = True
    return net


def batch(vocab, n, seed=11):
    from vqa_amd import synth
    return (torch.from_numpy(synth.synth_features(seed, n, (128, 14, 14))).to(dev()),
            torch.from_numpy(synth.synth_programs(seed, n, vocab, max_len=12, max_nodes=9)).to(dev()),
            torch.from_numpy(synth.synth_answers(seed, n)).to(dev()))


def masks(net, n, offset, seed):
    """The factor of every hidden activation, per layer, from the generator's definition."""
    from vqa_amd.dropout import threshold
    thr, out = threshold(net.hidden_dropout), []
    for fo in net._dims['fcs']:
        keep = torch.from_numpy(bits16(n * fo, seed, offset) >= thr).view(n, fo)
        out.append(keep.double() * (65536.0 / (65536 - thr)))
        offset += (n * fo + 7) // 8
    return out


@pytest.mark.parametrize('precision,fuse_head', [('bf16', True), ('bf16', False), ('fp32', True)])
@pytest.mark.parametrize('fcs', [(256,), (256, 128)])
def test_hidden_dropout_of_the_executor(vocab, precision, fuse_head, fcs):
    """The classifier's linear layers from their own stored input, in 64 bits with the masks of the definition: logits,
    activations and the gradients of every layer behind the first hidden one, within the path's tolerance (fp32 1e-3, bf16
    2e-2).  A bias gradient is the column sum of the same gradient as the weight's."""
    n = 10
    net = executor(vocab, fcs, precision)
    net.fuse_head = fuse_head
    x, prog, ans = batch(vocab, n)
    net.hidden_dropout, net.dropout_seed, net.dropout_offset = 0.3, 77, 1000
    logits = net(x, prog)
    dl = torch.randn(logits.shape, generator=torch.Generator().manual_seed(1)).to(dev())
    st = net.last_state
    acts = [a.view(-1, w)[:n].float().cpu() for a, w in zip(st['acts'][1:], fcs)]
    c1 = st['acts'][0].view(-1, net._dims['p'] * 196)[:n].double().cpu()
    logits.backward(dl)
    assert net.dropout_offset == 1000 + sum((n * f + 7) // 8 for f in fcs)

    tol = 2e-2 if precision == 'bf16' else 1e-3
    params = [(net.classifier[i].weight.detach().double().cpu().requires_grad_(True),
               net.classifier[i].bias.detach().double().cpu().requires_grad_(True)) for i in net._fc_idx]
    if precision == 'bf16':                                   # channels-last maps: to the order of the weight's columns
        c1 = c1.view(n, 196, -1).permute(0, 2, 1).reshape(n, -1)
    h = c1
    for (w, b), m, stored in zip(params, masks(net, n, 1000, 77), acts):
        h = torch.relu(h @ w.t() + b) * m
        assert (stored[m == 0] == 0).all()
        assert rel(stored, h) <= tol
    out = h @ params[-1][0].t() + params[-1][1]
    assert rel(logits, out) <= tol
    out.backward(dl.double().cpu())
    for i, (w, b) in zip(net._fc_idx, params):
        assert rel(net.classifier[i].weight.grad, w.grad) <= tol, i
        assert rel(net.classifier[i].bias.grad, b.grad) <= tol, i

    # the next call takes other masks, evaluation takes none, and without dropout nothing has changed
    again = net(x, prog)
    assert not torch.equal(again, logits)
    net.eval()
    with torch.no_grad():
        plain = net(x, prog)
    net.train()
    net.hidden_dropout = 0.0
    with torch.no_grad():
        assert torch.equal(net(x, prog), plain)
    net.hidden_dropout = 1.5
    with pytest.raises(ValueError):
        net(x, prog)


def test_same_masks_same_bits(vocab):
    """A step repeated from the same counter has the same logits and gradients, bit for bit."""
    x, prog, ans = batch(vocab, 7)
    net = executor(vocab)
    net.hidden_dropout = 0.5
    got = []
    for _ in range(2):
        net.dropout_offset = 3
        net.zero_grad(set_to_none=True)
        logits = net(x, prog)
        logits.sum().backward()
        got.append([logits.detach()] + [p.grad for p in net.parameters() if p.grad is not None])
    assert len(got[0]) == len(got[1]) and all(torch.equal(a, b) for a, b in zip(*got))


def test_a_round_of_sampling_scoring_and_training(vocab):
    """Programs are sampled token by token into the array that the device scheduler reads, scored there, and the reward goes
    back through their log-probabilities; then the executor takes a training step on them with dropout."""
    from vqa_amd.loss import cross_entropy, token_log_probs
    from vqa_amd.sampling import sample
    n, T, V = 24, 10, len(vocab['program_token_to_idx'])
    t2i = vocab['program_token_to_idx']
    x, _, ans = batch(vocab, n)
    g = torch.Generator().manual_seed(5)
    first = torch.randn(n, V, generator=g).to(dev())
    table = torch.randn(V, V, generator=g).to(dev()).requires_grad_(True)       # logits of the next token given the last
    u = torch.rand(T, n, generator=g).to(dev())
    never = torch.zeros(V, device=dev())
    never[t2i['<START>']] = -float('inf')
    programs = torch.zeros(n, T, dtype=torch.int64, device=dev())
    behaviour = torch.zeros(n, T, device=dev())
    step = first + never
    for t in range(T):
        tk, behaviour[:, t] = sample(step, u[t], temperature=0.8, out=programs[:, t], return_log_probs=True)
        step = table.detach()[programs[:, t]] + never
    assert (programs != t2i['<START>']).all() and (programs >= 0).all() and (programs < V).all()

    net = executor(vocab)
    net.schedule_on_device = True
    net.hidden_dropout = 0.2
    net.eval()
    with torch.no_grad():
        scores = net(x, programs)
    net.raise_for_schedule_error()
    net.schedule_on_device = False
    with torch.no_grad():
        assert torch.equal(scores, net(x, programs))          # the host scheduler on a copy of the same programs
    reward = (scores.argmax(1) == ans).float() - 0.5

    logits = torch.cat([first[:, None], table[programs[:, :-1]]], 1) + never     # [n, T, V]
    lp, ent = token_log_probs(logits, programs, temperature=0.8, ignore_index=t2i['<NULL>'], entropy=True)
    live = programs != t2i['<NULL>']
    # without a filter the distribution that was drawn from is the one that is scored: fp32 against 64 bits, |lp| < 20
    assert ((lp - behaviour).abs()[live] <= 2.0 ** -24 * (80 + 4 * 25)).all()
    loss = -(reward[:, None] * lp).sum() - 0.01 * ent.sum()
    (dt,) = torch.autograd.grad(loss, table)

    tab = table.detach().double().cpu().requires_grad_(True)
    pc = programs.cpu()
    z = (torch.cat([first.double().cpu()[:, None], tab[pc[:, :-1]]], 1) + never.double().cpu()) / 0.8
    logp = torch.log_softmax(z, -1)
    ref_lp = logp.gather(-1, pc[..., None])[..., 0]
    ref_ent = -(logp.exp() * torch.where(logp.isinf(), 0.0, logp)).sum(-1)
    ok = live.cpu()
    ref = -(reward.double().cpu()[:, None] * ref_lp)[ok].sum() - 0.01 * ref_ent[ok].sum()
    (dr,) = torch.autograd.grad(ref, tab)
    assert abs(loss.item() - ref.item()) <= 1e-4 * (1 + ref_lp[ok].abs().sum().item() * 0.5)
    assert rel(dt, dr) <= 1e-4

    net.train()
    before = net.dropout_offset
    loss = cross_entropy(net(x, programs), ans)
    loss.backward()
    assert net.dropout_offset > before and np.isfinite(loss.item())
    assert all(torch.isfinite(p.grad).all() for p in net.parameters() if p.grad is not None)


def test_saved_tensors_left_on_the_host_are_refused():
    """A saved-tensor hook that moves to the host and does not move back."""
    from vqa_amd.dropout import dropout
    from vqa_amd.loss import token_log_probs
    x = torch.randn(4, 44, device='cuda:0', requires_grad=True)
    tk = torch.zeros(4, dtype=torch.int64, device='cuda:0')
    state = torch.tensor([1, 2], dtype=torch.int64, device='cuda:0')
    for left in (lambda t: True, lambda t: t.dtype == torch.int64, lambda t: t.numel() == 16):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu() if left(t) else t, lambda t: t):
            lp, y = token_log_probs(x, tk), dropout(x, 0.5, state)
        with pytest.raises(RuntimeError, match='no CPU fallback'):
            lp.sum().backward()
        if left(state):
            with pytest.raises(RuntimeError, match='no CPU fallback'):
                y.sum().backward()


def test_tokens_written_over_before_backward_are_refused():
    from vqa_amd.loss import token_log_probs
    from vqa_amd.sampling import sample
    x = torch.randn(4, 44, device='cuda:0', requires_grad=True)
    u, tk = torch.rand(4, device='cuda:0'), torch.zeros(4, dtype=torch.int64, device='cuda:0')
    lp = token_log_probs(x, tk)
    sample(x, u, out=tk)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        lp.sum().backward()
    with torch.inference_mode():
        out = torch.zeros(4, dtype=torch.int64, device='cuda:0')
        assert torch.equal(sample(x, u, out=out), tk)
