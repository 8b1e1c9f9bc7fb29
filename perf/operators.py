"""The operators of the program policy around the executor, as cases to be timed and compared: sampling the next program
token of every row, log-probability and entropy of chosen tokens with their gradient, and dropout with its gradient.

`own = False`: `run` computes them in their plain form, elementary torch operations in 32 bits, in 64 where cumulative
sums are compared with a border.  `own = True`: `run` calls vqa_amd.sampling, vqa_amd.loss and vqa_amd.dropout.

Definitions
  sample        tokens of a row in descending order of their logit, equal ones by index; weights w = exp((x - max) / T).
                Kept is a prefix of that order: at most top_k tokens, those with w >= min_p, and of these the tokens
                whose exclusive cumulative weight is below top_p times the sum.  The answer is the first kept token whose
                inclusive cumulative weight exceeds u times the sum of the kept weights; its log-probability among the
                kept ones comes with it.  T = 0 takes the first token.
  token_log_probs  z = x / T;  lp = z[token] - logsumexp(z),  H = -sum p log p;  with g and h the gradients that arrive,
                dx = (g (onehot - p) - h p (log p + H)) / T.  A token below 0 is padding: zeros throughout.
  dropout       16 random bits per element from Philox4x32-10 (key: the seed; counter: offset + index // 8); an element
                whose bits are below t = round(65536 p) becomes 0, the others are scaled by 65536 / (65536 - t).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
BYTES = {'bf16': 2, 'fp16': 2, 'fp32': 4}
PADDING = -1


def listed():
    return [
        # one decoding step of the program generator for a batch of 1024 questions (44 program tokens), written into
        # a column of the [N, 30] program tensor that the executor's device scheduler reads
        dict(name='sample programs', op='sample', rows=1024, vocab=44, dtype='fp32', mode='free', masked=0.0),
        # a single request with a large vocabulary: the latency of one answer
        dict(name='sample one row', op='sample', rows=1, vocab=50001, dtype='bf16', mode='top_k', masked=0.0),
        # a serving batch in which every request has its own temperature, top-k, top-p and min-p, under a grammar mask
        dict(name='sample mixed requests', op='sample', rows=64, vocab=131072, dtype='bf16', mode='mixed', masked=0.3),
        # rollouts of a whole batch from a large vocabulary in single precision
        dict(name='sample rollouts', op='sample', rows=512, vocab=131072, dtype='fp32', mode='top_p', masked=0.0),
        # log-probabilities of 1024 programs of 30 tokens for the policy gradient, with the entropy bonus
        dict(name='log-probs programs', op='logp', rows=30720, vocab=44, dtype='fp32', entropy=True, temperature=1.0),
        # a few tokens over a large vocabulary of odd size
        dict(name='log-probs few rows', op='logp', rows=3, vocab=100003, dtype='bf16', entropy=False, temperature=0.7),
        # a training batch over a middle-sized vocabulary
        dict(name='log-probs batch', op='logp', rows=2048, vocab=32768, dtype='fp16', entropy=True, temperature=1.0),
        # a long training batch over a large vocabulary
        dict(name='log-probs largest', op='logp', rows=4096, vocab=131072, dtype='bf16', entropy=False, temperature=1.0),
        # the classifier's hidden layer at the default batch
        dict(name='dropout hidden layer', op='dropout', rows=1024, cols=1024, dtype='bf16', p=0.5),
        # embeddings of odd width
        dict(name='dropout odd', op='dropout', rows=333, cols=299, dtype='fp32', p=0.1),
        # activations of a training batch in half precision
        dict(name='dropout activations', op='dropout', rows=8192, cols=4096, dtype='fp16', p=0.1),
        # the largest activations
        dict(name='dropout largest', op='dropout', rows=32768, cols=8192, dtype='bf16', p=0.2),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['sample', 'logp', 'dropout'])
    dtype = rng.choice(['bf16', 'fp16', 'fp32'])
    if op == 'dropout':
        cols = _log_uniform(rng, 1, 8192)
        rows = _log_uniform(rng, max(1, 64 // cols), 32768)
        if dtype == 'fp32':
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, p=round(rng.uniform(0.02, 0.7), 3))
    vocab = _log_uniform(rng, 2, 131072)
    if op == 'sample':
        rows = min(_log_uniform(rng, 1, 1024), 2 ** 26 // vocab)
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, mode=rng.choice(['free', 'top_k', 'top_p', 'mixed']),
                    masked=rng.choice([0.0, 0.0, 0.5]))
    rows = min(_log_uniform(rng, 1, 32768), 2 ** 28 // vocab)
    return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, entropy=rng.random() < 0.5,
                temperature=rng.choice([1.0, 0.7, 1.3]))


def _logits(case, g, dev):
    """Rows from flat to peaked: a spread of their own each, and a few tokens that stand out."""
    rows, vocab = case['rows'], case['vocab']
    x = torch.randn(rows, vocab, generator=g, device=dev)
    x *= torch.rand(rows, 1, generator=g, device=dev) * 2.5 + 0.5
    at = torch.randint(0, vocab, (rows, 5), generator=g, device=dev)
    x.scatter_add_(1, at, torch.rand(rows, 5, generator=g, device=dev) * 6 + 2)
    if case.get('masked'):
        off = torch.rand(rows, vocab, generator=g, device=dev) < case['masked']
        off[:, 0] = False
        x.masked_fill_(off, float('-inf'))
    return x.to(DTYPES[case['dtype']])


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case)
    if case['op'] == 'dropout':
        t = DTYPES[case['dtype']]
        shape = (case['rows'], case['cols'])
        s['x'] = torch.randn(shape, generator=g, device=dev).to(t).requires_grad_(True)
        s['dy'] = torch.randn(shape, generator=g, device=dev).to(t)
        s['seed'], s['offset'] = seed * 0x9E3779B97F4A7C15 % 2 ** 63, seed * 1000003 % 2 ** 40
        return s
    rows, vocab = case['rows'], case['vocab']
    s['x'] = _logits(case, g, dev)
    if case['op'] == 'logp':
        s['x'].requires_grad_(True)
        tokens = torch.randint(0, vocab, (rows,), generator=g, device=dev)
        pad = torch.rand(rows, generator=g, device=dev) < 0.2          # the padding behind the programs' ends
        pad[0] = False
        s['tokens'] = tokens.masked_fill(pad, PADDING)
        s['g'] = torch.randn(rows, generator=g, device=dev)            # advantages
        s['h'] = torch.full((rows,), 0.01, device=dev) if case['entropy'] else None
        return s
    s['u'] = torch.rand(rows, generator=g, device=dev)
    s['out'] = torch.zeros(rows, 30, dtype=torch.int64, device=dev)[:, 7]
    s['params'] = dict(temperature=0.9, top_k=0, top_p=1.0, min_p=0.0)
    if case['mode'] == 'free':
        s['params']['temperature'] = 1.0
    elif case['mode'] == 'top_k':
        s['params'].update(top_k=50, top_p=0.95)
    elif case['mode'] == 'top_p':
        s['params']['top_p'] = 0.95
    else:                                                              # every row its own, some of them greedy
        pick = lambda: torch.rand(rows, generator=g, device=dev)       # noqa: E731
        temp = (pick() + 0.5).masked_fill(pick() < 0.1, 0.0)
        k = torch.randint(1, 200, (rows,), generator=g, device=dev, dtype=torch.int32).masked_fill(pick() < 0.5, 0)
        top_p = (pick() * 0.5 + 0.5).masked_fill(pick() < 0.3, 1.0)
        min_p = (pick() * 0.1).masked_fill(pick() < 0.5, 0.0)
        s['params'] = dict(temperature=temp, top_k=k, top_p=top_p, min_p=min_p)
    return s


# ---------------------------------------------------------------------------------------- plain forms
def _column(v, rows, dtype, dev):
    if not isinstance(v, torch.Tensor):
        v = torch.full((rows,), v, dtype=dtype, device=dev)
    return v.to(dtype)[:, None]


def _sample_plain(s):
    x, rows, vocab = s['x'], s['rows'], s['vocab']
    p = {k: _column(v, rows, torch.int64 if k == 'top_k' else torch.float64, x.device) for k, v in s['params'].items()}
    greedy = p['temperature'] == 0
    temp = torch.where(greedy, 1.0, p['temperature'])
    k = torch.where(greedy, 1, torch.where(p['top_k'] <= 0, vocab, p['top_k']))
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    xs = xs.double()
    w = torch.exp((xs - xs[:, :1]) / temp)
    keep = (torch.arange(vocab, device=x.device) < k) & (w >= p['min_p'])
    w = torch.where(keep, w, 0.0)
    cum = w.cumsum(1)
    before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], 1)
    keep &= (before < p['top_p'] * cum[:, -1:]) | (p['top_p'] >= 1)
    last = keep.sum(1, keepdim=True) - 1
    total = cum.gather(1, last)
    j = torch.minimum((cum <= s['u'].double()[:, None] * total).sum(1, keepdim=True), last)
    s['out'].copy_(order.gather(1, j)[:, 0])
    return s['out'], (torch.log(w.gather(1, j)) - torch.log(total))[:, 0].float()


def _log_probs_plain(s):
    x, tokens, it = s['x'].detach(), s['tokens'], 1.0 / s['temperature']
    live = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    z = x.float() * it
    z = z - z.amax(1, keepdim=True)
    lp = z - z.exp().sum(1, keepdim=True).log()
    del z
    out = torch.where(live, lp.gather(1, at)[:, 0], 0.0)
    p = lp.exp()
    g = torch.where(live, s['g'], 0.0)[:, None]
    dz = p * -g
    dz.scatter_add_(1, at, g)
    if s['h'] is None:
        return out, (dz * it).to(x.dtype)
    plp = torch.where(p > 0, p * lp, 0.0)
    ent = -plp.sum(1)
    h = torch.where(live, s['h'], 0.0)[:, None]
    dz -= h * (plp + p * ent[:, None])
    return out, torch.where(live, ent, 0.0), (dz * it).to(x.dtype)


def _philox_plain(seed, offset, blocks, dev):
    """[blocks, 8] 16-bit numbers of Philox4x32-10, in int64 arithmetic (products wrap to their low 64 bits)."""
    low = 0xFFFFFFFF
    at = torch.arange(blocks, dtype=torch.int64, device=dev) + offset
    c0, c1 = at & low, (at >> 32) & low
    c2, c3 = torch.zeros_like(c0), torch.zeros_like(c0)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32) & low ^ c1 ^ k0, b & low, (a >> 32) & low ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([h for c in (c0, c1, c2, c3) for h in (c & 0xFFFF, c >> 16)], 1)


def _dropout_plain(s):
    x = s['x'].detach()
    t = int(math.floor(s['p'] * 65536 + 0.5))
    keep = (_philox_plain(s['seed'], s['offset'], -(-x.numel() // 8), x.device).view(-1)[:x.numel()] >= t).view(x.shape)
    scale = 65536.0 / (65536 - t)
    return torch.where(keep, x.float() * scale, 0.0).to(x.dtype), torch.where(keep, s['dy'].float() * scale, 0.0).to(x.dtype)


# ---------------------------------------------------------------------------------------- one pass
def run(s):
    if not own:
        return {'sample': _sample_plain, 'logp': _log_probs_plain, 'dropout': _dropout_plain}[s['op']](s)
    if s['op'] == 'sample':
        from vqa_amd.sampling import sample
        return sample(s['x'], s['u'], out=s['out'], return_log_probs=True, **s['params'])
    x = s['x']
    x.grad = None
    if s['op'] == 'logp':
        from vqa_amd.loss import token_log_probs
        if s['h'] is None:
            lp = token_log_probs(x, s['tokens'], temperature=s['temperature'], ignore_index=PADDING)
            lp.backward(s['g'])
            return lp.detach(), x.grad
        lp, ent = token_log_probs(x, s['tokens'], temperature=s['temperature'], ignore_index=PADDING, entropy=True)
        torch.autograd.backward((lp, ent), (s['g'], s['h']))
        return lp.detach(), ent.detach(), x.grad
    from vqa_amd.dropout import dropout
    y = dropout(x, s['p'], s['seed'], s['offset'])
    y.backward(s['dy'])
    return y.detach(), x.grad


def work(case):
    size = BYTES[case['dtype']]
    if case['op'] == 'dropout':      # x and dy read, y and dx written; a random number and a product for each
        n = case['rows'] * case['cols']
        return dict(bytes=4 * n * size, flops=4 * n)
    n = case['rows'] * case['vocab']
    if case['op'] == 'sample':       # the logits read; a difference, an exponential and a sum for each
        return dict(bytes=n * size + case['rows'] * (4 + 8 + 4), flops=4 * n)
    # the logits read, their gradient written; per logit an exponential and a sum forward, a difference and products back
    return dict(bytes=2 * n * size + case['rows'] * 24, flops=8 * n)


# ---------------------------------------------------------------------------------------- 64 bits
def _sample_exact(case, s):
    if case['rows'] * case['vocab'] > 2 ** 26:
        return None
    x, u = s['x'].double().cpu().numpy(), s['u'].double().cpu().numpy()
    tokens, logs = np.zeros(case['rows'], np.int64), np.zeros(case['rows'])
    for r in range(case['rows']):
        par = {k: float(v[r]) if isinstance(v, torch.Tensor) else v for k, v in s['params'].items()}
        order = np.argsort(-x[r], kind='stable')
        if par['temperature'] == 0:
            tokens[r] = order[0]
            continue
        w = np.exp((x[r][order] - x[r].max()) / par['temperature'])
        n = len(w) if par['top_k'] <= 0 else min(len(w), int(par['top_k']))
        n = min(n, int(np.searchsorted(-w, -par['min_p'], side='right')))
        cum = np.cumsum(w[:n])
        if par['top_p'] < 1:
            n = min(n, 1 + int(np.searchsorted(cum, par['top_p'] * cum[-1], side='left')))
        j = min(int(np.searchsorted(cum[:n], u[r] * cum[n - 1], side='right')), n - 1)
        tokens[r], logs[r] = order[j], np.log(w[j] / cum[n - 1])
    return tokens, logs


def _log_probs_exact(case, s):
    if case['rows'] * case['vocab'] > 2 ** 27:
        return None
    step = max(1, 2 ** 22 // case['vocab'])
    tokens, g = s['tokens'].cpu().numpy(), s['g'].double().cpu().numpy()
    lp, ent, dx = np.zeros(case['rows']), np.zeros(case['rows']), np.zeros((case['rows'], case['vocab']))
    for lo in range(0, case['rows'], step):
        z = s['x'].detach()[lo:lo + step].double().cpu().numpy() / case['temperature']
        live = np.flatnonzero(tokens[lo:lo + step] >= 0)
        z, tk = z[live], tokens[lo:lo + step][live]
        top = z.max(1, keepdims=True)
        e = np.exp(z - top)
        total = e.sum(1, keepdims=True)
        p, lse = e / total, top[:, 0] + np.log(total[:, 0])
        at = np.arange(len(live))
        lp[lo + live] = z[at, tk] - lse
        mean = (p * z).sum(1)
        ent[lo + live] = lse - mean
        d = -p * g[lo + live][:, None]
        d[at, tk] += g[lo + live]
        if s['h'] is not None:                 # log p + H = z - lse + lse - mean
            d -= s['h'].double().cpu().numpy()[lo + live][:, None] * p * (z - mean[:, None])
        dx[lo + live] = d / case['temperature']
    return (lp, dx) if s['h'] is None else (lp, ent, dx)


def _dropout_exact(case, s):
    n = case['rows'] * case['cols']
    if n > 2 ** 26:
        return None
    u64, low = np.uint64, np.uint64(0xFFFFFFFF)
    at = np.arange(-(-n // 8), dtype=u64) + u64(s['offset'])
    c = [at & low, at >> u64(32), np.zeros_like(at), np.zeros_like(at)]
    key = [s['seed'] % 2 ** 32, s['seed'] // 2 ** 32]
    for r in range(10):
        k0, k1 = (u64((k + r * step) % 2 ** 32) for k, step in zip(key, (0x9E3779B9, 0xBB67AE85)))
        a, b = c[0] * u64(0xD2511F53), c[2] * u64(0xCD9E8D57)
        c = [(b >> u64(32)) ^ c[1] ^ k0, b & low, (a >> u64(32)) ^ c[3] ^ k1, a & low]
    bits = np.stack([v.astype(np.uint32) for v in c], 1).astype('<u4').view('<u2').reshape(-1)[:n]
    t = int(np.floor(case['p'] * 65536 + 0.5))
    gain = (bits >= t) * (65536.0 / (65536 - t))
    shape = (case['rows'], case['cols'])
    return tuple(v.detach().double().cpu().numpy() * gain.reshape(shape) for v in (s['x'], s['dy']))


def exact(case, seed):
    f = {'sample': _sample_exact, 'logp': _log_probs_exact, 'dropout': _dropout_exact}[case['op']]
    return f(case, prepare(case, seed))
