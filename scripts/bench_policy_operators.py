"""What the figures of the policy operators rest on, besides the cases of perf/operators.py: rates of this card, host time of a
call and of an empty autograd round trip, the same steps by torch's own operators, sizes in fp32, rows that the sampler has to search
by radix or whose guessed range fails, and a training step with hidden_dropout.  Microseconds; the best of a few repetitions.

    python scripts/bench_policy_operators.py > profiles/policy_operators_times.txt
"""
import os
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, 'perf'))
import torch

import operators
from vqa_amd import ops, synth
from vqa_amd import vocab as V
from vqa_amd.dropout import dropout
from vqa_amd.loss import CrossEntropyLoss, token_log_probs
from vqa_amd.module_net import ModuleNet
from vqa_amd.sampling import sample

operators.own = True
DEV = torch.device('cuda:0')


def say(*a):
    print(*a, flush=True)


def passes(f, n=30, repeat=5):
    """us of a pass among others: whichever of host and device takes longer."""
    for _ in range(5):
        f()
    best = 1e9
    for _ in range(repeat):
        torch.cuda.synchronize()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / n)
    return best


def host(f, n=200, repeat=5):
    """us of host time of a call that does not wait for the device."""
    best = 1e9
    for _ in range(repeat):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(n):
            f()
        best = min(best, (time.perf_counter() - t) * 1e6 / n)
    return best


def replayed(f, n=10):
    """us of a call inside a captured graph of n of them: the device's time."""
    for _ in range(3):
        f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(n):
            f()
    return passes(graph.replay, 1, 8) / n


class Empty(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, dy):
        return dy


def rates():
    a = torch.empty(2 ** 28, dtype=torch.bfloat16, device=DEV)
    b = torch.empty_like(a)
    for what, f in (("torch's copy", lambda: b.copy_(a)), ('vqa_dropout', lambda: ops.dropout(a, b, 6554, 1, 2))):
        us = passes(f, 10)
        say('%s, 512 MiB read and 512 MiB written: %.0f us, %.2f TB/s' % (what, us, 2 ** 30 / us / 1e6))


def host_times():
    x = torch.zeros(1024, 44, device=DEV, requires_grad=True)
    dy, u, out = torch.zeros(1024, 44, device=DEV), torch.rand(1024, device=DEV), torch.zeros(1024, dtype=torch.int64, device=DEV)
    tk = torch.zeros(1024, dtype=torch.int64, device=DEV)
    g = torch.zeros(1024, device=DEV)

    def round_trip(f, dy):
        def go():
            x.grad = None
            f(x).backward(dy)
        return host(go)
    d = x.detach()
    say('sample(), 1024 x 44 fp32, into a column: %.1f' % host(lambda: sample(d, u, out=out)))
    say('an empty autograd.Function, forward and backward: %.1f' % round_trip(Empty.apply, dy))
    say('x * 2, forward and backward: %.1f' % round_trip(lambda t: t * 2, dy))
    say('dropout(), forward and backward: %.1f' % round_trip(lambda t: dropout(t, 0.5, 1), dy))
    say('token_log_probs(), forward and backward: %.1f' % round_trip(lambda t: token_log_probs(t, tk), g))


def by_torch():
    for case in operators.listed():
        if case['op'] == 'sample':
            continue
        s = operators.prepare(case, 1)
        x = s['x']

        def go():
            x.grad = None
            if case['op'] == 'dropout':
                torch.nn.functional.dropout(x, case['p']).backward(s['dy'])
                return
            z = torch.log_softmax(x.float() / case['temperature'], -1)
            lp = z.gather(1, s['tokens'].clamp(min=0)[:, None])[:, 0]
            if s['h'] is None:
                lp.backward(s['g'])
            else:
                torch.autograd.backward((lp, -(z.exp() * z).sum(1)), (s['g'], s['h']))
        say('%s: here %.0f, torch %.0f' % (case['name'], passes(lambda: operators.run(s)), passes(go, 5)))
        del s, x


def single_precision():
    for case in (dict(op='logp', rows=2048, vocab=32768, dtype='fp32', entropy=True, temperature=1.0),
                 dict(op='logp', rows=4096, vocab=131072, dtype='fp32', entropy=False, temperature=1.0),
                 dict(op='dropout', rows=8192, cols=4096, dtype='fp32', p=0.1),
                 dict(op='dropout', rows=32768, cols=8192, dtype='fp32', p=0.2)):
        s = operators.prepare(case, 1)
        us = passes(lambda: operators.run(s))
        say('%s %d x %d: %.0f, %.2f TB/s of what it cannot do without' %
            (case['op'], case['rows'], case.get('vocab') or case['cols'], us, operators.work(case)['bytes'] / us / 1e6))
        del s


def rows_of(rows, V, dtype):
    g = torch.Generator(device=DEV).manual_seed(V + rows)
    x = torch.randn(rows, V, generator=g, device=DEV) * (torch.rand(rows, 1, generator=g, device=DEV) * 2.5 + 0.5)
    return x.to(dtype), torch.rand(rows, generator=g, device=DEV)


def sampler():
    for rows, V in ((512, 131072), (64, 131072), (1, 50001), (1024, 16000)):
        for dtype in (torch.bfloat16, torch.float32):
            x, u = rows_of(rows, V, dtype)
            out = torch.empty(rows, dtype=torch.int64, device=DEV)
            time_of = lambda x, **kw: replayed(lambda: sample(x, u, out=out, **kw))    # noqa: E731
            g = torch.Generator(device=DEV).manual_seed(1)
            few = (torch.randint(0, 40, x.shape, generator=g, device=DEV) * 0.25).to(dtype)
            late = x.clone()
            late[:, 12000:14500] += 40                                    # above all that the guess has looked at
            say('%d x %d %s: top-p 0.9 %.0f%s; 40 values %.0f; constant rows %.0f; top-k 50 %.0f, 900 %.0f, 2100 %.0f, 10000 %.0f' %
                (rows, V, str(dtype)[6:], time_of(x, top_p=0.9),
                 '; where its guess of the range fails %.0f' % time_of(late, top_p=0.9) if rows > 64 else '', time_of(few, top_p=0.9),
                 time_of(torch.zeros_like(x), top_p=0.9), *(time_of(x, top_k=k) for k in (50, 900, 2100, 10000))))
    for rows, V in ((1024, 44), (1024, 100), (1024, 2000)):
        for kw in (dict(), dict(top_k=10, top_p=0.9)):
            x, u = rows_of(rows, V, torch.float32)
            out = torch.empty(rows, dtype=torch.int64, device=DEV)
            say('%d x %d float32%s: %.1f' % (rows, V, ', top-k 10, top-p 0.9' if kw else '', replayed(lambda: sample(x, u, out=out, **kw))))


def executor():
    vocab = V.make_vocab()
    net = ModuleNet(False, vocab)
    net.load_state_dict(synth.synth_state_dict(17, vocab))
    net.to(DEV).train()
    x = torch.randn(1024, 1024, 14, 14, device=DEV).clamp_(min=0)
    prog = torch.from_numpy(synth.synth_programs(3000, 1024, vocab)).to(DEV)
    ans = torch.from_numpy(synth.synth_answers(0, 1024)).to(DEV)
    lf = CrossEntropyLoss()

    def step():
        net.zero_grad(set_to_none=True)
        lf(net(x, prog), ans).backward()
    for repeat in range(2):
        for p in (0.0, 0.5):
            net.hidden_dropout = p
            say('hidden_dropout %.1f: %.0f' % (p, passes(step, 10)))


if __name__ == '__main__':
    for title, f in (('Rates', rates), ('Host time of a call', host_times), ('With gradient, next to torch (log_softmax and gather; dropout)', by_torch),
                     ('fp32, with gradient', single_precision),
                     ('Sampler, device time of a call in a row of them (lists beyond 2048 tokens, or 1024 in 1024 x 16000, go to the '
                      'radix search)', sampler),
                     ('Executor, forward, cross-entropy and backward, batch 1024', executor)):
        say('== ' + title)
        f()
