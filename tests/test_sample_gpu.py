"""Token sampling (vqa_amd.sampling over vqa_sample) against its definition: a sorted row, weights in 64 bits rounded to
2^-s, and sums of Python integers.  Tokens have to be equal; a log-probability is off by at most half a step of fp32 and the
64-bit roundings behind it (1e-12)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def dev():
    return torch.device('cuda:0')


def draw_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log-probability) of one row, x float64 numpy."""
    x = np.where(np.isnan(x), -np.inf, x)
    V = len(x)
    if x.max() == -np.inf:
        return -1, -math.inf
    order = np.argsort(-x, kind='stable')
    if not temperature > 0:
        return int(order[0]), 0.0
    s = min(51, 62 - (V - 1).bit_length())
    with np.errstate(invalid='ignore'):
        z = np.where(x == x.max(), 0.0, (x - x.max()) / temperature)[order]
    live = x[order] > -np.inf
    e = np.where(live, np.exp(z), 0.0)
    if min_p > 0:
        live &= z >= math.log(min(min_p, 1.0))     # (as logarithms: exp rounds to 1 next to 0)
    n = int(live.sum())
    w = [int(v) for v in np.rint(e[:n] * 2.0 ** s)]
    if top_k > 0:
        w = w[:top_k]
    if not top_p >= 1:
        end, acc, kept = max(1, math.ceil(top_p * float(sum(w)))) if top_p > 0 else 1, 0, 0
        while kept < len(w) and acc < end:
            acc += w[kept]
            kept += 1
        w = w[:kept]
    total = sum(w)
    t = min(int(min(u, 2.0) * float(total)), total - 1) if u > 0 else 0
    acc = 0
    for i, wi in enumerate(w):
        acc += wi
        if acc > t:
            return int(order[i]), float(z[i] - math.log(total) + s * math.log(2.0))
    raise AssertionError


def check(x, u, **params):
    from vqa_amd.sampling import sample
    as_dev = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in params.items()}
    tk, lp = sample(x, u.to(dev()), return_log_probs=True, **as_dev)
    assert tk.dtype == torch.int64 and lp.dtype == torch.float32 and tk.shape == lp.shape == (x.size(0),)
    assert torch.equal(tk, sample(x, u.to(dev()), **as_dev))
    xs, tk, lp = x.double().cpu().numpy(), tk.tolist(), lp.tolist()
    for r in range(x.size(0)):
        par = {k: v[r].item() if isinstance(v, torch.Tensor) else v for k, v in params.items()}
        token, logp = draw_row(xs[r], u[r].item(), **par)
        assert tk[r] == token, (r, tk[r], token, par)
        assert lp[r] == logp or abs(lp[r] - logp) <= abs(logp) * 2.0 ** -24 + 1e-12, (r, lp[r], logp)


def logits(rows, V, seed, dtype, scale=3.0):
    return (torch.randn(rows, V, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(dev())


def uniform(rows, seed):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed))


SIZES = [(3, 1), (5, 2), (40, 44), (9, 64), (9, 65), (7, 100), (7, 128), (7, 129), (6, 300), (5, 1023), (5, 2049), (4, 8192), (4, 8193), (3, 50001), (2, 131072)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,V', SIZES)
def test_no_filter(dtype, rows, V):
    check(logits(rows, V, V, dtype), uniform(rows, V))
    check(logits(rows, V, V, dtype, 0.01), uniform(rows, V + 1), temperature=0.7)       # flat: many ties in 16 bits


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,V', SIZES)
@pytest.mark.parametrize('params', [dict(top_k=1), dict(top_k=7), dict(top_p=0.9), dict(top_p=0.3, top_k=40), dict(min_p=0.05),
                                    dict(min_p=0.001, top_p=0.95, top_k=300, temperature=1.4)],
                         ids=['k1', 'k7', 'p.9', 'p.3k40', 'minp', 'all'])
def test_filters(dtype, rows, V, params):
    check(logits(rows, V, V + 5, dtype), uniform(rows, V), **params)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V', [44, 700, 9000, 83000])
def test_every_row_its_own_parameters(dtype, V):
    rows = 48
    g = torch.Generator().manual_seed(V)
    pick = lambda: torch.rand(rows, generator=g)                       # noqa: E731
    check(logits(rows, V, V, dtype), pick(), temperature=(pick() * 2).masked_fill(pick() < 0.2, 0.0),
          top_k=torch.randint(0, V + 5, (rows,), generator=g, dtype=torch.int32).masked_fill(pick() < 0.3, 0),
          top_p=(pick() * 1.2).clamp(max=1.0), min_p=(pick() * 0.3 - 0.1).clamp(min=0.0))


@pytest.mark.parametrize('V', [44, 700, 9000])
def test_parameters_outside_their_range_in_a_tensor(V):
    f = lambda *v: torch.tensor(v, dtype=torch.float32)                # noqa: E731
    x = logits(6, V, 3, torch.float32)
    u = torch.full((6,), 0.6)
    check(x, u, temperature=f(-1, math.nan, math.inf, 1e-30, 1, 0))
    check(x, u, top_k=torch.tensor([-5, 0, 1, V, V + 1, 2 ** 31 - 1], dtype=torch.int32))
    check(x, u, top_p=f(-1, 0, math.nan, 2, 1, 1e-30))
    check(x, u, min_p=f(-1, 0, math.nan, 2, 1, 1e-38))
    check(x, f(-0.5, math.nan, 1.0, 7.0, math.inf, 0.0))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V', [44, 64, 100, 300, 9001, 50009])
def test_masks_infinities_and_nan(dtype, V):
    x = logits(12, V, V, dtype)
    x[0, :] = -math.inf
    x[1, :] = math.nan
    x[2, 1:] = -math.inf
    x[3, ::2] = math.nan
    x[4, ::3] = torch.finfo(dtype).min
    x[5, :] = torch.finfo(dtype).min
    x[6, V // 2] = math.inf
    x[7, 3::5] = math.inf
    x[8, :] = 0.0
    x[8, ::2] = -0.0                            # equal to +0: the index alone decides
    x[9, : V - 1] = -math.inf
    x[10, :] = torch.finfo(dtype).max
    for u in (0.0, 0.37, 1 - 2.0 ** -24):
        for params in (dict(), dict(temperature=0.5, top_k=3), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=0.0)):
            check(x, torch.full((12,), u), **params)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V', [50, 1000, 10000, 40000])
def test_ties_go_by_index(dtype, V):
    """Constant rows and rows of two values: the cut of top-k and top-p falls among equals."""
    x = torch.zeros(4, V, dtype=dtype, device=dev())
    x[1, V // 3:] = 1.0
    x[2, ::2] = 1.0
    x[3, 1::3] = -2.0
    from vqa_amd.sampling import sample
    for u in (0.0, 0.25, 0.5, 0.999):
        for params in (dict(), dict(top_k=5), dict(top_k=V - 2), dict(top_p=0.5), dict(top_p=0.37, top_k=V // 2)):
            check(x, torch.full((4,), u), **params)
            # and in a batch of more rows, which other kernels do
            us = torch.full((300,), u, device=dev())
            many = sample(x.repeat(75, 1), us, **params)
            assert torch.equal(many.view(75, 4), sample(x, us[:4], **params).expand(75, 4))


def test_frequencies_over_all_numbers():
    """One row under 4096 evenly spaced numbers (a broadcast row): a token is drawn as often as its weight says, to one."""
    from vqa_amd.sampling import sample
    for V in (44, 777):
        x = logits(1, V, V, torch.float32, 1.5)
        n = 4096
        tk = sample(x.expand(n, V), ((torch.arange(n) + 0.5) / n).to(dev()))
        got = torch.bincount(tk, minlength=V).double().cpu()
        want = torch.softmax(x[0].double().cpu(), 0) * n
        assert ((got - want).abs() <= 1 + 1e-6).all()


def test_strides_columns_and_what_is_behind_them():
    from vqa_amd.sampling import sample
    big = logits(4 * 7, 333, 5, torch.bfloat16).view(4, 7, 333)
    u = uniform(4, 5)
    check(big[:, 3], u)                          # the last step of a [N, T, V] tensor
    check(big[:, 3, 5:50], u)                    # rows that start at odd elements
    check(big[0, :4].t()[:100, :], uniform(100, 2))      # columns: copied
    programs = torch.full((4, 30), -7, dtype=torch.int64, device=dev())
    got = sample(big[:, 3], u.to(dev()), out=programs[:, 4])
    assert got.data_ptr() == programs[:, 4].data_ptr()
    assert torch.equal(programs[:, 4], sample(big[:, 3], u.to(dev())))
    programs[:, 4] = -7
    assert (programs == -7).all()
    assert sample(big[:0, 3], u[:0].to(dev())).shape == (0,)


def test_more_rows_than_workgroups():
    """The launch has at most 65536 workgroups of 4 rows: the rest comes in a second round."""
    from vqa_amd.sampling import sample
    rows = 4 * 65536 + 9
    x = logits(64, 4, 1, torch.float32).repeat(rows // 64 + 1, 1)[:rows]
    u = uniform(64, 3).repeat(rows // 64 + 1)[:rows].to(dev())
    tk = sample(x, u)
    assert torch.equal(tk[64:], tk[:64].repeat(rows // 64 + 1)[:rows][64:])
    check(x[:64], u[:64].cpu())


@pytest.mark.parametrize('V', [2000, 12000, 20000, 100003])
def test_the_same_row_in_batches_of_every_size(V):
    """How many rows a call has decides how a row is split and by how many threads it is done: the answers agree."""
    from vqa_amd.sampling import sample
    x = logits(300, V, V, torch.float32)
    u = uniform(300, V).to(dev())
    for params in (dict(top_p=0.9), dict(top_k=30), dict(temperature=0.5)):
        want = sample(x, u, return_log_probs=True, **params)
        for n in (1, 64, 65, 256):
            got = sample(x[:n], u[:n], return_log_probs=True, **params)
            assert torch.equal(got[0], want[0][:n])
            assert ((got[1] - want[1][:n]).abs() <= want[1][:n].abs() * 2.0 ** -23).all()


def test_another_stream_and_a_captured_graph():
    from vqa_amd.sampling import sample
    for V in (44, 5000, 20000, 70000):
        x = logits(6, V, V, torch.float32)
        u = uniform(6, V).to(dev())
        want = sample(x, u, top_p=0.8, return_log_probs=True)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = sample(x, u, top_p=0.8, return_log_probs=True)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = sample(x, u, top_p=0.8, return_log_probs=True)
        for k in range(3):
            u.copy_(uniform(6, V + k))
            graph.replay()
            torch.cuda.synchronize()
            want = sample(x, u, top_p=0.8, return_log_probs=True)
            assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_lone_token_has_log_probability_zero():
    from vqa_amd.sampling import sample
    for V in (2, 44, 700, 9000):
        x = torch.full((3, V), -math.inf, device=dev())
        x[:, V - 1] = torch.tensor([0.3, -7.0, 1e30], device=dev())
        tk, lp = sample(x, uniform(3, 1).to(dev()), temperature=0.7, top_p=0.9, return_log_probs=True)
        assert tk.tolist() == [V - 1] * 3 and lp.tolist() == [0.0] * 3
        x[:, 0] = x[:, V - 1]
        tk, lp = sample(x, uniform(3, 1).to(dev()), top_k=1, return_log_probs=True)
        assert tk.tolist() == [0] * 3 and lp.tolist() == [0.0] * 3


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V', [1025, 5000, 30011, 50021])
def test_lists_of_every_length(dtype, V):
    """Around the capacity of the list of candidates (2048): top-k beyond it, many equal logits at the cut, a bin edge that
    falls on 0 (symmetric rows), rows far from 0, tiny and huge spreads."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(11, V, generator=g) * 2
    x[1] = torch.linspace(-10, 10, V)
    x[2] = torch.randint(0, 3, (V,), generator=g).float()
    x[3] = torch.randint(0, 40, (V,), generator=g) * 0.25
    x[4] = 1000 + x[4]
    x[5] = x[5] * 1e-4
    x[6] = x[6] * 1e3
    x[7, : V // 2] = 5.0
    x[8] = torch.linspace(-1e-30, 1e-30, V)
    x[9, 0] = -1e30
    x[10] = torch.arange(V) * 1e-43 - 3e-41          # subnormal numbers (zeros in fp16)
    x = x.to(dtype).to(dev())
    for params in (dict(), dict(top_k=2000), dict(top_k=2048), dict(top_k=2049, top_p=0.9), dict(top_p=0.7),
                   dict(top_p=0.999, min_p=0.01), dict(min_p=1.0), dict(temperature=0.01, top_p=0.9), dict(temperature=100.0)):
        for u in (0.0, 0.4, 0.93, 1 - 2.0 ** -24):
            check(x, torch.full((11,), u), **params)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('V', [8192, 20011])
def test_rows_whose_parts_differ(dtype, V):
    """Long rows are laid out by what a sixteenth of them shows: rows that rise or fall, whose front is masked, constant or
    narrow, with a few or many tokens above and below everything in front of them."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(14, V, generator=g) * 2
    end = slice(V - 2500, V)
    x[0] = torch.linspace(-9, 9, V)
    x[1] = torch.linspace(9, -9, V)
    x[2, : V - 3000] = -math.inf
    x[3, : V - 3000] = 1.0
    x[4, V - 40: V - 37] = torch.tensor([14.0, 15.0, 16.0])
    x[5, V - 40: V - 30] = -16.0
    x[6, V - 3] = math.inf
    x[7, end] = math.nan
    x[8, end] = 11.0
    x[9, V - 5] = 60.0
    x[10, : V - 3000] *= 1e-3
    x[11, end] = -12.0
    x[12, V - 700: V - 100] = 10 + torch.rand(600, generator=g) * 3
    x[13, V - 30: V - 10] = -3000.0
    x = x.to(dtype).to(dev())
    for params in (dict(), dict(top_k=1), dict(top_k=30), dict(top_k=1500), dict(top_p=0.9), dict(top_p=0.2), dict(top_p=0.9999),
                   dict(temperature=0.05, top_p=0.9), dict(temperature=20.0), dict(min_p=0.01), dict(temperature=0.0)):
        for u in (0.0, 0.3, 0.8, 1 - 2.0 ** -24):
            check(x, torch.full((14,), u), **params)


@pytest.mark.parametrize('V', [44, 100, 700, 12000, 70000])
def test_the_smallest_temperatures(V):
    """Down to numbers whose reciprocal is infinite: the largest logits share all the weight."""
    x = logits(6, V, V, torch.float32)
    x[1, 3:9] = x[1].max()
    x[2, ::2] = 40.0
    x[3] = torch.arange(V, device=dev()) * 1e-45
    for t in (5e-324, 1e-310, 1e-290, 1e-45):
        for params in (dict(), dict(top_p=0.6), dict(top_k=3), dict(min_p=0.1)):
            check(x, uniform(6, V), temperature=t, **params)


@pytest.mark.parametrize('rows,V', [(300, 3000), (300, 20000), (4, 20000), (4, 70000)])
def test_lists_around_the_lengths_of_sorted_runs(rows, V):
    """Top-k lists of one to thirty-two runs of 64 and a few more, in the kernels of 256, 512 and 1024 threads and in split
    rows; u all over [0, 1), so that every part of the sorted list is looked up."""
    from vqa_amd.sampling import sample
    g = torch.Generator().manual_seed(V + rows)
    x = torch.randn(4, V, generator=g) * 0.7
    x[1] = torch.randperm(V, generator=g) * 1e-4                       # no ties
    x[2] = torch.randint(0, 400, (V,), generator=g) * 0.01             # many
    x = x.to(dev()).repeat(rows // 4, 1)
    u = torch.tensor([0.0, 0.25, 0.5, 0.999]).repeat(rows // 4)
    for k in (63, 65, 128, 129, 255, 256, 257, 320, 511, 512, 513, 577, 1023, 1024, 1025, 1100, 1500, 1999):
        for shift in range(4):
            at = u.roll(shift)
            tk, lp = sample(x, at.to(dev()), top_k=k, return_log_probs=True)
            for r in range(4):
                want, logp = draw_row(x[r].double().cpu().numpy(), float(at[r]), top_k=k)
                assert tk[r].item() == want, (k, r, shift)
                assert abs(lp[r].item() - logp) <= abs(logp) * 2.0 ** -24 + 1e-12
