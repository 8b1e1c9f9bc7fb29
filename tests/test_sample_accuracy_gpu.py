"""Token sampling against exponentials in 64 bits that nothing has rounded.  A weight that the kernels sum as an integer is
rounded to 2^-s, s = min(51, 62 - ceil(log2 V)), so a sum is within V 2^-(s + 1), and 2^-42 of itself, of the sum of the
exponentials."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
# a wave a row, a list of all tokens, and bins: of 256, 512 and 1024 threads, with and without a guess of the range, split rows
SIZES = [(5, 44), (5, 64), (5, 65), (5, 100), (5, 128), (5, 300), (5, 9001), (300, 3000), (300, 20000), (5, 70000), (2, 131072),
         (300, 131072)]


def dev():
    return torch.device('cuda:0')


@pytest.mark.parametrize('rows,V', SIZES)
@pytest.mark.parametrize('scale', [0.5, 3.0])
def test_against_weights_that_are_not_rounded(rows, V, scale):
    """A number in the middle of a token's share draws it, and log-probabilities are off by the sums' error over the weight
    kept."""
    from vqa_amd.sampling import sample
    x = (torch.randn(1, V, generator=torch.Generator().manual_seed(V)) * scale)
    s = min(51, 62 - (V - 1).bit_length())
    z = x[0].double().numpy()
    order = np.argsort(-z, kind='stable')
    w = np.exp(z[order] - z.max())
    behind = np.cumsum(w)
    total = behind[-1]
    tol = V * 2.0 ** -(s + 1) + 2.0 ** -42 * total
    rank = np.unique(np.geomspace(1, V, 60).astype(int) - 1)
    u = np.float32((behind[rank] - w[rank] / 2) / total)
    t = u.astype(np.float64) * total
    sure = (t > behind[rank] - w[rank] + tol) & (t < behind[rank] - tol) & (u < 1)
    rank, u = rank[sure], u[sure]
    assert len(rank) >= 10
    reps = -(-len(rank) // rows)
    at = torch.from_numpy(np.resize(u, reps * rows)).to(dev())
    xs = x.to(dev()).expand(rows, V)
    for i in range(reps):
        tk, lp = sample(xs, at[i * rows:(i + 1) * rows], return_log_probs=True)
        want = np.resize(rank, reps * rows)[i * rows:(i + 1) * rows]
        assert np.array_equal(tk.cpu().numpy(), order[want])
        exact = np.log(w[want] / total)
        assert (np.abs(lp.double().cpu().numpy() - exact) <= np.abs(exact) * 2.0 ** -24 + 2 * tol / total + 1e-12).all()
