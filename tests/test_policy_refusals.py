"""What the row operators refuse, and the generator's known answers; none of it needs a GPU."""
import ctypes as C
import math

import pytest
import torch

from philox_oracle import philox
from vqa_amd import _lib, dropout, loss, ops, sampling


def test_generator_known_answers():
    """Vectors published with the generator."""
    pi = [0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344]
    for ctr, key, want in (([0] * 4, [0] * 2, '6627e8d5 e169c58d bc57ac4c 9b00dbd8'),
                           ([2 ** 32 - 1] * 4, [2 ** 32 - 1] * 2, '408f276d 41c83b0e a20bc7c6 6d5451fd'),
                           (pi, [0xa4093822, 0x299f31d0], 'd16cfe09 94fdcceb 5001e420 24126ea1')):
        assert ' '.join('%08x' % int(v) for v in philox(ctr, key)) == want


def test_no_cpu_path():
    x = torch.zeros(2, 5)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        dropout.dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        loss.token_log_probs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        sampling.sample(x, torch.zeros(2))


def test_python_refusals():
    x, tk, u = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    for bad in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError):
            dropout.dropout(x, bad, 1)
        with pytest.raises(ValueError):
            dropout.Dropout(bad)
    with pytest.raises(ValueError):
        dropout.dropout(x.double(), 0.5, 1)
    for args in ((x.double(), tk), (x, tk.int()), (x, tk[:1]), (x[:, :0], tk), (torch.zeros(()), tk), (x, tk[:, None])):
        with pytest.raises(ValueError):
            loss.token_log_probs(*args)
    for t in (0.0, -1.0, math.nan, math.inf, 1e-9):
        with pytest.raises(ValueError):
            loss.token_log_probs(x, tk, temperature=t)
    for args in ((x.double(), u), (x[0], u), (x, u.double()), (x, u[:1]), (x[:, :0], u)):
        with pytest.raises(ValueError):
            sampling.sample(*args)
    for out in (torch.zeros(2), torch.zeros(3, dtype=torch.int64), torch.zeros(1, dtype=torch.int64).expand(2)):
        with pytest.raises(ValueError):
            sampling.sample(x, u, out=out)


def test_sampling_parameters():
    x = torch.zeros(2, 5)
    check = lambda name, v: sampling._per_row(name, v, 2, x.device)    # noqa: E731
    for name, bad in (('temperature', -1), ('temperature', math.nan), ('top_k', -1), ('top_p', 1.5), ('min_p', -0.1),
                      ('temperature', torch.ones(3)), ('top_k', torch.ones(2)), ('top_p', torch.ones(2, dtype=torch.int32)),
                      ('min_p', torch.ones(2, 1)), ('top_k', torch.ones(2, dtype=torch.bool))):
        with pytest.raises(ValueError):
            check(name, bad)
    assert check('top_k', torch.tensor([2 ** 40, 3])).tolist() == [2 ** 31 - 1, 3]
    assert check('top_p', torch.ones(2, dtype=torch.bfloat16)).dtype == torch.float32


def test_row_layouts():
    t = torch.arange(2 * 5 * 7, dtype=torch.float32).view(2, 5, 7)
    for v in (t, t[:, :-1], t[:, 1:, 2:5], t.permute(1, 0, 2), t.permute(2, 1, 0), t[0], t[0, 0], t[:1], t[:0], t[:, :, :1],
              t[0, :1].expand(3, 7), t.view(2, 5, 1, 7)[:, ::2].expand(2, 3, 4, 7)):
        x, rows, inner, ld_inner, ld_outer = ops.row_layout(v)
        flat, V = v.reshape(-1, v.size(-1)), v.size(-1)
        assert rows == flat.size(0)
        base = torch.as_strided(x, (x.untyped_storage().nbytes() // 4 - x.storage_offset(),), (1,), x.storage_offset())
        for r in range(rows):
            at = (r // inner) * ld_outer + (r % inner) * ld_inner
            assert torch.equal(base[at:at + V], flat[r])


def _refused(rc, who):
    lib = _lib.load()
    assert rc == 1 and lib.vqa_last_error().decode().startswith(who)


def test_c_entry_refusals():
    """Bad arguments come back as VQA_EINVAL with a message before anything is launched (the pointers below are never
    looked at)."""
    lib = _lib.load()
    p, odd = 0x1000, 0x1001
    bad = lambda *a: _refused(lib.vqa_dropout(*a, None), 'vqa_dropout')              # noqa: E731
    bad(None, p, 8, 0, 1, 0, 0, None)
    bad(p, None, 8, 0, 1, 0, 0, None)
    bad(p, p, -1, 0, 1, 0, 0, None)
    bad(p, p, 8, 3, 1, 0, 0, None)
    bad(p, p, 8, 0, -1, 0, 0, None)
    bad(p, p, 8, 0, 65537, 0, 0, None)
    bad(odd, p, 8, 0, 1, 0, 0, None)
    bad(p, p, 8, 0, 1, 0, 0, 0x1004)
    assert lib.vqa_dropout(None, None, 0, 0, 1, 0, 0, None, None) == 0

    good = [p, 1, 5, 5, p, p, None, p, None, 3, 5, 0, 1.0, -1]
    for i, v in ((0, None), (0, odd), (1, 0), (4, None), (4, 0x1004), (5, None), (7, None), (7, 0x1008), (9, -1), (10, 0), (11, 7),
                 (12, 0.0), (12, math.nan), (12, math.inf)):
        a = list(good)
        a[i] = v
        _refused(lib.vqa_token_logp(*a, None), 'vqa_token_logp')
    a = list(good)
    a[10] = 100000                                             # few long rows need a workspace
    assert lib.vqa_token_logp_workspace(3, 100000, 0) > 0
    _refused(lib.vqa_token_logp(*a, None), 'vqa_token_logp')
    good = [p, 1, 5, 5, p, p, p, None, p, 3, 5, 0, 1.0, -1]
    for i, v in ((0, None), (1, 0), (4, None), (5, None), (8, None), (8, odd), (9, -1), (10, 0), (11, -1), (12, -1.0)):
        a = list(good)
        a[i] = v
        _refused(lib.vqa_token_logp_backward(*a, None), 'vqa_token_logp_backward')

    def params(**kw):
        q = _lib.SampleParams()
        for k, v in dict(dict(logits=p, u=p, token=p, ld=5, ld_token=1, rows=3, V=5, dtype=2, temperature_value=1.0,
                              top_p_value=1.0), **kw).items():
            setattr(q, k, v)
        return C.byref(q)
    _refused(lib.vqa_sample(None, None), 'vqa_sample')
    for kw in (dict(logits=None), dict(u=None), dict(token=None), dict(rows=-1), dict(V=0), dict(V=2 ** 30 + 1), dict(dtype=3),
               dict(logits=0x1002), dict(token=0x1004), dict(u=0x1002), dict(top_k=0x1002), dict(logp=0x1001), dict(ld=-1)):
        _refused(lib.vqa_sample(params(**kw), None), 'vqa_sample')
    assert lib.vqa_sample_workspace(2, 100000) > 0 and lib.vqa_sample_workspace(1000, 100000) == 0
    _refused(lib.vqa_sample(params(rows=2, V=100000, ld=100000), None), 'vqa_sample')          # few long rows need a workspace
    assert lib.vqa_sample(params(rows=0, logits=None), None) == 0


def test_struct_matches_the_header():
    assert C.sizeof(_lib.SampleParams) == 9 * 8 + 3 * 8 + 3 * 8 + 4 * 4


def test_hidden_dropout_takes_its_counters_and_ranks_differ(vocab, monkeypatch):
    from vqa_amd.module_net import ModuleNet
    net = ModuleNet(False, vocab, feature_dim=(128, 14, 14), classifier_proj_dim=128, classifier_fc_layers=(256, 128))
    assert net._start_dropout(5) is None
    net.hidden_dropout, net.dropout_seed, net.dropout_offset = 0.25, 7, 10
    assert net._start_dropout(5) == (16384, 7, [10, 10 + 160])
    assert net.dropout_offset == 10 + 160 + 80
    monkeypatch.setattr(torch.distributed, 'is_initialized', lambda: True)
    monkeypatch.setattr(torch.distributed, 'get_rank', lambda: 3)
    assert net._start_dropout(5)[1] == 10
    net.eval()
    assert net._start_dropout(5) is None
    net.hidden_dropout = -0.1
    with pytest.raises(ValueError):
        net._start_dropout(5)


def test_hidden_dropout_is_refused_in_a_captured_graph(vocab, monkeypatch):
    from vqa_amd.module_net import ModuleNet
    net = ModuleNet(False, vocab, feature_dim=(128, 14, 14), classifier_proj_dim=128, classifier_fc_layers=(256, 128))
    monkeypatch.setattr(torch.cuda, 'is_available', lambda: True)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    assert net._start_dropout(5) is None
    net.hidden_dropout = 0.25
    with pytest.raises(RuntimeError, match='counts on the host'):
        net._start_dropout(5)
    assert net.dropout_offset == 0
    assert net.eval()._start_dropout(5) is None


def test_a_module_pickled_without_hidden_dropout_still_runs(vocab):
    import pickle

    from vqa_amd.module_net import ModuleNet
    net = ModuleNet(False, vocab, feature_dim=(128, 14, 14), classifier_proj_dim=128, classifier_fc_layers=(256, 128))
    for name in ('hidden_dropout', 'dropout_seed', 'dropout_offset'):
        net.__dict__.pop(name, None)
    net = pickle.loads(pickle.dumps(net))
    assert net._start_dropout(5) is None and net.dropout_offset == 0
    net.hidden_dropout = 0.5
    assert net._start_dropout(5) == (32768, 0, [0, 160])
