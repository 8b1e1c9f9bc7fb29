"""Per-row sampling parameters of every type: what the kernel gets to read.  None of it needs a GPU."""
import pytest
import torch

from vqa_amd import sampling


def check(name, v):
    return sampling._per_row(name, v, 2, torch.device('cpu'))


@pytest.mark.parametrize('dtype', [torch.int8, torch.uint8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64,
                                   torch.uint64])
def test_top_k_of_every_integer_type(dtype):
    """Values beyond 32 bits are as good as the largest one, or as none (0): no vocabulary is that large."""
    most = torch.iinfo(dtype).max
    got = check('top_k', torch.tensor([3, most], dtype=dtype))
    assert got.dtype == torch.int32 and got[0] == 3
    assert got[1] == min(most, 2 ** 31 - 1) or (most > 2 ** 31 and got[1] <= 0)
    if most > 2 ** 33:
        assert check('top_k', torch.tensor([2 ** 32 + 3, 2 ** 31], dtype=dtype)).tolist() == [2 ** 31 - 1] * 2


def test_complex_numbers_are_refused():
    for name in ('temperature', 'top_k', 'top_p', 'min_p'):
        with pytest.raises(ValueError):
            check(name, torch.ones(2, dtype=torch.complex64))
