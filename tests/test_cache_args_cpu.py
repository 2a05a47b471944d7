"""Indexes that pass 32 bits in calls on a KV cache; no GPU needed (a call that gets through ends at a null cache)."""
import pytest
import torch

from crispasr_b200 import abi


@pytest.mark.parametrize("bad", [1 << 32, -(1 << 32), (1 << 31), (1 << 63)])
def test_append_takes_no_index_by_its_low_half(b200, bad):
    """Layer 2^32 is not layer 0, row 2^32 not row 0."""
    x = torch.zeros(1, 1, 1, 64)
    with pytest.raises(OverflowError):
        b200.op._kv_append(0, bad, x, x, None, 0, 0)
    with pytest.raises(OverflowError):
        b200.op._kv_append(0, 0, x, x, None, bad, 0)


@pytest.mark.parametrize("index", [0, -1, (1 << 31) - 1, -(1 << 31)])
def test_append_hands_32_bit_indexes_on(b200, index):
    x = torch.zeros(1, 1, 1, 64)
    for layer, pos0 in ((index, 0), (0, index)):
        with pytest.raises(b200.B200Error) as e:
            b200.op._kv_append(0, layer, x, x, None, pos0, 0)
        assert e.value.code == abi.E_NULL
