"""Refusals and page bookkeeping of prefixes held as codes, on the CPU."""
import pytest
import torch

from embodied_efficiency_b200 import ActionExpert, ActionExpertConfig
from embodied_efficiency_b200.expert import _prefix_pages
from embodied_efficiency_b200.fleet import FleetSampler


def test_pages_of_prefixes():
    cu = torch.tensor([0, 64, 65, 65, 195], dtype=torch.int32)
    pages, table, lens = _prefix_pages(cu, 195, 64)
    assert pages == 5 and lens.tolist() == [64, 1, 0, 130] and table.dtype == lens.dtype == torch.int32
    assert table.tolist() == [[0, -1, -1], [1, -1, -1], [-1, -1, -1], [2, 3, 4]]
    pages, table, lens = _prefix_pages(torch.zeros(1, dtype=torch.int32), 0, 64)
    assert pages == 0 and table.shape == (0, 0) and lens.numel() == 0
    pages, table, lens = _prefix_pages(torch.zeros(3, dtype=torch.int32), 0, 64)
    assert pages == 0 and table.shape == (2, 0) and lens.tolist() == [0, 0]


@pytest.mark.parametrize("cu", [[0, 5, 9], [1, 5, 10], [0, 11, 10], []])
def test_offsets_that_do_not_cover_the_rows(cu):
    with pytest.raises(ValueError, match="cu must"):
        _prefix_pages(torch.tensor(cu, dtype=torch.int32), 10, 64)


def test_refusals():
    m = ActionExpert(ActionExpertConfig(d_model=128, n_layers=1, n_heads=2, prefix_len=4))
    pre, cu = torch.zeros(4, 128), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="kv_bits"):
        m.encode_packed(pre, cu, kv_bits=16)
    with pytest.raises(ValueError, match="page_size"):
        m.encode_packed(pre, cu, kv_bits=8, page_size=48)
    with pytest.raises(ValueError, match="int32"):
        m.encode_packed(pre, cu.long(), kv_bits=8)
    with pytest.raises(ValueError, match="kv_bits"):
        FleetSampler(2, 0, 1, sample_fn=lambda p, x: x, kv_bits=8)
    with pytest.raises(ValueError, match="kv_bits"):
        FleetSampler(2, 0, 1, expert=m, kv_bits=5)
