"""Lengths outside the table, pools that cannot hold what is asked for: what a call leaves out stays as it was."""
import pytest
import torch

from smlm_b200 import paged
from test_gpu_paged import DEV

pytestmark = pytest.mark.gpu


def test_extend_by_more_pages_than_31_bits_count():
    """65535 rows that want 32769 pages each, 2.1e9 in all, of a pool that has them for one row."""
    rows, blocks = 65535, 32769
    table = torch.full((rows, blocks), -1, dtype=torch.int32, device=DEV)
    lengths = torch.zeros(rows, dtype=torch.int32, device=DEV)
    ref = torch.zeros(blocks + 5, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="no free page"):
        paged.pages_extend(table, lengths, ref, torch.arange(rows, dtype=torch.int32, device=DEV), blocks, 1)
    assert lengths[0] == blocks and not bool(lengths[1:].any())
    assert torch.equal(table[0], torch.arange(blocks, dtype=torch.int32, device=DEV))
    assert bool((table[1:] == -1).all()) and ref.tolist() == [1] * blocks + [0] * 5
