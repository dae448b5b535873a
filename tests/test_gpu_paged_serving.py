"""PagedKVCache, its views and PagedDecoder between steps."""
import math

import pytest
import torch

from smlm_b200 import paged
from smlm_b200.decode import PagedDecoder
from smlm_b200.model import ModelConfig, Transformer
from test_gpu_paged import DEV, F32
from test_gpu_paged_decode import ids

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dense():
    """A model without memory layers."""
    torch.manual_seed(1)
    return Transformer(ModelConfig(vocab_size=256, d_model=64, n_layers=2, n_heads=4, ffn_hidden=128, max_seq_len=96,
                                   mem_layers=[])).to(DEV).eval()


def test_a_chunk_after_trimmed_pages_reads_no_other_sequence(dense):
    """Page 0 belongs to a sequence whose keys and values are infinite and NaN; a chunk prefilled into a sequence that has
    released pages to its window does not see it."""
    outs = []
    for bad in (0.0, math.nan, math.inf):
        dec = PagedDecoder(dense, 2, page_size=4, window=8, sinks=2)
        dec.prefill(ids(4, 1), [0])
        dec.prefill(ids(24, 2), [1])
        assert int(dec.cache.table[0, 0]) == 0 and -1 in dec.cache.table[1, :6].tolist()
        dec.cache.pool[:, :, 0] = bad
        outs.append(dec.prefill(ids(6, 3), [1]))
    assert bool(outs[0].isfinite().all())
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_a_pass_of_several_tokens_over_the_view_of_all_rows_writes_nothing(dense):
    cache = paged.PagedKVCache.for_model(dense, 2, page_size=4, dtype=F32)
    cache.extend([0, 1], 5)
    cache.pool.fill_(2.0)
    with torch.no_grad():
        with pytest.raises(ValueError, match="several tokens"):
            dense(ids(3, 1).expand(2, -1), kv_caches=cache.view().caches())
        assert bool((cache.pool == 2.0).all())
        assert dense(ids(5, 1).expand(2, -1), kv_caches=cache.view([0, 1]).caches()).shape == (2, 5, 256)


def test_extending_by_less_than_nothing_changes_nothing():
    cache = paged.PagedKVCache(1, 4, 4, 1, 16, 2, 16, F32, DEV)
    cache.extend([0], 6)
    with pytest.raises(ValueError, match="-5"):
        cache.extend([0], -5)
    assert cache.length(0) == 6 and cache.free_pages() == 2 and cache.lengths.tolist() == [6, 0]
    cache.extend([0], 0)
    assert cache.length(0) == 6 and cache.lengths.tolist() == [6, 0]
