"""PagedKVCache, its views and PagedDecoder between steps."""
import ctypes
import math

import pytest
import torch

from smlm_b200 import _lib as L
from smlm_b200 import engram, paged
from smlm_b200.decode import PagedDecoder
from smlm_b200.model import ModelConfig, Transformer
from test_gpu_paged import BF16, DEV, F32, make
from test_gpu_paged_decode import close, growing, ids, model  # noqa: F401

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


def test_a_reordering_in_a_full_pool_that_frees_the_pages_it_needs(model):
    """All 3 x 8 pages are in use. [1, 1, 0] drops row 2's eight pages and copies two partly filled ones: the device
    completes that, so it must not be refused; one that needs more than is dropped still is."""
    dec = PagedDecoder(model, 3, page_size=4, max_len=32)
    prompts = [ids(30, s) for s in (20, 21, 22)]
    dec.prefill(torch.cat(prompts), range(3))
    assert dec.cache.free_pages() == 0
    dec.reorder([1, 1, 0])
    fed = dec.tokens.clone()
    dec.step()
    for r, p in enumerate([1, 1, 0]):
        close(dec.logits[r], growing(model, prompts[p], fed[r].view(1))[1:])
    cache = paged.PagedKVCache(1, 4, 4, 1, 16, 4, 16, F32, DEV)
    cache.extend([0], 6)
    cache.extend([1, 2], 3)
    with pytest.raises(RuntimeError, match="pages needed"):
        cache.fork([0, 0], [1, 3])                    # frees one page, needs two
    assert cache.lengths.tolist() == [6, 3, 3, 0] and cache.table.tolist()[1:] == [[2, -1, -1, -1], [3, -1, -1, -1],
                                                                                  [-1] * 4]
    cache.fork([0], [1])                              # frees one, needs one
    assert cache.lengths.tolist() == [6, 6, 3, 0] and cache.table.tolist()[:2] == [[0, 1, -1, -1], [0, 2, -1, -1]]


def test_logits_follow_prefills_forks_and_reorderings(model):
    """Sampling from dec.logits works after every call, on a decoder that has already stepped: row r of the logits belongs
    to the sequence that row r holds."""
    dec = PagedDecoder(model, 4, page_size=4)
    history = {}

    def prefill(row, n, seed):
        p = ids(n, seed)
        got = dec.prefill(p, [row])
        history[row] = p
        assert torch.equal(dec.logits[row, 0], got[0, -1])

    def agree():
        for r, h in history.items():
            with torch.no_grad():
                close(dec.logits[r], model(h)[0, -1:])
            assert int(dec.tokens[r]) == int(dec.logits[r, 0].argmax())

    def step():
        second = dec.logits[:, 0].topk(2).indices[:, 1:]               # the second best token of every row
        dec.step(second)
        for r in history:
            history[r] = torch.cat((history[r], second[r:r + 1]), 1)
        agree()

    prefill(0, 9, 1)
    step()
    prefill(2, 13, 2)                  # a row joins one that has stepped
    agree()
    step()
    dec.fork(0, [1, 3])
    history[1] = history[3] = history[0]
    agree()
    step()
    dec.reorder([2, 0, 1, 1])
    history = {0: history[2], 1: history[0], 2: history[1], 3: history[1]}
    agree()
    step()
    dec.free([1])
    del history[1]
    prefill(1, 5, 3)
    agree()
    step()


def test_steps_in_inference_mode_and_forks_outside(model):
    dec = PagedDecoder(model, 2, page_size=4)
    with torch.inference_mode():
        dec.prefill(ids(7, 1), [0])
        dec.step()
    dec.fork(0, [1])
    assert torch.equal(dec.logits[0], dec.logits[1]) and not dec.logits.is_inference()
    with torch.inference_mode():
        dec.step()
    assert torch.equal(dec.tokens[0], dec.tokens[1])


def test_a_backward_pass_through_the_paged_calls_raises(model):
    """Forward passes without no_grad work as before; their backward says that there is no gradient."""
    cache = paged.PagedKVCache.for_model(model, 2, page_size=4, dtype=F32)
    cache.extend([0, 1], 5)
    x = ids(5, 1).expand(2, -1)
    with torch.no_grad():
        want = model(x, kv_caches=cache.view([0, 1]).caches())
    out = model(x, kv_caches=cache.view([0, 1]).caches())
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="paged_append has no gradient"):
        out.sum().backward()
    model.zero_grad(set_to_none=True)
    q, k, v, table, lengths = make([9], 2, 2, 32, 16, F32)
    q.requires_grad_()
    for outs in (paged.paged_attention(q, k, v, table, lengths, return_lse=True),
                 (paged.paged_attention(q * 2, k, v, table, lengths),)):
        for o in outs:
            with pytest.raises(RuntimeError, match="paged_attention has no gradient"):
                o.sum().backward()
    assert q.grad is None
    qkv = torch.randn(1, 1, 6 * 32, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="paged_append has no gradient"):
        paged.paged_append(qkv, k, v, table, lengths).sum().backward()
    with torch.no_grad():
        assert not paged.paged_attention(q, k, v, table, lengths).requires_grad
        assert not paged.paged_append(qkv, k, v, table, lengths).requires_grad
    assert not paged.paged_attention(q.detach(), k, v, table, lengths).requires_grad
    # keys and values with a gradient of their own
    with pytest.raises(RuntimeError, match="paged_attention has no gradient"):
        paged.paged_attention(q.detach(), k, v.clone().requires_grad_(), table, lengths).sum().backward()


def kernels_of(fn):
    """How many kernels the call launches: the nodes of its captured graph."""
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        fn()
    n = ctypes.c_size_t()
    rc = ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n))
    assert rc == 0
    return n.value


@pytest.mark.parametrize("n,batch,launches", [(64, 1, 1), (3000, 40, 2)])
def test_the_launches_counted_are_those_made(n, batch, launches):
    """One launch where a cluster takes an item, two with the list and its join."""
    q, k, v, table, lengths = make([n] * batch, 6, 6, 64, 16, BF16, stale=0.0)
    call = lambda: paged.paged_attention(q, k, v, table, lengths)  # noqa: E731
    call()
    assert kernels_of(call) == launches
    L.PROFILE = []
    try:
        call()
        counted = [x[3] for x in L.PROFILE]
    finally:
        L.PROFILE = None
    assert counted == [launches]


def test_engram_memories_over_a_paged_cache_see_their_history_or_are_refused(monkeypatch):
    """The n-gram history of a paged sequence is not kept: a pass over whole sequences needs none, a later one is refused
    (it would look up n-grams of padding)."""
    # token compression needs the GPT-2 vocabulary, which is not reachable offline
    monkeypatch.setattr(engram, "canonical_ids", lambda vocab: (torch.arange(vocab, dtype=torch.int64), vocab))
    torch.manual_seed(3)
    m = Transformer(ModelConfig(vocab_size=512, d_model=64, n_layers=2, n_heads=4, ffn_hidden=128, max_seq_len=96,
                                mem_layers=[], eng_layers=[1], eng_heads=2, eng_head_dim=8, eng_rows=101)).to(DEV).eval()
    cache = paged.PagedKVCache.for_model(m, 1, page_size=4, dtype=F32)
    x = ids(9, 1)
    with torch.no_grad():
        cache.extend([0], 9)
        close(m(x, kv_caches=cache.view([0]).caches()), m(x))
        cache.extend([0], 1)
        with pytest.raises(ValueError, match="Engram"):
            m(x[:, :1], kv_caches=cache.view([0]).caches())
        with pytest.raises(ValueError, match="Engram"):
            m(x[:, :1], kv_caches=cache.view().caches())
