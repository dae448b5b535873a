"""PagedDecoder: the model over a paged cache gives what the growing cache gives, for prompts of different lengths in one
batch, forks, reorderings, windows with sinks, freed and compacted pages."""
import pytest
import torch

from smlm_b200.decode import GraphDecoder, PagedDecoder
from smlm_b200.model import ModelConfig, Transformer

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def model():
    cfg = ModelConfig(vocab_size=256, d_model=64, n_layers=4, n_heads=4, ffn_hidden=128, max_seq_len=96,
                      mem_layers=[1, 3], mem_n_keys=64, mem_heads=2, mem_knn=8, mem_k_dim=256,
                      mem_share_values=True, mem_value_grad="row_sparse")
    torch.manual_seed(0)
    return Transformer(cfg).to(DEV).eval()


def ids(n, seed):
    return torch.randint(0, 256, (1, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


def growing(m, prompt, fed):
    """The logits after the prompt and after every fed token, over the growing cache."""
    caches = [dict() for _ in range(m.cfg.n_layers)]
    with torch.no_grad():
        out = [m(prompt, kv_caches=caches, pos0=0)[:, -1]]
        for i, t in enumerate(fed):
            out.append(m(t.view(1, 1), kv_caches=caches, pos0=prompt.shape[1] + i)[:, -1])
    return torch.cat(out)


def close(a, b):
    # fp32 end to end, but the dense layers' products may run in another order for another batch
    torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-4)


def decode(dec, steps):
    """Greedy steps; the logits and the fed tokens of every row."""
    logits, fed = [], []
    for _ in range(steps):
        fed.append(dec.tokens.clone())
        dec.step()
        logits.append(dec.logits[:, 0].clone())
    return torch.stack(logits), torch.stack(fed)[:, :, 0]


@pytest.mark.parametrize("page", [1, 4, 16, 32])
def test_rows_of_different_lengths_match_the_growing_cache(model, page):
    dec = PagedDecoder(model, 4, page_size=page)
    prompts = {0: ids(11, 1), 2: ids(32, 2), 3: ids(1, 3)}         # row 1 stays idle
    first = {r: dec.prefill(p, [r])[:, -1].clone() for r, p in prompts.items()}
    logits, fed = decode(dec, 9)
    for r, p in prompts.items():
        want = growing(model, p, fed[:, r])
        close(first[r], want[:1])
        close(logits[:, r], want[1:])
        assert torch.equal(fed[1:, r], logits[:-1, r].argmax(-1))
    assert dec.cache.lengths.tolist() == [20, 0, 41, 10]


def test_same_as_the_static_cache_in_one_batch(model):
    prompt = torch.cat([ids(12, s) for s in range(3)])
    with torch.no_grad():
        a, b = PagedDecoder(model, 3, max_len=40), GraphDecoder(model, 3, max_len=40)
        close(a.prefill(prompt, range(3)), b.prefill(prompt))
        for _ in range(10):
            a.step()
            b.step()
            close(a.logits, b.logits)
    # fresh rows join and a chunk continues cached ones
    with torch.no_grad():
        a.free([1])
        more = ids(7, 9).expand(2, -1)
        got = a.prefill(more, [0, 2])
        caches = [dict() for _ in range(model.cfg.n_layers)]
        model(torch.cat((prompt[:1], ids(0, 0)), 1), kv_caches=caches)
    assert got.shape == (2, 7, 256) and a.cache.lengths.tolist() == [29, 0, 29]


def test_forked_continuations_share_the_prompt_and_diverge(model):
    dec = PagedDecoder(model, 5, page_size=8, n_pages=40)
    prompt = ids(29, 4)
    dec.prefill(prompt, [2])
    assert dec.cache.free_pages() == 40 - 4
    dec.fork(2, [0, 1, 4])
    assert dec.cache.free_pages() == 40 - 4 - 3                      # only the partly filled page is copied
    start = torch.tensor([[5], [6], [7], [0], [9]], device=DEV)
    dec.step(start)
    logits, fed = decode(dec, 12)
    fed = torch.cat((start.view(1, -1), fed))
    for r in (0, 1, 2, 4):
        close(logits[:, r], growing(model, prompt, fed[:, r])[2:])
    dec.free([0, 1, 2])
    dec.cache.compact()
    more, fed2 = decode(dec, 3)
    close(more[:, 4], growing(model, prompt, torch.cat((fed[:, 4], fed2[:, 4])))[-3:])
    assert dec.rows() == [4]


def test_reorder_as_a_beam_does(model):
    dec = PagedDecoder(model, 3, page_size=4)
    prompts = [ids(9, 10), ids(9, 11), ids(9, 12)]
    dec.prefill(torch.cat(prompts), range(3))
    _, fed = decode(dec, 3)
    history = [torch.cat((p[0], fed[:, r])) for r, p in enumerate(prompts)]
    dec.reorder([1, 1, 0])
    logits, fed = decode(dec, 4)
    for r, parent in enumerate([1, 1, 0]):
        close(logits[:, r], growing(model, history[parent].view(1, -1), fed[:, r])[1:])


@pytest.mark.parametrize("window,sinks", [(16, 0), (16, 3), (10, 20), (96, 4)])
def test_window_and_sinks(model, window, sinks):
    """Decoding with a window equals a full forward pass whose attention has that mask; pages outside it are released."""
    import torch.nn.functional as F
    dec = PagedDecoder(model, 2, page_size=4, window=window, sinks=sinks)
    prompt = ids(37, 6)
    first = dec.prefill(prompt, [1])
    logits, fed = decode(dec, 30)
    whole = torch.cat((prompt[0], fed[:, 1])).view(1, -1)
    n = whole.shape[1]
    t, j = torch.arange(n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
    seen = (j <= t) & ((j > t - window) | (j < sinks))
    plain = F.scaled_dot_product_attention
    F.scaled_dot_product_attention = lambda q, k, v, **kw: plain(q, k, v, attn_mask=seen)
    try:
        with torch.no_grad():
            want = model(whole)[0]
    finally:
        F.scaled_dot_product_attention = plain
    close(first[0], want[:37])
    close(logits[:, 1], want[37:])
    if window == 16:
        held = -(-sinks // 4) + -(-window // 4) + 2
        assert dec.cache.refcount.shape[0] - dec.cache.free_pages() <= held


def test_bf16_autocast_is_near_fp32_and_the_graph_replays_the_eager_step(model):
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        a, b = PagedDecoder(model, 2), PagedDecoder(model, 2)
        p = torch.cat((ids(20, 1), ids(20, 2)))
        torch.testing.assert_close(a.prefill(p, [0, 1]), b.prefill(p, [0, 1]), rtol=0, atol=0)
        for _ in range(6):
            a.step()
            b.cache.reserve([0, 1], 1)
            b._body()
            assert torch.equal(a.logits, b.logits) and torch.equal(a.tokens, b.tokens)
        assert a.cache.pool.dtype == torch.bfloat16


def test_running_out_of_pages_or_length_raises_before_a_launch(model):
    dec = PagedDecoder(model, 3, page_size=8, n_pages=5, max_len=32)
    dec.prefill(ids(16, 1), [0])
    with pytest.raises(RuntimeError, match="free"):
        dec.prefill(ids(30, 1), [1])
    assert dec.cache.lengths.tolist() == [16, 0, 0]
    dec.fork(0, [1, 2])                               # whole pages only: nothing is copied
    dec.step()
    assert dec.cache.free_pages() == 0
    for _ in range(7):
        dec.step()
    with pytest.raises(RuntimeError, match="free"):
        dec.step()
    dec.free([2])
    assert dec.cache.free_pages() == 1
    dec.free([1])
    for _ in range(8):
        dec.step()
    with pytest.raises(ValueError, match="max_len"):
        dec.step()
    with pytest.raises(ValueError, match="no sequence"):
        dec.free([0])
        dec.step()


def test_resize_keeps_the_sequences(model):
    dec = PagedDecoder(model, 2, page_size=4, n_pages=60)
    prompt = ids(21, 3)
    dec.prefill(prompt, [1])
    _, a = decode(dec, 3)
    dec.cache.resize(9)
    logits, b = decode(dec, 5)
    close(logits[:, 1], growing(model, prompt, torch.cat((a, b))[:, 1])[4:])
    with pytest.raises(ValueError, match="in use"):
        dec.cache.resize(3)
