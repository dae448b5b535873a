"""Lengths outside the table, pools that cannot hold what is asked for: what a call leaves out stays as it was."""
import math

import pytest
import torch

import paged_ref as R
from smlm_b200 import _lib as L
from smlm_b200 import paged
from test_gpu_paged import BF16, DEV, F32, make, roomy

pytestmark = pytest.mark.gpu


def unchecked(monkeypatch):
    """Calls return although flags are raised, as they do in use."""
    monkeypatch.setenv("SMLM_B200_CHECK", "0")


def flags():
    torch.cuda.synchronize()
    return L.read_status(torch.device(DEV, torch.cuda.current_device()))


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


@pytest.mark.parametrize("bad", [10 ** 6, 49, -1, -10 ** 6])
@pytest.mark.parametrize("tokens", [1, 5])
def test_append_leaves_out_rows_whose_length_is_outside_the_table(monkeypatch, bad, tokens):
    """The table has room for 48 tokens: a row of 49 is left out whole, with queries of 0."""
    unchecked(monkeypatch)
    _, k, v, table, lengths = make([20, 30], 4, 2, 32, 16, BF16, stale=1.0)
    table[0] = table[0].clamp(min=0)                      # every entry is a page
    lengths[0] = bad
    qkv = torch.randn(2, tokens, 8 * 32, device=DEV).to(BF16)
    cos, sin = (x.to(DEV) for x in R.rotary(32, 64))
    ok = torch.tensor([0, 30], dtype=torch.int32, device=DEV)
    rq, rk, rv = R.append(qkv, k, v, table, ok, cos, sin)
    flags()
    q = paged.paged_append(qkv, k, v, table, lengths, cos, sin)
    assert flags() & L.FLAG_INDEX_RANGE
    assert not bool(q[0].any()) and bool(q[1].any())
    for got, ref in ((k, rk), (v, rv)):
        assert bool(((got.double().cpu() - ref).abs() <= 2.0 ** -7 * ref.abs() + 2.0 ** -20).all())


@pytest.mark.parametrize("bad", [10 ** 6, 49, -1])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("window", [0, 10])
def test_attention_leaves_out_rows_whose_length_is_outside_the_table(monkeypatch, bad, dtype, room, window):
    unchecked(monkeypatch)
    q, k, v, table, lengths = make([20, 30, 3], 4, 2, 32, 16, dtype, stale=1.0)
    if room:
        table = roomy(table, 16)
        bad = bad if bad < 49 else 100000 // 16 * 16 + 1
    want, wlse = paged.paged_attention(q, k, v, table, lengths, window=window, return_lse=True)
    lengths[0] = bad
    flags()
    out, lse = paged.paged_attention(q, k, v, table, lengths, window=window, return_lse=True)
    assert flags() & L.FLAG_INDEX_RANGE
    assert not bool(out[0].any()) and bool((lse[0] == -math.inf).all())
    # (the work is cut by the lengths, so the other rows' sums may be split elsewhere)
    torch.testing.assert_close(out[1:].float(), want[1:].float(), rtol=2.0 ** -7, atol=1e-5)
    torch.testing.assert_close(lse[1:], wlse[1:], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("bad", [25, 10 ** 9, -1])
def test_fork_and_trim_leave_out_rows_whose_length_is_outside_the_table(monkeypatch, bad):
    """Three blocks of 8 tokens: a row of 25 is neither copied nor trimmed, the other rows of the call are."""
    unchecked(monkeypatch)
    t = lambda *r: torch.tensor(r, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.tensor([[0, 1, 2], [3, 4, -1], [5, -1, -1], [-1, -1, -1]], dtype=torch.int32, device=DEV)
    lengths, ref = t(bad, 16, 8, 0), t(1, 1, 1, 1, 1, 1, 0)
    pool = torch.zeros(1, 2, 7, 1, 8, 16, dtype=BF16, device=DEV)
    flags()
    paged.pages_fork(pool, table, lengths, ref, t(0, 1), t(2, 3))
    assert flags() & L.FLAG_INDEX_RANGE
    assert table.tolist() == [[0, 1, 2], [3, 4, -1], [5, -1, -1], [3, 4, -1]]
    assert lengths.tolist() == [bad, 16, 8, 16] and ref.tolist() == [1, 1, 1, 2, 2, 1, 0]
    paged.pages_trim(table, lengths, ref, t(0, 1), 8, 2)
    assert flags() & L.FLAG_INDEX_RANGE
    assert table.tolist() == [[0, 1, 2], [-1, 4, -1], [5, -1, -1], [3, 4, -1]]
    assert ref.tolist() == [1, 1, 1, 1, 2, 1, 0]


def test_a_row_that_could_not_grow_is_left_out_by_the_append(monkeypatch):
    """Rows 0 and 1 share a full page and one page is free: row 0 grows, row 1 does not, and its token must not land on
    the shared page's last slot."""
    unchecked(monkeypatch)
    t = lambda *r: torch.tensor(r, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.tensor([[0, -1], [0, -1], [-1, -1]], dtype=torch.int32, device=DEV)
    lengths, ref, grown = t(16, 16, 0), t(2, 0), t(7, 7, 7)
    k, v = torch.randn(2, 2, 1, 16, 32, device=DEV).to(BF16)
    k0, v0 = k.clone(), v.clone()
    flags()
    paged.pages_extend(table, lengths, ref, t(0, 1, -1), 1, 16, grown=grown)
    assert flags() & L.FLAG_NO_PAGES
    assert lengths.tolist() == [17, 16, 0] and grown.tolist() == [1, 0, 7]
    qkv = torch.randn(3, 1, 3 * 32, device=DEV).to(BF16)
    q = paged.paged_append(qkv, k, v, table, lengths, grown=grown)
    assert torch.equal(k[0], k0[0]) and torch.equal(v[0], v0[0])
    assert torch.equal(k[1, 0, 0], qkv[0, 0, 32:64]) and torch.equal(v[1, 0, 0], qkv[0, 0, 64:])
    assert torch.equal(q[0, 0, 0], qkv[0, 0, :32]) and not bool(q[1].any())
    # a chunk of which only the last token is new: the ones before it are as padding
    chunk = torch.randn(1, 3, 3 * 32, device=DEV).to(BF16)
    k1 = k.clone()
    q = paged.paged_append(chunk, k, v, table[:1], lengths[:1], grown=t(1))
    assert not bool(q[0, :2].any()) and torch.equal(q[0, 2, 0], chunk[0, 2, :32])
    k1[1, 0, 0] = chunk[0, 2, 32:64]
    assert torch.equal(k, k1)


def test_extend_says_what_each_listed_row_grew_by(monkeypatch):
    unchecked(monkeypatch)
    t = lambda *r: torch.tensor(r, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.full((5, 2), -1, dtype=torch.int32, device=DEV)
    lengths, ref, grown = t(0, 30, 0, 3, -5), torch.zeros(9, dtype=torch.int32, device=DEV), t(-1, -1, -1, -1, -1)
    paged.pages_extend(table, lengths, ref, t(3, -1, 0, 1, 77, 4), 9, 16, grown=grown)
    assert grown.tolist() == [9, 0, -1, 9, 0] and lengths.tolist() == [9, 30, 0, 12, -5]
    flags()
    for bad in (grown[:4], grown.long(), grown.cpu()):
        with pytest.raises(ValueError):
            paged.pages_extend(table, lengths, ref, t(3), 1, 16, grown=bad)
    qkv = torch.zeros(2, 1, 3 * 32, device=DEV, dtype=BF16)
    k = torch.zeros(9, 1, 16, 32, device=DEV, dtype=BF16)
    for bad in (grown[:1], grown[:2].long(), grown[:2].cpu()):
        with pytest.raises(ValueError):
            paged.paged_append(qkv, k, k.clone(), table[:2], lengths[:2], grown=bad)
