"""The paged key-value cache's kernels against 64-bit and pure-Python forms: attention of one new token (types, head
layouts, lengths from nothing to long, windows and sinks, holes, strides), append, and the pages' management."""
import math
import random

import pytest
import torch

import paged_ref as R
from smlm_b200 import paged

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(lens, hq, hkv, d, page, dtype, seed=0, order="hnd", slack=3, stale=float("nan")):
    """A cache whose pages lie in random order in the pool; everything outside the sequences is `stale`."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in lens]
    pages = sum(blocks) + slack
    perm = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(1, max(blocks)) + 1), -1, dtype=torch.int32)
    pool = torch.full((2, pages, hkv, page, d), stale, dtype=dtype)
    at = 0
    for b, n in enumerate(lens):
        for j in range(blocks[b]):
            p = int(perm[at])
            at += 1
            table[b, j] = p
            m = min(page, n - j * page)
            pool[:, p, :, :m] = torch.randn(2, hkv, m, d, generator=g).to(dtype)
    if order == "nhd":
        pool = pool.transpose(2, 3).contiguous().to(DEV).transpose(2, 3)
    else:
        pool = pool.to(DEV)
    q = torch.randn(len(lens), hq, d, generator=g).to(dtype).to(DEV)
    return q, pool[0], pool[1], table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)


def check(q, k, v, table, lengths, scale=None, window=0, sinks=0):
    out, lse = paged.paged_attention(q, k, v, table, lengths, scale=scale, window=window, sinks=sinks, return_lse=True)
    sc = q.shape[2] ** -0.5 if scale is None else scale
    ref, rlse, mag, reach = R.attention(q, k, v, table, lengths, sc, window, sinks)
    bound = R.attention_bound(ref, mag, reach, q.dtype, int(lengths.max()) if len(lengths) else 0)
    err = (out.double().cpu() - ref).abs()
    assert not bool((err > bound).any()) and not bool(err.isnan().any()), float((err / bound).max())
    seen = rlse > -math.inf
    assert torch.equal(lse.cpu() == -math.inf, ~seen)
    # the logarithm of a sum whose terms are off by 2^-16 reach (2^-19 in fp32) and that is rounded to fp32
    near = (2.0 ** -16 * reach[..., 0] + 2.0 ** -20 + int(lengths.max()) * 2.0 ** -24 + 2.0 ** -22 * rlse.abs())[seen]
    assert not bool(((lse.double().cpu() - rlse)[seen].abs() > near).any())
    assert torch.equal(out, paged.paged_attention(q, k, v, table, lengths, scale=scale, window=window, sinks=sinks))
    return out


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(6, 6, 64, 16), (8, 1, 128, 32), (32, 8, 128, 16), (4, 4, 16, 8),
                                           (7, 7, 80, 64), (20, 2, 96, 128), (6, 3, 256, 16), (3, 1, 48, 1),
                                           (17, 1, 32, 4), (40, 2, 64, 256)])
def test_attention_head_layouts_and_types(dtype, hq, hkv, d, page):
    check(*make([1, 37, 0, 300, page, page + 1], hq, hkv, d, page, dtype, seed=hq + d))


def roomy(table, page):
    """The table with room for sequences of 100000 tokens: how the work is cut follows from what the table could hold
    (one cluster per item while that is little, a list over the whole card else)."""
    out = torch.full((table.shape[0], 100000 // page), -1, dtype=torch.int32, device=DEV)
    out[:, :table.shape[1]] = table
    return out


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,hkv,d,page", [(6, 6, 64, 16), (8, 1, 128, 32), (32, 8, 128, 16), (4, 4, 16, 8),
                                           (7, 7, 80, 64), (20, 2, 96, 128), (6, 3, 256, 16), (3, 1, 48, 1),
                                           (17, 1, 32, 4), (40, 2, 64, 256)])
def test_attention_in_tables_with_room(dtype, hq, hkv, d, page):
    q, k, v, table, lengths = make([1, 37, 0, 300, 0, page, 700], hq, hkv, d, page, dtype, seed=hq + d)
    check(q, k, v, roomy(table, page), lengths)
    check(q, k, v, roomy(table, page), lengths, window=50, sinks=5)


@pytest.mark.parametrize("batch", [1, 2, 31, 33, 128, 129, 500])
def test_attention_batches_in_tables_with_room(batch):
    """The list's cut for batches of less and more rows than a warp has lanes and a block has threads; empty rows among
    them, alone and last."""
    r = random.Random(batch)
    lens = [r.choice([0, 0, 1, 16, 33, 90, 400]) for _ in range(batch)]
    lens[-1] = 0 if batch > 1 else 5
    q, k, v, table, lengths = make(lens, 4, 2, 32, 16, BF16, seed=batch)
    check(q, k, v, roomy(table, 16), lengths)
    lengths.zero_()
    out = paged.paged_attention(q, k, v, roomy(table, 16), lengths)
    assert not bool(out.any())


@pytest.mark.parametrize("room", [False, True])
@pytest.mark.parametrize("n", [300, 1100, 2300])
def test_attention_clusters_of_every_size(n, room):
    for batch in (1, 3, 9, 24, 40):
        q, k, v, table, lengths = make([n - 7 * i for i in range(batch)], 6, 6, 64, 16, BF16, seed=n + batch)
        check(q, k, v, roomy(table, 16) if room else table, lengths)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 1000, 5003])
def test_attention_every_small_length_and_long_ones(dtype, n):
    check(*make([n], 6, 6, 64, 16, dtype, seed=n))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (16, 16), (33, 1), (64, 0), (100, 40), (4096, 4)])
def test_attention_window_and_sinks(dtype, window, sinks):
    check(*make([0, 1, 5, 16, 39, 40, 64, 139, 140, 141, 513], 4, 2, 64, 16, dtype, seed=window), window=window,
          sinks=sinks)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_sequences_with_holes_and_rows_that_see_nothing(dtype):
    """Entries of -1 (trimmed pages) are not seen, whatever lies beside them; a row of holes gives 0."""
    q, k, v, table, lengths = make([300, 300, 40, 17], 8, 4, 64, 16, dtype, seed=5)
    table[0, 2:9] = -1
    table[1, :] = -1
    table[2, 0] = -1
    table[3, 1] = -1
    out = check(q, k, v, table, lengths)
    assert not bool(out[1].any())
    check(q, k, v, table, lengths, window=120, sinks=20)
    check(q, k, v, table, lengths, window=3, sinks=1)


@pytest.mark.parametrize("batch", [1, 5, 300])
def test_attention_uneven_batches(batch):
    """Batches whose sequences differ by orders of magnitude (the work is cut across sequences)."""
    r = random.Random(batch)
    lens = [int(math.exp(r.uniform(0, math.log(3000)))) - 1 for _ in range(batch)]
    check(*make(lens, 6, 2, 64, 16, BF16, seed=batch))


@pytest.mark.parametrize("order", ["hnd", "nhd"])
def test_attention_strides(order):
    """Heads next to tokens or tokens next to heads, pages a stride apart, keys and values laid out differently, rows of
    a wider table, queries that are a slice."""
    q, k, v, table, lengths = make([70, 9, 33], 6, 3, 32, 8, BF16, seed=3, order=order, stale=0.0)
    check(q, k, v, table, lengths)
    wide = torch.zeros(k.shape[0], 2, *k.shape[1:], dtype=k.dtype, device=DEV)
    wide[:, 1] = k
    other = v.transpose(1, 2).contiguous().transpose(1, 2)
    broad = torch.full((3, table.shape[1] + 5), 99999, dtype=torch.int32, device=DEV)
    broad[:, :table.shape[1]] = table
    full = torch.randn(3, 12, 32, device=DEV).to(BF16)
    check(full[:, ::2], wide[:, 1], other, broad[:, :table.shape[1]], lengths)


def test_strides_of_dimensions_with_one_element_do_not_matter():
    q, k, v, table, lengths = make([40, 7], 4, 1, 64, 16, BF16, seed=6)
    odd = k.as_strided(k.shape, (k.stride(0), 7, k.stride(2), 1))
    want = paged.paged_attention(q, k, v, table, lengths)
    assert torch.equal(paged.paged_attention(q, odd, v, table, lengths), want)
    one = table[:1].as_strided((1, table.shape[1]), (3, 1))
    assert torch.equal(paged.paged_attention(q[:1], k, v, one, lengths[:1]),
                       paged.paged_attention(q[:1], k, v, table[:1], lengths[:1]))
    k1 = k[int(table[1, 0]):int(table[1, 0]) + 1]
    v1 = v[int(table[1, 0]):int(table[1, 0]) + 1]
    single = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    check(q[1:], k1.as_strided(k1.shape, (5, 3, k1.stride(2), 1)), v1, single, lengths[1:])


def test_attention_scores_of_infinity_and_large_scores():
    """Visible keys may give scores of -inf (weight 0); scores of thousands do not overflow."""
    q, k, v, table, lengths = make([40, 20], 2, 2, 64, 16, F32, seed=8)
    q.abs_()
    p = int(table[0, 1])
    k[p, :, 3] = -math.inf
    k[int(table[1, 0])] = -math.inf
    k[int(table[1, 1])] = -math.inf
    out, lse = paged.paged_attention(q, k, v, table, lengths, return_lse=True)
    assert not bool(out[1].any()) and bool((lse[1] == -math.inf).all())
    kept = [j for j in range(40) if j != 19]
    pages = table[0].long()[torch.tensor([j // 16 for j in kept], device=DEV)]
    slots = torch.tensor([j % 16 for j in kept], device=DEV)
    for h in range(2):
        kk, vv = k[pages, h, slots].double(), v[pages, h, slots].double()
        ref = torch.softmax(kk @ q[0, h].double() / 8, 0) @ vv
        torch.testing.assert_close(out[0, h].double(), ref, rtol=1e-5, atol=1e-5)
    q, k, v, table, lengths = make([200], 2, 2, 64, 16, BF16, seed=9)
    out = paged.paged_attention(q * 64, k * 64, v, table, lengths)
    ref, _, mag, reach = R.attention(q * 64, k * 64, v, table, lengths, 0.125)
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= R.attention_bound(ref, mag, reach, BF16, 200)).all())
    assert bool(torch.isnan(paged.paged_attention(q * math.nan, k, v, table, lengths)).all())


def test_attention_offsets_beyond_32_bits():
    """Pages whose element offsets pass 2^31 and 2^32."""
    page, d = 16, 64
    pool = torch.empty(2, 2 ** 32 // (page * d) // 2 + 64, 1, page, d, dtype=BF16, device=DEV)
    pages = pool.shape[1]
    ids = torch.tensor([pages - 1, 5, pages // 2 + 9, pages - 30], dtype=torch.int32, device=DEV)
    pool[:, ids.long()] = torch.randn(2, 4, 1, page, d, device=DEV).to(BF16)
    both = pool.view(-1, 1, page, d)                   # keys and values from one range: offsets up to 2^32
    ids2 = ids + pages
    q = torch.randn(2, 3, d, device=DEV).to(BF16)
    table, lengths = torch.stack((ids, ids2)), torch.tensor([64, 50], dtype=torch.int32, device=DEV)
    check(q, both, both, table, lengths)
    qkv = torch.randn(2, 3, 3 * d, device=DEV).to(BF16)
    values = both.clone()
    paged.paged_append(qkv, both, values, table, lengths)
    assert torch.equal(both[ids2[3].long(), 0, 1], qkv[1, 2, d:2 * d])
    assert torch.equal(values[ids2[3].long(), 0, 1], qkv[1, 2, 2 * d:])


def test_attention_on_another_stream_and_in_a_graph():
    q, k, v, table, lengths = make([400, 3, 77], 6, 6, 64, 16, BF16, seed=2)
    want = paged.paged_attention(q, k, v, table, lengths)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = paged.paged_attention(q, k, v, table, lengths)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = paged.paged_attention(q, k, v, table, lengths)
    lengths.copy_(torch.tensor([399, 0, 50], dtype=torch.int32))        # a replay reads the lengths of its time
    g.replay()
    assert torch.equal(out, paged.paged_attention(q, k, v, table, lengths))
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):                                                  # calls in flight together
        with torch.cuda.stream(streams[i % 4]):
            outs.append(paged.paged_attention(q, k, v, table, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for o in outs)


def test_attention_table_entries_outside_the_pool_are_flagged():
    q, k, v, table, lengths = make([40, 40], 2, 2, 64, 16, BF16, seed=4, stale=0.0)
    table[1, 1] = k.shape[0] + 7
    with pytest.raises(IndexError):
        paged.paged_attention(q, k, v, table, lengths)
    table[1, 1] = 0
    lengths[0] = 10 ** 6
    with pytest.raises(IndexError):
        paged.paged_attention(q, k, v, table, lengths)


def test_attention_empty_batch():
    q, k, v, table, lengths = make([4], 2, 2, 64, 16, BF16)
    assert paged.paged_attention(q[:0], k, v, table[:0], lengths[:0]).shape == (0, 2, 64)


# ---------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq,hkv,d,page,T,lens", [
    (6, 6, 64, 16, 1, [1, 17, 2175, 16]), (8, 2, 128, 32, 1, [5]), (4, 4, 16, 8, 37, [37, 40, 77]),
    (6, 3, 80, 4, 5, [3, 9, 0, 5]), (3, 1, 256, 64, 130, [131]), (5, 5, 48, 1, 3, [3, 4]), (1, 1, 32, 16, 2, [20])])
@pytest.mark.parametrize("rope,order", [(True, "hnd"), (True, "nhd"), (False, "hnd")])
def test_append(dtype, hq, hkv, d, page, T, lens, rope, order):
    _, k, v, table, lengths = make(lens, hq, hkv, d, page, dtype, seed=T, order=order, stale=3.0)
    qkv = torch.randn(len(lens), T, (hq + 2 * hkv) * d, device=DEV).to(dtype)
    cos, sin = (x.to(DEV) for x in R.rotary(d, max(lens) + 1)) if rope else (None, None)
    rq, rk, rv = R.append(qkv, k, v, table, lengths, cos, sin)
    q = paged.paged_append(qkv, k, v, table, lengths, cos, sin)
    # two products and their sum in fp32 (3 roundings of at most |x| + |y|), then one rounding to the type
    size = qkv.abs().max().double().cpu() * 2
    for got, ref in ((q, rq), (k, rk), (v, rv)):
        err = (got.double().cpu() - ref).abs()
        assert bool((err <= R.UNIT[dtype] * ref.abs() + size * 2.0 ** -22 + 2.0 ** -25).all()), float(err.max())
    held = torch.zeros_like(rk, dtype=torch.bool)          # tokens outside the chunk are not touched
    for b, n in enumerate(lens):
        for pos in range(max(0, n - T), n):
            held[int(table[b, pos // page]), :, pos % page] = True
    assert torch.equal(k.double().cpu()[~held], rk[~held]) and torch.equal(v.double().cpu(), rv)


def test_append_without_a_page_and_beyond_the_rotary_table_is_flagged():
    _, k, v, table, lengths = make([20, 20], 2, 2, 32, 16, BF16, stale=0.0)
    qkv = torch.randn(2, 1, 6 * 32, device=DEV).to(BF16)
    cos, sin = (x.to(DEV) for x in R.rotary(32, 10))
    before = k.clone()
    with pytest.raises(IndexError):
        paged.paged_append(qkv, k, v, table, lengths, cos, sin)
    table[:, 1] = -1
    with pytest.raises(RuntimeError, match="no free page"):
        paged.paged_append(qkv, k, v, table, lengths)
    assert torch.equal(k, before)


# ----------------------------------------------------------------------------------------------------- pages
class Device:
    """A cache on the GPU, driven beside a Book."""

    def __init__(self, rows, blocks, pages, page, layers=2, heads=3, d=16, dtype=BF16):
        self.book = R.Book(rows, blocks, pages, page)
        self.table = torch.full((rows, blocks), -1, dtype=torch.int32, device=DEV)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=DEV)
        self.refcount = torch.zeros(pages, dtype=torch.int32, device=DEV)
        self.pool = torch.zeros(layers, 2, pages, heads, page, d, dtype=dtype, device=DEV)
        # every plane, head and column holds the token's value times a factor of its own
        f = torch.arange(1, layers * 2 * heads * d + 1, device=DEV) % 7 + 1
        self.factor = f.view(layers, 2, 1, heads, 1, d).to(dtype)
        self.token = 0

    def rows(self, r):
        return torch.tensor(r, dtype=torch.int32, device=DEV)

    def same(self):
        assert self.table.tolist() == self.book.table
        assert self.lengths.tolist() == self.book.len
        assert self.refcount.tolist() == self.book.ref
        data = torch.tensor(self.book.data, device=DEV).to(self.pool.dtype)
        want = data.view(1, 1, len(self.book.ref), 1, -1, 1) * self.factor
        used = torch.zeros(data.shape, dtype=torch.bool)
        for row, n in zip(self.book.table, self.book.len):
            for t in range(n):
                if row[t // self.book.page] >= 0:
                    used[row[t // self.book.page], t % self.book.page] = True
        diff = (self.pool != want).any(5).any(3).any(1).any(0).cpu()
        assert not bool((diff & used).any())

    def extend(self, rows, n):
        start = [self.book.len[r] for r in rows]
        paged.pages_extend(self.table, self.lengths, self.refcount, self.rows(rows), n, self.book.page)
        self.book.extend(rows, n)
        for r, a in zip(rows, start):
            for t in range(a, a + n):
                p, s = self.book.table[r][t // self.book.page], t % self.book.page
                self.token += 1
                self.book.data[p][s] = float(self.token % 31)
                self.pool[:, :, p, :, s] = self.factor[:, :, 0, :, 0] * (self.token % 31)

    def fork(self, parents, children):
        paged.pages_fork(self.pool, self.table, self.lengths, self.refcount, self.rows(parents), self.rows(children))
        self.book.fork(parents, children)

    def free(self, rows):
        paged.pages_free(self.table, self.lengths, self.refcount, self.rows(rows))
        self.book.free(rows)

    def trim(self, rows, window, sinks):
        paged.pages_trim(self.table, self.lengths, self.refcount, self.rows(rows), self.book.page, window, sinks)
        self.book.trim(rows, window, sinks)

    def compact(self):
        paged.pages_compact(self.pool, self.table, self.refcount)
        self.book.compact()


@pytest.mark.parametrize("page,dtype", [(1, BF16), (4, F32), (8, F16), (16, BF16)])
def test_pages_random_operations(page, dtype):
    """A few hundred random calls: tables, lengths, counts and tokens are those of the lists after each."""
    r = random.Random(page)
    dev = Device(12, 9, 160, page, dtype=dtype)
    for step in range(120):
        op = r.choice(["extend", "extend", "extend", "fork", "fork", "free", "trim", "compact"])
        if op == "extend":
            n = r.choice([1, 1, 2, page, page + 1])
            rows = [x for x in range(12) if dev.book.len[x] + n <= 9 * page and r.random() < 0.5]
            need = sum(-(-(dev.book.len[x] + n) // page) + (dev.book.len[x] // -page) for x in rows)
            if rows and need <= dev.book.ref.count(0):
                r.shuffle(rows)
                dev.extend(rows, n)
        elif op == "fork":
            m = r.randrange(1, 8)
            children = r.sample(range(12), m)
            parents = [r.randrange(12) for _ in range(m)]
            if dev.book.ref.count(0) >= m:
                dev.fork(parents, children)
        elif op == "free":
            dev.free(r.sample(range(12), 2))
        elif op == "trim":
            dev.trim(r.sample(range(12), 3), r.choice([1, page, 2 * page + 1]), r.choice([0, 1, page + 1]))
        else:
            dev.compact()
        dev.same()


@pytest.mark.parametrize("rows,blocks,pages", [(300, 40, 5000), (3, 2000, 30011)])
def test_pages_large_pools(rows, blocks, pages):
    """More rows, blocks and pages than one thread block has threads."""
    page = 4
    dev = Device(rows, blocks, pages, page, layers=1, heads=1)
    n = 41 if rows > 3 else 4003
    half = list(range(0, rows, 2))
    paged.pages_extend(dev.table, dev.lengths, dev.refcount, dev.rows(half), n, page)
    dev.book.extend(half, n)
    dev.same()
    dev.fork(half[:len(half) // 2 + 1], [x + 1 for x in half[:len(half) // 2 + 1]] if rows > 3 else [1, 0])
    dev.same()
    dev.free(half[1::2])
    dev.same()
    dev.compact()
    dev.same()
    dev.free(list(range(rows)))
    dev.same()
    assert not bool(dev.refcount.any())


def test_pages_beam_reordering():
    """Rows that are parents and children at once: every child gets what its parent was before the call."""
    dev = Device(6, 4, 40, 8)
    for i in range(6):
        dev.extend([i], 3 + 4 * i)
    for parents in ([1, 2, 3, 4, 5, 0], [0, 0, 1, 1, 2, 2], [5, 4, 3, 2, 1, 0], [3, 3, 3, 3, 3, 3]):
        dev.fork(parents, list(range(6)))
        dev.same()
        dev.extend(list(range(6)), 1)
        dev.same()


def test_pages_exhaustion_and_bad_rows_are_flagged_and_leave_the_rest():
    t = lambda *r: torch.tensor(r, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.full((4, 4), -1, dtype=torch.int32, device=DEV)
    lengths, ref = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="no free page"):
        paged.pages_extend(table, lengths, ref, t(0, 1), 16, 8)          # the second row finds one page of two
    assert lengths.tolist() == [16, 0, 0, 0] and ref.tolist() == [1, 1, 0]
    assert table.tolist()[0] == [0, 1, -1, -1] and table.tolist()[1] == [-1] * 4
    with pytest.raises(IndexError):
        paged.pages_extend(table, lengths, ref, t(0, 9, -1), 17, 8)      # beyond the table's columns, bad rows
    assert lengths.tolist() == [16, 0, 0, 0] and ref.tolist() == [1, 1, 0]
    with pytest.raises(IndexError):
        paged.pages_extend(table, lengths, ref, t(1, 1), 3, 8)           # a row listed twice grows once
    assert lengths.tolist() == [16, 3, 0, 0]
    pool = torch.zeros(1, 2, 3, 1, 8, 16, dtype=BF16, device=DEV)
    with pytest.raises(RuntimeError, match="no free page"):
        paged.pages_fork(pool, table, lengths, ref, t(1), t(2))          # no page for the copied part
    assert lengths.tolist() == [16, 3, 3, 0] and table.tolist()[2] == [-1] * 4
    with pytest.raises(IndexError):
        paged.pages_fork(pool, table, lengths, ref, t(0, 0, 7), t(3, 3, 1))
    assert lengths.tolist() == [16, 3, 3, 16] and ref.tolist() == [2, 2, 1]
    paged.pages_free(table, lengths, ref, t(0, 0, 3))                    # a row listed twice is released once
    assert ref.tolist() == [0, 0, 1] and lengths.tolist() == [0, 3, 3, 0]
    with pytest.raises(IndexError):
        paged.pages_free(table, lengths, ref, t(4))
