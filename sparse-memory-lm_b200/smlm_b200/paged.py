"""A paged key-value cache and attention over it (no counterpart in the reference, whose decoding loop concatenates one
growing cache per layer, smlm/model.py:91-104).

A layer's keys and values lie in pages of `page_size` tokens; a table row lists a sequence's pages in order (-1: none),
`lengths` counts its tokens, and one reference count per page (0 = free) is the allocator's whole state. All of it is
on the device, so every function here can be captured in a CUDA graph:

    paged_attention     one new token per sequence over the cache, with a sliding window and first tokens that stay
                        visible (sinks)
    paged_append        rotary positions on a fused projection's queries and keys; keys and values into their pages
    pages_extend / pages_fork / pages_free / pages_trim / pages_compact
                        the pages of sequences that grow, split into several, end, slide out of a window, and the pool
                        made dense again

PagedKVCache keeps these tensors together for a model; smlm_b200.decode.PagedDecoder generates with it.

The cache and the activations are fp32, bf16 or fp16, of one type; scores, softmax sums and outputs are accumulated in
fp32 and rounded once. What a row's table and length do not cover is never used, whatever its bits. Rows of the table
outside their range, pages outside the pool and an exhausted pool do not fault: the token or row is left out and a flag
of the device status word is set (SMLM_B200_CHECK=1 turns it into an exception). A sequence that an exhausted pool kept
from growing is left out by the append that follows if it is given what pages_extend wrote to `grown`; PagedKVCache counts
pages on the host and never lets it come to that. There are no gradients: a backward pass through these calls raises.
"""
import importlib.machinery
import importlib.util
import os

import torch

from . import _lib as L

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _load():
    """The native binding (csrc/binding.cpp): checks, outputs, scratch and launch in one call."""
    path = os.path.join(os.path.dirname(L.LIB_PATH), "_paged.so")
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                          "or `make -C sparse-memory-lm_b200/csrc binding`")
    loader = importlib.machinery.ExtensionFileLoader("_paged", path)
    module = importlib.util.module_from_spec(importlib.machinery.ModuleSpec("_paged", loader, origin=path))
    loader.exec_module(module)
    module.init(lambda index: L.status_int(torch.device("cuda", index)))
    return module


class _AtFirstUse:
    """In the binding's place until a call needs it: modules that import this one work without it."""

    def __getattr__(self, name):
        global _native
        _native = _load()
        return getattr(_native, name)


_native = _AtFirstUse()


def _instrumented():
    """Whether calls are timed, ranged or checked."""
    return L.PROFILE is not None or L.NVTX or _native.checking()


def _call(name, launches, device, fn, *args):
    """A call that is timed, ranged or checked."""
    with L.timed(name, launches):
        out = fn(*args)
    L.after(device, name)
    return out


def paged_attention(q, k_pages, v_pages, table, lengths, *, scale=None, window=0, sinks=0, return_lse=False):
    """Attention of one new token per sequence: q (B, query heads, d), k_pages / v_pages (pages, key heads, page_size, d)
    with any page, head and token strides (multiples of 16 bytes), table (B, blocks) and lengths (B,) int32 -> (B,
    query heads, d). The newest token is expected in the cache already (paged_append), so lengths counts it.

    Query head i reads key head i // (query heads // key heads). Token j is visible if j < lengths[b] and its table
    entry is not -1; with window > 0 only the last `window` tokens and the first `sinks` are. scale defaults to
    d ** -0.5. A row that sees nothing gives 0. return_lse: also the logarithm of the softmax's sum, fp32 (B, query
    heads), -inf for such a row."""
    if not _instrumented():
        return _native.attention(q, k_pages, v_pages, table, lengths, scale, window, sinks, return_lse)
    launches = 0 if L.PROFILE is None else _native.attention_launches(q, k_pages, v_pages, table, lengths, window, sinks)
    return _call("paged_attention", launches, q.device, _native.attention, q, k_pages, v_pages, table, lengths, scale,
                 window, sinks, return_lse)


def paged_append(qkv, k_pages, v_pages, table, lengths, cos=None, sin=None, grown=None):
    """The last T tokens of every sequence: qkv (B, T, (query heads + 2 key heads) d), queries, then keys, then values;
    keys and values are written to their pages (positions lengths[b] - T .. lengths[b] - 1; a negative one is padding
    before a shorter chunk and is not stored), queries are returned, (B, T, query heads, d). With cos / sin (fp32,
    (positions, d / 2)) queries and keys are turned by the half-split rotary embedding of their position, in fp32,
    rounded once.

    grown (int32 (B,), what pages_extend wrote for these rows): only the last grown[b] tokens of the chunk are taken, the
    others are as padding. Without it, the chunk of a sequence that pages_extend could not extend overwrites the tokens at
    its end."""
    if not _instrumented():
        return _native.append(qkv, k_pages, v_pages, table, lengths, cos, sin, grown)
    return _call("paged_append", 1, qkv.device, _native.append, qkv, k_pages, v_pages, table, lengths, cos, sin, grown)


# --------------------------------------------------------------------------------------------- the pages
def pages_free(table, lengths, refcount, rows):
    """The sequences `rows` (int32) end: their pages are released, their table entries become -1, their lengths 0."""
    if not _instrumented():
        return _native.pages_free(table, lengths, refcount, rows)
    return _call("pages_free", 1, table.device, _native.pages_free, table, lengths, refcount, rows)


def pages_trim(table, lengths, refcount, rows, page_size, window, sinks=0):
    """Releases the pages of the sequences `rows` that paged_attention with this window and these sinks no longer reads:
    those that hold only tokens in [sinks, length - window)."""
    if not _instrumented():
        return _native.pages_trim(table, lengths, refcount, rows, page_size, window, sinks)
    return _call("pages_trim", 1, table.device, _native.pages_trim, table, lengths, refcount, rows, page_size,
                 window, sinks)


def pages_extend(table, lengths, refcount, rows, n_new, page_size, grown=None):
    """Every sequence in `rows` grows by n_new tokens: lengths[r] += n_new, with the lowest free pages (row by row) where
    its last page is full. A sequence that finds too few keeps its length; an append for it has to know (its positions
    are counted back from the length): grown, int32 (table rows,), receives n_new at the rows that grew and 0 at the
    listed ones that did not, and paged_append takes it."""
    if not _instrumented():
        return _native.pages_extend(table, lengths, refcount, rows, n_new, page_size, grown)
    return _call("pages_extend", 1, table.device, _native.pages_extend, table, lengths, refcount, rows, n_new,
                 page_size, grown)


def pages_fork(pool, table, lengths, refcount, parents, children):
    """Sequence children[i] becomes a copy of sequence parents[i] as it was before the call, for all i at once (a row may
    be a parent and a child: a beam's reordering); what the children held is released. Whole pages are shared, the
    tokens of a partly filled last page are copied in all layers. pool: (layers, 2, pages, key heads, page_size, d)."""
    if not _instrumented():
        return _native.pages_fork(table, lengths, refcount, pool, parents, children)
    return _call("pages_fork", 2, table.device, _native.pages_fork, table, lengths, refcount, pool, parents, children)


def pages_compact(pool, table, refcount):
    """Moves the pages in use to the lowest numbers, in the pool, the table and the counts: with n in use, the k-th used
    page numbered n or above goes to the k-th free page below n."""
    if not _instrumented():
        return _native.pages_compact(table, refcount, pool)
    return _call("pages_compact", 2, table.device, _native.pages_compact, table, refcount, pool)


# ----------------------------------------------------------------------------------------------- the cache
class PagedKVCache:
    """Keys and values of up to max_seqs sequences for all layers of a model, in n_pages pages of page_size tokens.

    A page number means the same page in every layer, so one table serves them all: pool (layers, 2, pages, key heads,
    page_size, d), table (max_seqs, blocks), lengths, refcount as the functions above take them. The lengths and the
    number of free pages are also known on the host (from the calls made here), so a call that would run out of pages
    raises before anything is launched, without a synchronisation in steps that only grow sequences."""

    def __init__(self, n_layers, n_pages, page_size, n_kv_heads, head_dim, max_seqs, max_len, dtype=torch.bfloat16,
                 device="cuda"):
        if page_size < 1 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} (a power of two up to 4096)")
        if dtype not in _TYPES:
            raise ValueError(f"unsupported type {dtype} (fp32, bf16 or fp16)")
        if head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"head dimension {head_dim} (a multiple of 16 up to 256)")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("PagedKVCache runs on CUDA (there is no CPU path)")
        self.page_size, self.max_seqs, self.max_len = page_size, max_seqs, max_len
        blocks = -(-max_len // page_size)
        self.pool = torch.zeros(n_layers, 2, n_pages, n_kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.table = torch.full((max_seqs, blocks), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.refcount = torch.zeros(n_pages, dtype=torch.int32, device=device)
        self.version = 0                  # counts the pools (resize makes a new one; a captured graph reads the old)
        self._len = [0] * max_seqs
        self._free = n_pages              # free pages, None: to be counted again

    @classmethod
    def for_model(cls, model, max_seqs, max_len=None, page_size=16, n_pages=None, dtype=torch.bfloat16):
        """A cache of the model's shape; n_pages defaults to what max_seqs sequences of max_len tokens need."""
        cfg = model.cfg
        max_len = max_len or cfg.max_seq_len
        if n_pages is None:
            n_pages = max_seqs * -(-max_len // page_size)
        return cls(cfg.n_layers, n_pages, page_size, cfg.n_heads, cfg.head_dim, max_seqs, max_len, dtype,
                   model.tok_emb.weight.device)

    def _rows(self, rows):
        rows = list(rows)
        for r in rows:
            if not 0 <= r < self.max_seqs:
                raise ValueError(f"sequence {r} of {self.max_seqs}")
        if len(set(rows)) < len(rows):
            raise ValueError(f"sequences listed twice: {rows}")
        return rows

    def _device(self, rows):
        return torch.tensor(rows, dtype=torch.int32, device=self.table.device)

    def length(self, row):
        return self._len[row]

    def free_pages(self):
        """Pages no sequence holds (reads them from the device if a call since has released some)."""
        if self._free is None:
            self._free = int((self.refcount == 0).sum())
        return self._free

    def _take(self, need, what):
        # the count known is exact, so a shortage is one; shared pages make releases unpredictable, hence None above
        if need > self.free_pages():
            raise RuntimeError(f"{what}: {need} pages needed, {self._free} of {self.refcount.shape[0]} free")
        self._free -= need

    def reserve(self, rows, n):
        """Host side of extend: checks and counts n more tokens for each of `rows`."""
        if n < 0:
            raise ValueError(f"PagedKVCache.extend: {n} new tokens")
        p = self.page_size
        for r in rows:
            if self._len[r] + n > self.max_len:
                raise ValueError(f"sequence {r}: {self._len[r]} + {n} tokens, max_len {self.max_len}")
        self._take(sum(-(-(self._len[r] + n) // p) - -(-self._len[r] // p) for r in rows), "PagedKVCache.extend")
        for r in rows:
            self._len[r] += n

    def extend(self, rows, n):
        """Room for n more tokens of each of the sequences `rows` (their lengths grow by n; paged_append fills it)."""
        rows = self._rows(rows)
        self.reserve(rows, n)
        pages_extend(self.table, self.lengths, self.refcount, self._device(rows), n, self.page_size)

    def fork(self, parents, children):
        """children[i] becomes a copy of parents[i] (as both were before the call). Needs a page for every child whose
        parent's last page is partly filled, free before the call or released with what the children held."""
        children, parents = self._rows(children), list(parents)
        for r in parents:
            self._rows([r])
        if len(parents) != len(children):
            raise ValueError(f"{len(parents)} parents, {len(children)} children")
        pairs = [(p, c) for p, c in zip(parents, children) if p != c]
        need = sum(self._len[p] % self.page_size > 0 for p, _ in pairs)
        if need > self.free_pages():
            free = self._free_in_fork(pairs)
            if need > free:
                raise RuntimeError(f"PagedKVCache.fork: {need} pages needed, {free} of {self.refcount.shape[0]} free")
        pages_fork(self.pool, self.table, self.lengths, self.refcount, self._device(parents), self._device(children))
        self._free = None
        for c, n in zip(children, [self._len[p] for p in parents]):
            self._len[c] = n

    def _free_in_fork(self, pairs):
        """The pages a fork of these (parent, child) pairs has to hand out: those that nothing holds once the parents'
        are held and the children's released (reads the tables)."""
        table, count = self.table.cpu(), self.refcount.cpu()
        for p, c in pairs:
            held, old = table[p, :-(-self._len[p] // self.page_size)], table[c]
            count += torch.bincount(held[held >= 0], minlength=len(count))
            count -= torch.bincount(old[old >= 0], minlength=len(count))
        return int((count == 0).sum())

    def free(self, rows):
        """The sequences end; pages that no other sequence shares become free."""
        rows = self._rows(rows)
        pages_free(self.table, self.lengths, self.refcount, self._device(rows))
        self._free = None
        for r in rows:
            self._len[r] = 0

    def trim(self, rows, window, sinks=0):
        """Releases the pages that attention with this window and these sinks no longer reads. (A trimmed sequence can
        only be attended with a window and sinks no larger than these.)"""
        rows = self._rows(rows)
        pages_trim(self.table, self.lengths, self.refcount, self._device(rows), self.page_size, window, sinks)
        self._free = None

    def compact(self):
        """Moves the pages in use to the lowest numbers; returns how many there are (synchronises)."""
        pages_compact(self.pool, self.table, self.refcount)
        self._free = None
        return self.refcount.shape[0] - self.free_pages()

    def resize(self, n_pages):
        """A pool of n_pages pages (at least those in use) in place of this one: compacts, then copies the pages in
        use. Graphs captured over the old pool do not follow (version changes)."""
        used = self.compact()
        if n_pages < used:
            raise ValueError(f"{used} pages are in use, {n_pages} wanted")
        L_, two, _, h, p, d = self.pool.shape
        pool = torch.zeros(L_, two, n_pages, h, p, d, dtype=self.pool.dtype, device=self.pool.device)
        pool[:, :, :used] = self.pool[:, :, :used]
        count = torch.zeros(n_pages, dtype=torch.int32, device=self.pool.device)
        count[:used] = self.refcount[:used]
        self.pool, self.refcount, self._free = pool, count, n_pages - used
        self.version += 1

    def view(self, rows=None, window=0, sinks=0):
        """What a forward pass over these sequences (all of them by default) passes to the model."""
        if rows is None:
            return PagedView(self, self.table, self.lengths, None, window, sinks)
        rows = self._rows(rows)
        held = {self._len[r] for r in rows}
        if len(held) > 1:
            raise ValueError(f"sequences of one length, got {sorted(held)}")
        at = torch.tensor(rows, device=self.table.device)
        return PagedView(self, self.table[at], self.lengths[at], held.pop(), window, sinks)


class PagedView:
    """Some sequences of a PagedKVCache for one forward pass: their table rows and lengths, the length they all have (for
    passes of several tokens; None: any), and the window and sinks of the attention."""

    def __init__(self, cache, table, lengths, held, window, sinks):
        self.cache, self.table, self.lengths, self.held = cache, table, lengths, held
        self.window, self.sinks = window, sinks

    def caches(self):
        """The kv_caches argument of Transformer.forward."""
        return [{"paged": self, "layer": i} for i in range(self.cache.pool.shape[0])]

    def append(self, layer, qkv, cos, sin):
        k, v = self.cache.pool[layer]
        return paged_append(qkv, k, v, self.table, self.lengths, cos, sin)

    def attend(self, layer, q):
        k, v = self.cache.pool[layer]
        return paged_attention(q, k, v, self.table, self.lengths, window=self.window, sinks=self.sinks)

    def gather(self, layer):
        """keys and values of the sequences, (B, heads, held, d) each, in trimmed pages 0: a mask keeps their weights out,
        but not an infinity or NaN times 0 that another sequence's page would bring in."""
        rows = self.table[:, :-(-self.held // self.cache.page_size)]
        out = self.cache.pool[layer][:, rows.clamp(min=0).long()].masked_fill_((rows < 0)[..., None, None, None], 0)
        out = out.transpose(2, 3).flatten(3, 4)
        return out[0, :, :, :self.held], out[1, :, :, :self.held]

    def visible(self, tokens):
        """(tokens, held) bool: what each of the last `tokens` positions sees; None: all before it (plain causal)."""
        n = self.held
        if n == tokens and (not self.window or self.window >= n):
            return None
        dev = self.table.device
        j, t = torch.arange(n, device=dev)[None], torch.arange(n - tokens, n, device=dev)[:, None]
        seen = j <= t
        if self.window:
            seen &= (j > t - self.window) | (j < self.sinks)
        return seen
