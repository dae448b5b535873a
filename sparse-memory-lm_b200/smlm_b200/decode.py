"""Greedy decoding with the whole step in one CUDA graph (no counterpart in the reference).

The reference's decoding loop (smlm/train.py:283-315) runs the dense blocks eagerly and replays CUDA graphs of the
memory layers only (smlm/pkm.py:159-184); with about 30 PyTorch launches per block, a one-token step is bound by
the host. GraphDecoder gives every attention layer a static KV cache (preallocated (B, heads, max_len, head_dim)
buffers) and keeps the position on the device, so that one step (embedding, every block with its memory layers'
scoring + selection + value bag, the final norm, the LM head and the argmax that picks the next token) has fixed
shapes and replays as one captured graph. The model's own modules run inside it, unchanged: the same kernels as
the eager path, except that attention reads the masked static cache.

    dec = GraphDecoder(model, batch=1, max_len=2304)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        dec.prefill(prompt_ids)            # (B, P) -> logits of the prompt; next tokens in dec.tokens
        for _ in range(256):
            nxt = dec.step()                # (B, 1) greedy tokens, device tensor (replays the graph)

PagedDecoder serves sequences of different lengths from a paged cache (smlm_b200.paged): a step reads each sequence's
own tokens instead of max_len masked slots, sequences begin and end independently, several continuations share their
prompt's pages (fork), and with a sliding window the pages that have left it are released.

    dec = PagedDecoder(model, max_seqs=8, max_len=2304)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        dec.prefill(prompt_ids, rows=[0])   # one prompt
        dec.fork(0, range(1, 8))            # eight continuations of it
        for _ in range(256):
            dec.step(sample(dec.logits))
        dec.free([3])                       # a sequence ends; its pages serve others
"""
import torch

from .model import Transformer
from .paged import PagedKVCache, pages_extend


class GraphDecoder:
    def __init__(self, model: Transformer, batch: int, max_len: int = None, dtype=None):
        cfg = model.cfg
        if cfg.eng_layers:
            raise ValueError("GraphDecoder: Engram memories keep growing caches (decode them with the KV-cache loop)")
        if model.training:
            raise ValueError("GraphDecoder: put the model in eval mode first (BatchNorm uses its running statistics)")
        self.model = model
        self.batch = batch
        self.max_len = max_len or cfg.max_seq_len
        if self.max_len > cfg.max_seq_len:
            raise ValueError(f"max_len {self.max_len} exceeds the model's max_seq_len {cfg.max_seq_len}")
        dev = model.tok_emb.weight.device
        if dev.type != "cuda":
            raise ValueError("GraphDecoder runs on CUDA")
        if dtype is None:
            dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else torch.float32
        hd = cfg.d_model // cfg.n_heads
        arange = torch.arange(self.max_len, device=dev)
        self.caches = [{"kbuf": torch.zeros(batch, cfg.n_heads, self.max_len, hd, dtype=dtype, device=dev),
                        "vbuf": torch.zeros(batch, cfg.n_heads, self.max_len, hd, dtype=dtype, device=dev),
                        "arange": arange, "pos": None} for _ in range(cfg.n_layers)]
        self.tokens = torch.zeros(batch, 1, dtype=torch.long, device=dev)   # the next step's input tokens
        self.pos = torch.zeros(1, dtype=torch.long, device=dev)            # their position
        self.logits = None
        self.length = 0
        self._graph = None
        self._key = None

    def _set_pos(self, pos):
        for c in self.caches:
            c["pos"] = pos

    @torch.no_grad()
    def prefill(self, ids):
        """ids (B, P): fills the caches for positions 0 .. P-1 (eager) and sets the next tokens to the greedy
        choice after the prompt. Returns the prompt's logits (B, P, vocab)."""
        B, P = ids.shape
        if B != self.batch or P >= self.max_len:
            raise ValueError(f"prefill: ids {tuple(ids.shape)} for batch {self.batch}, max_len {self.max_len}")
        self._set_pos(torch.arange(P, device=ids.device))
        logits = self.model(ids, kv_caches=self.caches)
        self.tokens.copy_(logits[:, -1:].argmax(-1))
        self.pos.fill_(P)
        self.length = P
        return logits

    def _body(self):
        self._set_pos(self.pos)
        self.logits = self.model(self.tokens, kv_caches=self.caches)
        self.tokens.copy_(self.logits[:, -1:].argmax(-1))
        self.pos.add_(1)

    @torch.no_grad()
    def step(self, tokens=None):
        """One greedy step: feeds self.tokens (or `tokens`, (B, 1)) at the current position and leaves the
        argmax of its logits in self.tokens (returned; self.logits holds the logits). The first call captures
        the graph (with the memory layers' own one-token graphs switched off inside it)."""
        if self.length + 1 > self.max_len:
            raise ValueError("GraphDecoder: the static cache is full")
        if tokens is not None:
            self.tokens.copy_(tokens)
        ac = torch.is_autocast_enabled("cuda")
        key = (ac, torch.get_autocast_dtype("cuda") if ac else None)
        if self._graph is None or self._key != key:
            self._capture(key)
        self._graph.replay()
        self.length += 1
        return self.tokens

    def _capture(self, key):
        mems = self.model.memory_layers()
        flags = [getattr(m, "decode_graph", False) for m in mems]
        for m in mems:
            m.decode_graph = False
        ctx = (torch.autocast("cuda", dtype=key[1], cache_enabled=False) if key[0]
               else torch.autocast("cuda", enabled=False))
        saved_tok, saved_pos = self.tokens.clone(), self.pos.clone()
        try:
            s = torch.cuda.Stream(self.tokens.device)
            s.wait_stream(torch.cuda.current_stream(self.tokens.device))
            with torch.cuda.stream(s), ctx:
                for _ in range(2):              # warm-up: writes cache slots past the position, masked until used
                    self._body()
                    self.pos.copy_(saved_pos)
            torch.cuda.current_stream(self.tokens.device).wait_stream(s)
            self.tokens.copy_(saved_tok)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph), ctx:
                self._body()
            self.tokens.copy_(saved_tok)
            self.pos.copy_(saved_pos)
        finally:
            for m, f in zip(mems, flags):
                m.decode_graph = f
        self._graph, self._key = graph, key


class PagedDecoder:
    """Decoding over a PagedKVCache of max_seqs rows. Every step is one CUDA graph over all rows; rows that hold nothing
    idle in it. window / sinks: attention over the last `window` tokens and the first `sinks` only (0: all)."""

    def __init__(self, model: Transformer, max_seqs: int, max_len: int = None, page_size: int = 16, n_pages: int = None,
                 window: int = 0, sinks: int = 0, dtype=None):
        cfg = model.cfg
        if cfg.eng_layers:
            raise ValueError("PagedDecoder: Engram memories keep growing caches (decode them with the KV-cache loop)")
        if model.training:
            raise ValueError("PagedDecoder: put the model in eval mode first (BatchNorm uses its running statistics)")
        max_len = max_len or cfg.max_seq_len
        if max_len > cfg.max_seq_len:
            raise ValueError(f"max_len {max_len} exceeds the model's max_seq_len {cfg.max_seq_len}")
        if window < 0 or sinks < 0 or (sinks and not window):
            raise ValueError(f"window {window}, sinks {sinks}")
        dev = model.tok_emb.weight.device
        if dev.type != "cuda":
            raise ValueError("PagedDecoder runs on CUDA")
        if dtype is None:
            dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else torch.float32
        self.model, self.window, self.sinks = model, window, sinks
        self.cache = PagedKVCache.for_model(model, max_seqs, max_len, page_size, n_pages, dtype)
        self.tokens = torch.zeros(max_seqs, 1, dtype=torch.long, device=dev)  # the next step's input tokens
        self.live = torch.full((max_seqs,), -1, dtype=torch.int32, device=dev)  # row numbers, -1: idle
        self.logits = None       # what follows each row's last token, (max_seqs, 1, vocab); None before the first prefill
        self._graph = None
        self._key = None

    def rows(self):
        """The rows that hold a sequence."""
        return [r for r in range(self.cache.max_seqs) if self.cache.length(r)]

    def _set_live(self):
        on = set(self.rows())
        self.live.copy_(torch.tensor([r if r in on else -1 for r in range(self.cache.max_seqs)], dtype=torch.int32))

    @torch.no_grad()
    def prefill(self, ids, rows):
        """ids (B, P) appended to the sequences `rows` (all of one length: empty ones for prompts); sets their rows of
        self.logits to the last position's and their next tokens to the greedy choice. Returns the logits (B, P, vocab)."""
        rows = list(rows)
        if ids.dim() != 2 or ids.shape[0] != len(rows) or not ids.shape[1]:
            raise ValueError(f"prefill: ids {tuple(ids.shape)} for {len(rows)} sequences")
        if len({self.cache.length(r) for r in self.cache._rows(rows)}) > 1:
            raise ValueError("prefill: the sequences have to be of one length (prefill them one by one)")
        self.cache.extend(rows, ids.shape[1])
        logits = self.model(ids, kv_caches=self.cache.view(rows, self.window, self.sinks).caches())
        at = torch.tensor(rows, device=ids.device)
        self.tokens[at] = logits[:, -1:].argmax(-1)
        if self.logits is None:
            self._make_logits(logits)
        self.logits[at] = logits[:, -1:].to(self.logits.dtype)
        self._trim(rows)
        self._set_live()
        return logits

    def fork(self, parent, children):
        """Every row of `children` becomes a copy of the sequence `parent`, logits and next token included."""
        children = [c for c in children if c != parent]
        if not self.cache.length(parent):
            raise ValueError(f"fork: row {parent} holds no sequence")
        self.cache.fork([parent] * len(children), children)
        at = torch.tensor(children, dtype=torch.long, device=self.tokens.device)
        self.tokens[at] = self.tokens[parent].clone()
        if self.logits is not None:
            self.logits[at] = self.logits[parent].clone()
        self._set_live()

    def reorder(self, parents):
        """Row i becomes a copy of row parents[i], for all rows at once (a beam's selection)."""
        parents = list(parents)
        if len(parents) != self.cache.max_seqs:
            raise ValueError(f"reorder: {len(parents)} parents for {self.cache.max_seqs} rows")
        self.cache.fork(parents, range(len(parents)))
        at = torch.tensor(parents, device=self.tokens.device)
        self.tokens.copy_(self.tokens[at])
        if self.logits is not None:
            self.logits.copy_(self.logits[at])
        self._set_live()

    def free(self, rows):
        """The sequences end."""
        self.cache.free(rows)
        self._set_live()

    def _trim(self, rows):
        if self.window:
            self.cache.trim(rows, self.window, self.sinks)

    def _make_logits(self, like):
        # an ordinary tensor in inference mode too, so that prefill and fork can write its rows at any time
        with torch.inference_mode(False):
            self.logits = torch.zeros(self.cache.max_seqs, 1, like.shape[-1], dtype=like.dtype, device=like.device)

    def _body(self):
        c = self.cache
        pages_extend(c.table, c.lengths, c.refcount, self.live, 1, c.page_size)
        logits = self.model(self.tokens, kv_caches=c.view(None, self.window, self.sinks).caches())
        if self.logits is None or self.logits.dtype != logits.dtype:       # (in the warm-up: every row is written)
            self._make_logits(logits)
        self.logits.copy_(logits)
        self.tokens.copy_(logits[:, -1:].argmax(-1))

    @torch.no_grad()
    def step(self, tokens=None):
        """One step: feeds self.tokens (or `tokens`, (max_seqs, 1)) to every live row and leaves the argmax of the
        logits in self.tokens (returned; self.logits holds the logits; idle rows' entries mean nothing)."""
        rows = self.rows()
        if not rows:
            raise ValueError("PagedDecoder: no sequence to decode (prefill first)")
        if tokens is not None:
            self.tokens.copy_(tokens)
        ac = torch.is_autocast_enabled("cuda")
        key = (ac, torch.get_autocast_dtype("cuda") if ac else None, self.cache.version)
        if self._graph is None or self._key != key:
            self._capture(key)
        self.cache.reserve(rows, 1)
        self._graph.replay()
        if self.window and any(self.cache.length(r) % self.cache.page_size == 0 for r in rows):
            self._trim(rows)
        return self.tokens

    def _capture(self, key):
        """Warm-up passes run with every row idle (they change neither lengths nor pages), then the capture."""
        mems = self.model.memory_layers()
        flags = [getattr(m, "decode_graph", False) for m in mems]
        for m in mems:
            m.decode_graph = False
        ctx = (torch.autocast("cuda", dtype=key[1], cache_enabled=False) if key[0]
               else torch.autocast("cuda", enabled=False))
        dev = self.tokens.device
        saved, live, lengths = self.tokens.clone(), self.live.clone(), self.cache.lengths.clone()
        logits = None if self.logits is None else self.logits.clone()
        try:
            self.live.fill_(-1)
            self.cache.lengths.zero_()
            s = torch.cuda.Stream(dev)
            s.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(s), ctx:
                for _ in range(2):
                    self._body()
            torch.cuda.current_stream(dev).wait_stream(s)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph), ctx:
                self._body()
        finally:
            self.tokens.copy_(saved)
            self.live.copy_(live)
            self.cache.lengths.copy_(lengths)
            if logits is not None:
                self.logits.copy_(logits)
            for m, f in zip(mems, flags):
                m.decode_graph = f
        self._graph, self._key = graph, key
