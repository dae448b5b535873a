"""Plain 64-bit and pure-Python forms of the paged cache's operators, for the tests."""
import math

import torch


def visible_tokens(n, window, sinks, entries, page):
    """Positions of a sequence of n tokens that a query sees (entries: its table row)."""
    return [j for j in range(n) if (window == 0 or j >= n - window or j < sinks) and entries[j // page] >= 0]


def attention(q, k_pages, v_pages, table, lengths, scale, window=0, sinks=0):
    """out, lse, and what the error bound needs: mag = sum p |v| and reach = max sum |q k| |scale|, all float64 on the
    CPU. Reads the visible tokens one sequence at a time."""
    B, HQ, D = q.shape
    HKV, page = k_pages.shape[1], k_pages.shape[2]
    g = HQ // HKV
    out = torch.zeros(B, HQ, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((B, HQ), -math.inf, dtype=torch.float64)
    reach = torch.zeros(B, HQ, 1, dtype=torch.float64)
    tab = table.cpu().tolist()
    for b, n in enumerate(lengths.cpu().tolist()):
        at = visible_tokens(n, window, sinks, tab[b], page)
        if not at:
            continue
        pages = torch.tensor([tab[b][j // page] for j in at], device=k_pages.device)
        slots = torch.tensor([j % page for j in at], device=k_pages.device)
        k, v = (x[pages, :, slots].double().cpu() for x in (k_pages, v_pages))       # (n, HKV, D)
        for h in range(HQ):
            qh = q[b, h].double().cpu()
            s = (k[:, h // g] @ qh) * scale
            if bool((s == -math.inf).all()):
                continue
            p = torch.softmax(s, 0)
            out[b, h] = p @ v[:, h // g]
            lse[b, h] = torch.logsumexp(s, 0)
            mag[b, h] = p @ v[:, h // g].abs()
            reach[b, h] = (k[:, h // g].abs() @ qh.abs()).max() * abs(scale)
    return out, lse, mag, reach


# unit roundoffs of the types (half a unit in the last place of 8-, 11- and 24-bit significands)
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def attention_bound(out, mag, reach, dtype, longest):
    """How far the kernel may be from `out`.

    * the result is rounded once to the type: u |out| (fp16 also has subnormals: 2^-25);
    * the weights p may be rounded once to a 16-bit type before they meet v: u each, so u mag;
    * a score is a sum of d <= 256 products in fp32 (fp32 inputs: split into two parts of 11 bits or more, whose
      dropped product is below 2^-21): off by at most 2^-16 reach for 16-bit inputs and 2^-19 reach for fp32, which
      changes p by that factor and, through the sum, out by twice it;
    * exp, the maxima's rescaling and the fp32 sums over `longest` tokens: 2^-20 + longest 2^-24."""
    u = UNIT[dtype]
    score = 2.0 ** -19 if dtype == torch.float32 else 2.0 ** -16
    p = 0.0 if dtype == torch.float32 else u
    return u * out.abs() + mag * (p + 2 * score * reach + 2.0 ** -20 + longest * 2.0 ** -24) + 2.0 ** -25


def rotary(d, n):
    freq = 1.0 / 10000.0 ** (torch.arange(0, d, 2, dtype=torch.float32) / d)
    angle = torch.arange(n, dtype=torch.float32)[:, None] * freq[None]
    return angle.cos(), angle.sin()


def append(qkv, k_pages, v_pages, table, lengths, cos, sin):
    """float64 q, and the pages after the call (copies; CPU)."""
    B, T, W = qkv.shape
    HKV, page, D = k_pages.shape[1:]
    HQ = W // D - 2 * HKV
    k, v = k_pages.double().cpu().clone(), v_pages.double().cpu().clone()
    q = torch.zeros(B, T, HQ, D, dtype=torch.float64)
    x = qkv.double().cpu().view(B, T, HQ + 2 * HKV, D)
    for b, n in enumerate(lengths.tolist()):
        for t in range(T):
            pos = n - T + t
            if pos < 0:
                continue
            y = x[b, t].clone()
            if cos is not None:
                c, s = cos[pos].double().cpu(), sin[pos].double().cpu()
                a, e = y[:HQ + HKV, :D // 2].clone(), y[:HQ + HKV, D // 2:].clone()
                y[:HQ + HKV, :D // 2] = a * c - e * s
                y[:HQ + HKV, D // 2:] = e * c + a * s
            q[b, t] = y[:HQ]
            p = int(table[b, pos // page])
            if p < 0:
                continue
            k[p, :, pos % page] = y[HQ:HQ + HKV]
            v[p, :, pos % page] = y[HQ + HKV:]
    return q, k, v


class Book:
    """The page operations on plain lists; contents: one value per (page, slot)."""

    def __init__(self, rows, blocks, pages, page):
        self.page, self.blocks = page, blocks
        self.table = [[-1] * blocks for _ in range(rows)]
        self.len = [0] * rows
        self.ref = [0] * pages
        self.data = [[0.0] * page for _ in range(pages)]

    def take(self):
        p = self.ref.index(0)
        self.ref[p] = 1
        return p

    def _drop(self, r, j):
        p = self.table[r][j]
        if p >= 0:
            self.ref[p] -= 1
            self.table[r][j] = -1

    def free(self, rows):
        for r in rows:
            for j in range(self.blocks):
                self._drop(r, j)
            self.len[r] = 0

    def trim(self, rows, window, sinks):
        for r in rows:
            for j in range(self.blocks):
                if j * self.page >= sinks and (j + 1) * self.page <= self.len[r] - window:
                    self._drop(r, j)

    def extend(self, rows, n):
        for r in rows:
            a, b = -(-self.len[r] // self.page), -(-(self.len[r] + n) // self.page)
            for j in range(a, b):
                self.table[r][j] = self.take()
            self.len[r] += n

    def fork(self, parents, children):
        old = [(list(self.table[p]), self.len[p]) for p in parents]
        act = [i for i in range(len(parents)) if parents[i] != children[i]]
        parts = {}
        for i in act:
            row, n = old[i]
            for j in range(n // self.page):
                if row[j] >= 0:
                    self.ref[row[j]] += 1
            if n % self.page and row[n // self.page] >= 0:
                parts[i] = row[n // self.page]
                self.ref[parts[i]] += 1
        for i in act:
            self.free([children[i]])
        for i in act:
            row, n = old[i]
            new = [row[j] if j < n // self.page else -1 for j in range(self.blocks)]
            if i in parts:
                p = self.take()
                new[n // self.page] = p
                self.data[p][:n % self.page] = self.data[parts[i]][:n % self.page]
            self.table[children[i]], self.len[children[i]] = new, n
        for p in parts.values():
            self.ref[p] -= 1

    def compact(self):
        n = sum(x > 0 for x in self.ref)
        low = [p for p in range(n) if self.ref[p] == 0]
        high = [p for p in range(n, len(self.ref)) if self.ref[p] > 0]
        to = dict(zip(high, low))
        for s, d in to.items():
            self.ref[d], self.ref[s] = self.ref[s], 0
            self.data[d] = list(self.data[s])
        self.table = [[to.get(p, p) for p in row] for row in self.table]
