"""Ragged batches over a paged KV cache, on MI355X: what the cached denoising
step (kv_cache.attention_inputs, then the decode attention) is for a
rectangular batch, for sequences of any lengths that share one pool of pages.

`PagedKVCache` holds the pool and hands its pages to sequences; `batch(...)`
describes one step of some of them (a token, a block or a chunk of a prompt
each), and

    q = batch.attention_inputs(qkv, n_heads, sin_table, cos_table, layer)
    o = batch.attention(q, layer, block_size)

run a layer's attention for all of them, in two launches (three where the keys
are cut over workgroups). `paged_attention_inputs` and `paged_attention` are the
same calls on a caller's own pool, tables and lengths.

The pages may hold 8-bit codes with scales (`paged_attention_inputs8`, `paged_attention_pool`): half the
memory, half the bytes that the attention reads. And a step may read only the pages that promise
most for its queries, by bounds of each page's keys (`page_bounds`, `select_pages`,
`batch.attention(..., top=)`): its time no longer grows with the cache.

Tokens are packed: sequence b owns rows q_starts[b] .. q_starts[b + 1] - 1 of
every (tokens, ...) tensor. Its token i is at position kv_lens[b] - n + i, n the
chunk's tokens, and sees the keys up to the end of its block of block_size
positions (block_size 1: causal), at most kv_lens[b] of them: the rule of
block_sparse_decode_attention. Heads may share KV heads (n_heads a multiple of
the pool's).

Everything a call reads of the batch is on the device, so a captured graph may
be replayed with other lengths, tables and starts, within the bounds (max_q,
max_kv) it was captured with.
"""
from __future__ import annotations

import torch
from torch import Tensor

from kernels._native import host

D = 64
BLOCK = 16  # slots that share a scale


def paged_attention(
    q: Tensor,           # (tokens, heads, 64) bf16
    k_pages: Tensor,     # (pages, kv_heads, page_size, 64) bf16
    v_pages: Tensor,
    page_table: Tensor,  # (seqs, width) int32: the page of keys j // page_size == column
    q_starts: Tensor,    # (seqs + 1) int32, ascending
    kv_lens: Tensor,     # (seqs) int32, the chunk's tokens included
    block_size: int,
    max_q: int,                  # tokens of the longest chunk, or more
    max_kv: int | None = None,   # keys of the longest sequence, or more (default: the table's)
    total_kv: int | None = None,  # about the sum of kv_lens: decides how the work is cut
    out: Tensor | None = None,
) -> Tensor:
    """Attention of each sequence's chunk over its pages: (tokens, heads, 64).
    A token that sees no key gets 0. Rows of `out` behind the last sequence are
    left as they are (without `out` they are undefined). Keys of table entries
    that are no page (negative, or past the pool) are not seen. Slots past a
    sequence's keys may hold anything; its keys and values themselves must be
    finite, also those that only later tokens of the chunk see (their weights are
    zeros that multiply them). `out` overlaps no input."""
    return host().paged_attention(q, k_pages, v_pages, page_table, q_starts, kv_lens, block_size, max_q,
                                  -1 if max_kv is None else max_kv, -1 if total_kv is None else total_kv, out,
                                  None, None, None)


def paged_attention_inputs(
    qkv: Tensor,         # (tokens, (n_heads + 2 * kv_heads) * 64) bf16: q heads, k heads, v heads
    n_heads: int,
    sin_table: Tensor,   # (max_seq_len, 32) float32 (kv_cache.rope_tables)
    cos_table: Tensor,
    k_pages: Tensor,     # as in paged_attention; written at the tokens' positions
    v_pages: Tensor,
    page_table: Tensor,
    q_starts: Tensor,
    kv_lens: Tensor,
    out: Tensor | None = None,
) -> Tensor:
    """The rotated queries (tokens, n_heads, 64); rotated keys and values go to
    their slots in the pages. Computed in fp32 and rounded once, so a key
    differs from kv_cache.attention_inputs' (which repeats the eager path's bf16
    roundings) by up to two of its last bits. Positions beyond the RoPE tables
    use their last row; nothing is written where the table has no page. out,
    k_pages and v_pages overlap neither each other nor another argument."""
    return host().paged_attention_inputs(qkv, n_heads, sin_table, cos_table, k_pages, v_pages, page_table, q_starts,
                                         kv_lens, out, None, None)


def paged_attention_pool(
    q: Tensor,           # (tokens, heads, 64) bf16
    k_pages: Tensor,     # (pages, kv_heads, page_size, 64) bf16, int8 or float8_e4m3fn
    v_pages: Tensor,
    page_table: Tensor,
    q_starts: Tensor,
    kv_lens: Tensor,
    block_size: int,
    max_q: int,
    max_kv: int | None = None,
    total_kv: int | None = None,
    out: Tensor | None = None,
    k_scales: Tensor | None = None,  # of 8-bit pages: (pages, kv_heads, page_size // 16) float32, contiguous
    v_scales: Tensor | None = None,
    columns: Tensor | None = None,   # (tokens, kv_heads, top) int32 (select_pages)
) -> Tensor:
    """paged_attention over any kind of pool, and over selected pages.

    8-bit pages hold codes, value = scale * code with a scale for each 16 slots and
    head (paged_attention_inputs8 writes them); the scales of blocks that hold keys must
    be finite and at least 2 ** -100 (and values below about 2 ** 100: the sums over keys are fp32). Codes enter the products exactly, scales multiply
    scores and probabilities in fp32: the result is as near to the values as
    paged_attention's is to its bf16 ones.

    With `columns` the tokens of one block of block_size positions read, as far as they see them,
    only the pages in the table's columns columns[first of them in the chunk, KV head]. Of a list the
    first ceil(length / page_size) places are read (the sequence has no more columns with keys, and none
    may occur twice): a column behind them is not, also where some of them hold none. An entry that is no
    column that the block sees (-1) names nothing."""
    return host().paged_attention(q, k_pages, v_pages, page_table, q_starts, kv_lens, block_size, max_q,
                                  -1 if max_kv is None else max_kv, -1 if total_kv is None else total_kv, out,
                                  k_scales, v_scales, columns)


def paged_attention_inputs8(
    qkv: Tensor,         # as in paged_attention_inputs
    n_heads: int,
    sin_table: Tensor,
    cos_table: Tensor,
    k_pages: Tensor,     # (pages, kv_heads, page_size, 64) int8 or float8_e4m3fn; written
    v_pages: Tensor,
    k_scales: Tensor,    # (pages, kv_heads, page_size // 16) float32, contiguous; written
    v_scales: Tensor,
    page_table: Tensor,
    q_starts: Tensor,
    kv_lens: Tensor,
    out: Tensor | None = None,
) -> Tensor:
    """paged_attention_inputs into 8-bit pages. Each 16 slots (a block: slots 16 i to
    16 i + 15 of a page) and head take a scale: the one that their new values need
    (max|x| / 127, or for float8_e4m3fn the least power of two with 448 * scale >=
    max|x|; at least 2 ** -100), or, if the block holds earlier tokens of the sequence, its
    scale times the least power of two with which the new values fit; the block's
    other codes are then rounded to the new scale. A new value is off by at most half
    a step (the scale, or the spacing of e4m3 there); an earlier one in the
    end by less than one step.

    A block that holds earlier tokens keeps a scale that uncommitted ones, since overwritten,
    have raised. Values must be finite. Blocks are written whole: no two sequences of a
    call may write into the same one. No written tensor overlaps another argument."""
    return host().paged_attention_inputs(qkv, n_heads, sin_table, cos_table, k_pages, v_pages, page_table, q_starts,
                                         kv_lens, out, k_scales, v_scales)


def page_values(k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor) -> tuple[Tensor, Tensor]:
    """The values that 8-bit pages hold, as bf16 (pages, kv_heads, page_size, 64) each."""
    return host().page_values(k_pages, v_pages, k_scales, v_scales)


def page_bounds(
    k_pages: Tensor,     # as in paged_attention_pool
    bounds: Tensor,      # (pages, kv_heads, 2, 64) bf16, contiguous: the lowest, the highest key of each channel; written
    page_table: Tensor,
    q_starts: Tensor,
    kv_lens: Tensor,
    tokens: int,         # packed tokens of the batch
    k_scales: Tensor | None = None,
) -> Tensor:
    """Form the bounds of the pages that hold tokens of the chunks anew, over all
    keys that the sequence has in them; returns `bounds`. Other pages' stay, so after the
    call that writes a chunk's final keys this keeps the bounds of a sequence's pages."""
    return host().page_bounds(k_pages, bounds, page_table, q_starts, kv_lens, tokens, k_scales)


def select_pages(
    q: Tensor,           # (tokens, heads, 64) bf16
    bounds: Tensor,      # (pages, kv_heads, 2, 64) bf16 (page_bounds)
    page_table: Tensor,
    q_starts: Tensor,
    kv_lens: Tensor,
    block_size: int,
    page_size: int,
    top: int,            # pages for each block of queries and KV head
    max_q: int,
    max_kv: int | None = None,
    first: int = 1,      # columns always taken: the first ones,
    recent: int = 1,     # and those before the block's own
    out: Tensor | None = None,
) -> Tensor:
    """The pages that paged_attention_pool is to read, (tokens, kv_heads, top) int32
    columns of the page table, ascending, then -1. The tokens of one block of
    block_size positions choose together for each KV head: the first `first` columns,
    those that hold positions of the block and the `recent` before them, and of the others
    that they see the ones with the largest

        max over the block's tokens and the KV head's query heads of
        sum_d max(q_d * lowest_d, q_d * highest_d),

    which no key of the page exceeds in q . k (of 8-bit pages but for the bounds' rounding to bf16); equals by the lower column. The
    scores' order is exact. `top` must leave room for the columns always taken. Rows behind the last
    sequence are left as they are (without `out` undefined). Bounds of the columns always taken may
    be anything; those of the others must be finite."""
    return host().select_pages(q, bounds, page_table, q_starts, kv_lens, block_size, page_size, top, max_q,
                               -1 if max_kv is None else max_kv, first, recent, out)


class PagedKVCache:
    """A pool of pages for the post-RoPE keys and values of many sequences, the
    same page numbers in every layer, in bf16 or in 8 bits (`dtype`: int8 or
    float8_e4m3fn, with scales), with bounds of each page's keys for attention over selected
    pages (`bounds`). Host-side bookkeeping: a sequence is the int that `add`
    returned, until `free`."""

    def __init__(self, n_layers: int, n_pages: int, kv_heads: int, page_size: int = 64,
                 device: torch.device | str = "cuda", dtype: torch.dtype = torch.bfloat16, bounds: bool = False):
        assert n_layers >= 1 and n_pages >= 1 and kv_heads >= 1, "need at least one layer, page and KV head"
        assert 16 <= page_size <= 1024 and page_size & (page_size - 1) == 0, \
            "page_size must be a power of two in [16, 1024]"
        self.page_size = page_size
        shape = (n_layers, n_pages, kv_heads, page_size, D)
        assert dtype in (torch.bfloat16, torch.int8, torch.float8_e4m3fn), \
            "pages hold bfloat16, int8 or float8_e4m3fn"
        self.k_pages = torch.empty(shape, device=device, dtype=dtype)
        self.v_pages = torch.empty(shape, device=device, dtype=dtype)
        self.k_scales = self.v_scales = self.bounds = None
        if dtype != torch.bfloat16:  # 0: no scale yet
            self.k_scales = torch.zeros((*shape[:3], page_size // BLOCK), device=device)
            self.v_scales = torch.zeros_like(self.k_scales)
        if bounds:
            self.bounds = torch.zeros((*shape[:3], 2, D), device=device, dtype=torch.bfloat16)
        # of each layer: how many of a sequence's first tokens the bounds of its pages cover
        self._bounded: list[dict[int, int]] = [{} for _ in range(n_layers)]
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next = 0

    def scales(self, layer: int) -> tuple[Tensor | None, Tensor | None]:
        """(k_scales, v_scales) of a layer's 8-bit pages; (None, None) in bf16."""
        return (None, None) if self.k_scales is None else (self.k_scales[layer], self.v_scales[layer])

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def add(self) -> int:
        """A new sequence without tokens."""
        seq = self._next
        self._next += 1
        self._pages[seq], self._length[seq] = [], 0
        return seq

    def length(self, seq: int) -> int:
        """Committed tokens of a sequence."""
        return self._length[seq]

    def free(self, seq: int) -> None:
        """Give a sequence's pages back to the pool. The next batch may take them: what
        still runs on them must be before it in stream order."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._length[seq]
        for covered in self._bounded:
            covered.pop(seq, None)

    def batch(self, seqs: list[int], new_tokens: list[int]) -> "PagedBatch":
        """One step of these sequences, new_tokens[i] tokens of seqs[i] after its
        committed ones; pages are taken from the pool as needed (RuntimeError,
        nothing taken, if it has too few). Until `commit` the next batch of a
        sequence overwrites the step's keys and values."""
        assert len(seqs) == len(new_tokens), "one token count per sequence"
        assert len(set(seqs)) == len(seqs), "a sequence occurs once in a batch"
        assert all(s in self._pages for s in seqs), "unknown sequence"
        assert all(n >= 0 for n in new_tokens), "token counts must be >= 0"
        lens = [self._length[s] + n for s, n in zip(seqs, new_tokens)]
        more = [max(0, -(-kv // self.page_size) - len(self._pages[s])) for s, kv in zip(seqs, lens)]
        if sum(more) > len(self._free):
            raise RuntimeError(f"the pool has {len(self._free)} free pages, the batch needs {sum(more)}")
        for s, n in zip(seqs, more):
            self._pages[s].extend(self._free.pop() for _ in range(n))
        return PagedBatch(self, list(seqs), list(new_tokens), lens)


class PagedBatch:
    """One step of some sequences of a PagedKVCache: the device arrays that
    paged_attention takes, their bounds, and the two calls with them."""

    def __init__(self, cache: PagedKVCache, seqs: list[int], new_tokens: list[int], lens: list[int]):
        self.cache, self.seqs, self.new_tokens, self.lens = cache, seqs, new_tokens, lens
        self.tokens = sum(new_tokens)
        self.max_q, self.max_kv, self.total_kv = max(new_tokens, default=0), max(lens, default=0), sum(lens)
        width = max(1, -(-self.max_kv // cache.page_size))
        starts = [0]
        for n in new_tokens:
            starts.append(starts[-1] + n)
        rows = [cache._pages[s][:width] for s in seqs]
        table = [p for r in rows for p in r + [-1] * (width - len(r))]
        # one copy to the device for the three
        data = torch.tensor(starts + lens + table, dtype=torch.int32).to(cache.k_pages.device)
        n = len(seqs)
        self.q_starts, self.kv_lens = data[:n + 1], data[n + 1:2 * n + 1]
        self.page_table = data[2 * n + 1:].view(n, width)
        self._committed = False
        self._formed: set[int] = set()  # layers whose bounds cover this step
        self._checked: set[tuple] = set()  # selections whose bounds are known to be there

    def attention_inputs(self, qkv: Tensor, n_heads: int, sin_table: Tensor, cos_table: Tensor, layer: int,
                         out: Tensor | None = None) -> Tensor:
        """paged_attention_inputs, or paged_attention_inputs8, into this layer's pages."""
        c = self.cache
        k_scales, v_scales = c.scales(layer)
        return host().paged_attention_inputs(qkv, n_heads, sin_table, cos_table, c.k_pages[layer], c.v_pages[layer],
                                             self.page_table, self.q_starts, self.kv_lens, out, k_scales, v_scales)

    def update_bounds(self, layer: int) -> None:
        """page_bounds of the pages that hold this step's tokens: after the attention_inputs
        whose tokens are committed, and before an attention over selected pages
        if the step has more than one block of a sequence. (The pages of a query's own block are
        taken whatever their bounds.)"""
        c = self.cache
        assert c.bounds is not None, "the cache keeps no bounds: PagedKVCache(..., bounds=True)"
        page_bounds(c.k_pages[layer], c.bounds[layer], self.page_table, self.q_starts, self.kv_lens, self.tokens,
                    c.scales(layer)[0])
        self.bounds_formed(layer)

    def bounds_formed(self, layer: int) -> None:
        """Count this step's bounds in a layer as formed, as update_bounds does. For a caller whose replayed graph, or
        page_bounds itself, formed them."""
        layer = range(len(self.cache._bounded))[layer]  # -1: the last one, as for the tensors
        self._formed.add(layer)
        if self._committed:
            self._count_bounds(layer)

    def _covers(self, layer: int, seq: int, start: int) -> bool:
        """Whether the pages before the one that holds position `start` have their bounds."""
        page = self.cache.page_size
        return self.cache._bounded[layer].get(seq, 0) >= start // page * page

    def _count_bounds(self, layer: int) -> None:
        c = self.cache
        for s, n, kv in zip(self.seqs, self.new_tokens, self.lens):
            if n > 0 and s in c._length and self._covers(layer, s, kv - n):
                c._bounded[layer][s] = kv  # less than before if later tokens are there: the last page was formed without them

    def _check_bounds(self, layer: int, block_size: int, top: int, first: int, recent: int) -> None:
        """The pages that the last block of each sequence ranks, and earlier ones a part of, have bounds over all of their keys."""
        c = self.cache
        for s, n, kv in zip(self.seqs, self.new_tokens, self.lens):
            if n == 0 or -(-kv // c.page_size) <= top:
                continue
            ranked = (kv - 1) // block_size * block_size // c.page_size - recent  # [first, ranked)
            have = kv if layer in self._formed and self._covers(layer, s, kv - n) else c._bounded[layer].get(s, 0)
            assert ranked <= first or have >= ranked * c.page_size, \
                f"layer {layer}, sequence {s}: page bounds cover {have} of the {ranked * c.page_size} tokens whose pages are to be " \
                "ranked: update_bounds in every step that is committed, and before a step of several blocks selects"

    def attention(self, q: Tensor, layer: int, block_size: int, out: Tensor | None = None, top: int | None = None,
                  first: int = 1, recent: int = 1) -> Tensor:
        """paged_attention over this layer's pages; with `top` over those that select_pages
        takes by the cache's bounds, refused (AssertionError) while bounds that it ranks by have not been formed
        (update_bounds)."""
        c = self.cache
        columns = None
        if top is not None:
            assert c.bounds is not None, "the cache keeps no bounds: PagedKVCache(..., bounds=True)"
            asked = range(len(c._bounded))[layer], block_size, top, first, recent
            if asked not in self._checked:
                if block_size >= 1:  # else the call refuses it
                    self._check_bounds(*asked)
                self._checked.add(asked)
            columns = select_pages(q, c.bounds[layer], self.page_table, self.q_starts, self.kv_lens, block_size,
                                   c.page_size, top, self.max_q, self.max_kv, first, recent)
        k_scales, v_scales = c.scales(layer)
        return host().paged_attention(q, c.k_pages[layer], c.v_pages[layer], self.page_table, self.q_starts, self.kv_lens,
                                      block_size, self.max_q, self.max_kv, self.total_kv, out, k_scales, v_scales, columns)

    def commit(self) -> None:
        """Count the step's tokens as committed, in every layer. Once a batch,
        and only while its sequences hold what they held when it was made."""
        c = self.cache
        for s, n, kv in zip(self.seqs, self.new_tokens, self.lens):
            assert c._length.get(s) == kv - n, "the sequence has moved on since this batch was made"
        for s, kv in zip(self.seqs, self.lens):
            c._length[s] = kv
        self._committed = True
        for layer in self._formed:
            self._count_bounds(layer)
