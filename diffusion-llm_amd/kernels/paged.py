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
                                  -1 if max_kv is None else max_kv, -1 if total_kv is None else total_kv, out)


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
                                         kv_lens, out)


class PagedKVCache:
    """A pool of pages for the post-RoPE keys and values of many sequences, the
    same page numbers in every layer. Host-side bookkeeping: a sequence is the
    int that `add` returned, until `free`."""

    def __init__(self, n_layers: int, n_pages: int, kv_heads: int, page_size: int = 64,
                 device: torch.device | str = "cuda"):
        assert n_layers >= 1 and n_pages >= 1 and kv_heads >= 1, "need at least one layer, page and KV head"
        assert 16 <= page_size <= 1024 and page_size & (page_size - 1) == 0, \
            "page_size must be a power of two in [16, 1024]"
        self.page_size = page_size
        shape = (n_layers, n_pages, kv_heads, page_size, D)
        self.k_pages = torch.empty(shape, device=device, dtype=torch.bfloat16)
        self.v_pages = torch.empty(shape, device=device, dtype=torch.bfloat16)
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next = 0

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

    def attention_inputs(self, qkv: Tensor, n_heads: int, sin_table: Tensor, cos_table: Tensor, layer: int,
                         out: Tensor | None = None) -> Tensor:
        """paged_attention_inputs into this layer's pages."""
        c = self.cache
        return paged_attention_inputs(qkv, n_heads, sin_table, cos_table, c.k_pages[layer], c.v_pages[layer],
                                      self.page_table, self.q_starts, self.kv_lens, out)

    def attention(self, q: Tensor, layer: int, block_size: int, out: Tensor | None = None) -> Tensor:
        """paged_attention over this layer's pages."""
        c = self.cache
        return paged_attention(q, c.k_pages[layer], c.v_pages[layer], self.page_table, self.q_starts, self.kv_lens,
                               block_size, self.max_q, self.max_kv, self.total_kv, out)

    def commit(self) -> None:
        """Count the step's tokens as committed, in every layer. Once a batch,
        and only while its sequences hold what they held when it was made."""
        c = self.cache
        for s, n, kv in zip(self.seqs, self.new_tokens, self.lens):
            assert c._length.get(s) == kv - n, "the sequence has moved on since this batch was made"
        for s, kv in zip(self.seqs, self.lens):
            c._length[s] = kv
