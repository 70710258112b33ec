"""Operators that make the cached keys and values of a ragged serving step
cheaper to keep and to read, in plain form and as this library's kernels: a
paged cache held in 8 bits, and attention over the pages that a score of each
page's bounds selects.

A case is a dict of plain values; `kind` names the operator:

  append     split + RoPE of the chunk's projection, keys and values written into
             pages of 8-bit codes with a scale for each 16 slots and head
             (paged_attention_inputs8), and the pages read back
             (page_values)
  cache8     attention of each sequence's chunk over such pages, block-causal
             (paged_attention_pool)
  select     the bounds of the pages that the chunk wrote (page_bounds) and the
             pages that each query's attention is to read (select_pages)
  sparse     attention over the selected pages (paged_attention_pool with columns)

Chunks hold q_lo .. q_hi tokens and come after ctx_lo .. ctx_hi cached ones, a
length per sequence, spread over their logarithm. Heads are 64 wide and queries
bf16, as everywhere in this library; sizes are those of its tests, of bench.py
and of its sampling workload, with longer caches for the selected pages.
"""
import math
import os
import random
import sys

import torch

own = False

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
D = 64
BLOCK = 16  # slots of a page that share a scale
_CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
SMALLEST = 2.0 ** -100  # of a scale


def listed():
    return [
        # A token of each of a few sequences into a cache in use: launches and host work count.
        {"name": "append_token", "kind": "append", "type": "int8", "seqs": 4, "heads": 12, "kv_heads": 12, "q_lo": 1,
         "q_hi": 1, "ctx_lo": 100, "ctx_hi": 300, "page": 64},
        # The denoising step of a served batch.
        {"name": "append_batch", "kind": "append", "type": "e4m3", "seqs": 32, "heads": 12, "kv_heads": 12, "q_lo": 32,
         "q_hi": 32, "ctx_lo": 50, "ctx_hi": 2000, "page": 64},
        # Chunks of prompts, shared key heads, small pages, chunks that begin and end inside a block of slots.
        {"name": "append_chunks", "kind": "append", "type": "int8", "seqs": 24, "heads": 16, "kv_heads": 4, "q_lo": 100,
         "q_hi": 2000, "ctx_lo": 1, "ctx_hi": 700, "page": 16},
        # One sequence's denoising step over a cache of 3584.
        {"name": "cache8_single", "kind": "cache8", "type": "int8", "seqs": 1, "heads": 12, "kv_heads": 12, "q_lo": 16,
         "q_hi": 16, "ctx_lo": 3584, "ctx_hi": 3584, "page": 64, "bs": 16},
        # The denoising step of a served batch: sequences of very different ages.
        {"name": "cache8_batch", "kind": "cache8", "type": "int8", "seqs": 32, "heads": 12, "kv_heads": 12, "q_lo": 16,
         "q_hi": 16, "ctx_lo": 100, "ctx_hi": 8192, "page": 64, "bs": 16},
        # Three query heads to a key head and blocks of 32, small pages.
        {"name": "cache8_shared", "kind": "cache8", "type": "e4m3", "seqs": 24, "heads": 12, "kv_heads": 4, "q_lo": 32,
         "q_hi": 32, "ctx_lo": 500, "ctx_hi": 4000, "page": 16, "bs": 32},
        # Whole prompts of up to 4096 tokens, nothing cached.
        {"name": "cache8_prompts", "kind": "cache8", "type": "int8", "seqs": 4, "heads": 12, "kv_heads": 12,
         "q_lo": 1500, "q_hi": 4096, "ctx_lo": 0, "ctx_hi": 0, "page": 128, "bs": 32},
        # One token of one long sequence: its page's bounds and the pages it reads.
        {"name": "select_token", "kind": "select", "type": "bf16", "seqs": 1, "heads": 12, "kv_heads": 4, "q_lo": 1,
         "q_hi": 1, "ctx_lo": 16000, "ctx_hi": 16000, "page": 16, "bs": 1, "top": 64},
        # A batch's blocks over long caches.
        {"name": "select_batch", "kind": "select", "type": "int8", "seqs": 32, "heads": 12, "kv_heads": 12, "q_lo": 16,
         "q_hi": 16, "ctx_lo": 2000, "ctx_hi": 16000, "page": 32, "bs": 16, "top": 32},
        # The attention of that token, and of such a batch.
        {"name": "sparse_token", "kind": "sparse", "type": "bf16", "seqs": 1, "heads": 12, "kv_heads": 4, "q_lo": 1,
         "q_hi": 1, "ctx_lo": 16000, "ctx_hi": 16000, "page": 16, "bs": 1, "top": 64},
        {"name": "sparse_batch", "kind": "sparse", "type": "bf16", "seqs": 32, "heads": 12, "kv_heads": 12, "q_lo": 16,
         "q_hi": 16, "ctx_lo": 2000, "ctx_hi": 16000, "page": 32, "bs": 16, "top": 32},
        # Chunks of several blocks, each block with pages of its own, in 8 bits.
        {"name": "sparse_chunks", "kind": "sparse", "type": "int8", "seqs": 8, "heads": 12, "kv_heads": 4, "q_lo": 40,
         "q_hi": 300, "ctx_lo": 2000, "ctx_hi": 12000, "page": 32, "bs": 16, "top": 40},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "cache8", "cache8", "cache8", "cache8", "select", "select", "sparse",
                       "sparse", "sparse"])
    heads, kv_heads = rng.choice([(12, 12), (12, 12), (12, 4), (16, 2), (8, 8), (12, 1), (6, 3)])
    case = {"kind": kind, "type": rng.choice(["int8", "e4m3"]), "heads": heads, "kv_heads": kv_heads}
    if kind == "append":
        q_hi = _log(rng, 1, 2000)
        ctx_hi = _log(rng, 1, 1500)
        return {**case, "seqs": _log(rng, 1, max(1, min(48, 16000 // (q_hi + ctx_hi // 2)))),
                "q_lo": max(1, q_hi // rng.choice([1, 3, 20])), "q_hi": q_hi, "ctx_lo": 0, "ctx_hi": ctx_hi,
                "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "cache8":
        page = rng.choice([16, 32, 64, 128, 256])
        if rng.random() < 0.65:  # a token or a block of each sequence
            block = rng.choice([1, 4, 5, 8, 16, 16, 32, 64])
            ctx_hi = _log(rng, 20, 8192)
            return {**case, "seqs": _log(rng, 1, max(1, min(48, 100000 // ctx_hi))), "q_lo": block, "q_hi": block,
                    "ctx_lo": max(1, ctx_hi // rng.choice([1, 2, 30])), "ctx_hi": ctx_hi, "page": page, "bs": block}
        q_hi = _log(rng, 20, 2000)
        ctx_hi = _log(rng, 1, 6000)
        return {**case, "seqs": _log(rng, 1, max(1, min(16, 8000000 // (q_hi * (q_hi + ctx_hi))))),
                "q_lo": max(1, q_hi // rng.choice([1, 4, 50])), "q_hi": q_hi, "ctx_lo": rng.choice([0, ctx_hi]),
                "ctx_hi": ctx_hi, "page": page, "bs": rng.choice([1, 4, 7, 16, 32, 64])}
    # pages selected: a token or a block of each sequence, or a short chunk of several
    case["type"] = rng.choice(["bf16", "int8", "e4m3"])
    bs = rng.choice([1, 1, 4, 7, 16, 16, 32])
    q_hi = bs if rng.random() < 0.7 else _log(rng, bs, 200)
    page = rng.choice([16, 32, 64, 128])
    top = _log(rng, 5, 100)
    ctx_hi = _log(rng, 300, 20000)
    if (q_hi // bs + 1) * kv_heads * top * page > 1500000:
        q_hi = bs
    fits = min(120000 // ctx_hi, 1500000 // ((q_hi // bs + 1) * kv_heads * top * page))
    return {**case, "seqs": _log(rng, 1, max(1, min(48, fits))), "q_lo": max(1, q_hi // rng.choice([1, 1, 3])),
            "q_hi": q_hi, "ctx_lo": max(1, ctx_hi // rng.choice([1, 2, 10])), "ctx_hi": ctx_hi, "page": page, "bs": bs,
            "top": top}


def _lengths(case):
    """(chunk, context) lengths of each sequence: of the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))

    def one(lo, hi):
        return lo if lo == hi else _log(rng, max(lo, 1), hi)

    return [(one(case["q_lo"], case["q_hi"]), one(case["ctx_lo"], case["ctx_hi"])) for _ in range(case["seqs"])]


# ---------------------------------------------------------------------------
# inputs


def _randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _needed(top, kind):
    """The scale that values of up to `top` need."""
    if kind == "int8":
        return (top / 127.0).clamp(min=SMALLEST)
    m, e = torch.frexp(top)  # m in [0.5, 1): 448 = 0.875 * 2 ** 9
    return torch.where(top > 0, _power(e - 9 + (m > 0.875).int()), 0.0).clamp(min=SMALLEST)


def _power(e):
    """2 ** e, exactly."""
    return ((e.clamp(-126, 127) + 127) << 23).to(torch.int32).view(F32)


def _encode(x, scale, kind):
    dtype, most = _CODES[kind]
    y = (x / scale).clamp(-most, most)
    return torch.round(y).to(dtype) if dtype == torch.int8 else y.to(dtype)


def _pool(g, pages, kv_heads, page, kind, drift):
    """Pages of random keys or values, and their scales (None in bf16). With `drift` the heads' channels have a mean that
    wanders from page to page, as keys of a text do."""
    x = torch.randn((pages, kv_heads, page, D), generator=g, device="cuda")
    if drift:
        x += 1.5 * torch.randn((pages, kv_heads, 1, D), generator=g, device="cuda")
    if kind == "bf16":
        return x.to(BF), None
    b = x.view(pages, kv_heads, page // BLOCK, BLOCK, D)
    scales = _needed(b.abs().amax(dim=(3, 4)), kind)
    return _encode(b, scales[..., None, None], kind).view(x.shape), scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    lens = _lengths(case)
    n = [q for q, _ in lens]
    kv = [q + c for q, c in lens]
    page, H, KH = case["page"], case["heads"], case["kv_heads"]
    used = [-(-x // page) for x in kv]
    width = max(used) + 2
    pages = sum(used) + 5  # a few free ones
    # The pages of a pool in use for a while: any order, unused entries of the table -1.
    order = torch.randperm(pages, generator=g, device="cuda")[:sum(used)].to(torch.int32)
    at = torch.arange(width, device="cuda")
    first = torch.tensor([sum(used[:b]) for b in range(len(used))], device="cuda")
    count = torch.tensor(used, device="cuda")
    table = order[(first[:, None] + at).clamp(max=sum(used) - 1)]
    s["page_table"] = torch.where(at < count[:, None], table, -1).to(torch.int32)
    s["q_starts"] = torch.tensor([sum(n[:b]) for b in range(len(n) + 1)], device="cuda", dtype=torch.int32)
    s["kv_lens"] = torch.tensor(kv, device="cuda", dtype=torch.int32)
    s["max_q"], s["max_kv"], s["total_kv"], s["tokens"] = max(n), max(kv), sum(kv), sum(n)
    s["k_pages"], s["k_scales"] = _pool(g, pages, KH, page, case["type"], case["kind"] in ("select", "sparse"))
    if case["kind"] != "select":
        s["v_pages"], s["v_scales"] = _pool(g, pages, KH, page, case["type"], False)
    if case["kind"] == "append":
        s["qkv"] = _randn(g, sum(n), (H + 2 * KH) * D, scale=1.5)
        pos = torch.arange(max(kv) + 1, dtype=F64, device="cuda")
        freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=F64, device="cuda") / D)
        s["sin"], s["cos"] = torch.sin(pos[:, None] * freq).float(), torch.cos(pos[:, None] * freq).float()
        return s
    s["q"] = _randn(g, sum(n), H, D)
    if case["kind"] == "select":
        # Kept since the pages were full; those that the chunk wrote are not up to date.
        x = s["k_pages"].float()
        if s["k_scales"] is not None:
            x = x * s["k_scales"].repeat_interleave(BLOCK, dim=2)[..., None]
        s["bounds"] = torch.stack([x.amin(dim=2), x.amax(dim=2)], dim=2).to(BF)
        s["bounds"][order[-1].long()] = 0
    if case["kind"] == "sparse":
        # Lists as select_pages makes them: the first page, those of the block and the one before it, and others, in
        # ascending order, -1 where there are no more.
        block, last, own_first, _ = _blocks(s)
        col = torch.arange(width, device="cuda")
        rank = torch.rand((case["seqs"], block["count"], KH, width), generator=g, device="cuda")
        rank = rank + 2.0 * ((col < 1) | (col >= own_first[..., None] - 1))[:, :, None]
        rank = torch.where((col < last[..., None])[:, :, None], rank, -math.inf)
        s["columns"] = _lists(rank, case["top"])[block["seq"], block["of"]].contiguous()
    return s


def _blocks(s):
    """The blocks of the batch's chunks: of each packed token its sequence and its block's number in the chunk, the most
    blocks of a chunk, and of each block its columns (one past the last, the first that holds a token of its own) and the
    first key that it does not see."""
    starts, kv, bs, page = s["q_starts"], s["kv_lens"], s["bs"], s["page"]
    t = torch.arange(s["tokens"], device=kv.device)
    b = torch.searchsorted(starts[1:], t, right=True)
    c = (kv - (starts[1:] - starts[:-1]))[:, None]
    pos = (kv - starts[1:])[b] + t
    count = s["max_q"] // bs + 2
    begin = (c // bs + torch.arange(count, device=kv.device)) * bs
    end = torch.minimum(begin + bs, kv[:, None])
    of = pos // bs - (c[:, 0] // bs)[b]
    return {"seq": b, "of": of, "count": count}, -(-end // page), begin // page, end


def _lists(rank, top):
    """The `top` columns of highest rank (the lowest of equals), in ascending order; -1 in the place of those of rank
    -inf and behind the last."""
    width = rank.shape[-1]
    value, at = torch.sort(rank, dim=-1, descending=True, stable=True)
    at = torch.where(value > -math.inf, at, width)[..., :top]
    at = torch.nn.functional.pad(at, (0, top - at.shape[-1]), value=width)
    at = torch.sort(at, dim=-1).values
    return torch.where(at < width, at, -1).to(torch.int32)


# ---------------------------------------------------------------------------
# one pass

_entry = {}


def _own(name):
    if not _entry:
        pkg = os.path.join(os.getcwd(), "diffusion-llm_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from kernels import paged
        _entry.update(inputs=paged.paged_attention_inputs8, values=paged.page_values,
                      attention=paged.paged_attention_pool, bounds=paged.page_bounds, select=paged.select_pages)
    return _entry[name]


def run(s):
    kind = s["kind"]
    if own:
        batch = s["page_table"], s["q_starts"], s["kv_lens"]
        if kind == "append":
            q = _own("inputs")(s["qkv"], s["heads"], s["sin"], s["cos"], s["k_pages"], s["v_pages"], s["k_scales"],
                               s["v_scales"], *batch)
            k, v = _own("values")(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
            return q, k, v
        if kind == "select":
            _own("bounds")(s["k_pages"], s["bounds"], *batch, s["tokens"], k_scales=s["k_scales"])
            columns = _own("select")(s["q"], s["bounds"], *batch, s["bs"], s["page"], s["top"], max_q=s["max_q"],
                                     max_kv=s["max_kv"])
            return s["bounds"], columns
        return _own("attention")(s["q"], s["k_pages"], s["v_pages"], *batch, s["bs"], max_q=s["max_q"],
                                 max_kv=s["max_kv"], total_kv=s["total_kv"], k_scales=s["k_scales"],
                                 v_scales=s["v_scales"], columns=s["columns"] if kind == "sparse" else None)
    return {"append": _append, "cache8": _attention, "select": _select, "sparse": _sparse}[kind](s)


def _append(s):
    qkv, starts, kv, kind = s["qkv"], s["q_starts"], s["kv_lens"], s["type"]
    T, H, KH, page = qkv.shape[0], s["heads"], s["kv_heads"], s["page"]
    t = torch.arange(T, device=qkv.device)
    b = torch.searchsorted(starts[1:], t, right=True)
    pos = (kv - starts[1:])[b] + t
    x = qkv.float().view(T, H + 2 * KH, D)
    sin, cos = s["sin"][pos][:, None], s["cos"][pos][:, None]
    x1, x2 = x[:, :H + KH, :D // 2], x[:, :H + KH, D // 2:]
    y = torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1)
    # The blocks of slots that the chunks touch; past a chunk's last one it comes again.
    c = kv - (starts[1:] - starts[:-1])
    i = torch.arange(s["max_q"] // BLOCK + 2, device=qkv.device)
    blk = torch.minimum((c // BLOCK)[:, None] + i, ((kv - 1) // BLOCK)[:, None])
    p = blk[..., None] * BLOCK + torch.arange(BLOCK, device=qkv.device)
    new = (p >= c[:, None, None]) & (p < kv[:, None, None])
    token = (starts[:-1] - c)[:, None, None] + p
    token = torch.where(new, token, 0)
    where = s["page_table"].gather(1, blk // (page // BLOCK)).long()
    sub = blk % (page // BLOCK)
    kept = (blk * BLOCK < c[:, None])[..., None]  # the block holds earlier tokens
    for values, pages, scales in ((y[:, H:], s["k_pages"], s["k_scales"]), (x[:, H + KH:], s["v_pages"], s["v_scales"])):
        z = values[token].transpose(2, 3)  # (seqs, blocks, KH, 16, 64)
        here = new[:, :, None, :, None]
        need = _needed(torch.where(here, z.abs(), 0.0).amax(dim=(3, 4)), kind)
        old = scales[where, :, sub]
        m, e = torch.frexp(need / old)
        grow = (e - (m == 0.5).int()).clamp(min=0)  # the least with old * 2 ** grow >= need
        grow = torch.where(kept, grow, 0)
        scale = torch.where(kept, old * _power(grow), need)
        codes = pages.view(-1, KH, page // BLOCK, BLOCK, D)
        before = codes.view(torch.int8)[where, :, sub].view(pages.dtype).float() * _power(-grow)[..., None, None]
        before = (torch.round(before) if kind == "int8" else before).to(pages.dtype)
        after = torch.where(here, _encode(z, scale[..., None, None], kind).view(torch.int8), before.view(torch.int8))
        codes.view(torch.int8)[where, :, sub] = after
        scales[where, :, sub] = scale
    return y[:, :H].to(qkv.dtype), _values(s["k_pages"], s["k_scales"]).to(BF), _values(s["v_pages"], s["v_scales"]).to(BF)


def _values(pages, scales):
    x = pages.float()
    return x if scales is None else x * scales.repeat_interleave(BLOCK, dim=2)[..., None]


def _keys(s, name, where, slot):
    """The values, fp32, of slots of pages for every head: (..., kv_heads, 64)."""
    pages, scales = s[name + "_pages"], s[name + "_scales"]
    if scales is None:
        return pages[where, :, slot].float()
    x = pages.view(torch.int8)[where, :, slot].view(pages.dtype).float()
    return x * scales[where, :, slot // BLOCK][..., None]


def _attention(s):
    q, table, starts, kv = s["q"], s["page_table"], s["q_starts"], s["kv_lens"]
    T, H, _ = q.shape
    B, KH, page, bs = table.shape[0], s["kv_heads"], s["page"], s["bs"]
    n = starts[1:] - starts[:-1]
    i = torch.arange(s["max_q"], device=q.device)
    j = torch.arange(s["max_kv"], device=q.device)
    token = torch.where(i < n[:, None], starts[:-1, None] + i, T)  # T: no such token
    qs = q[token.clamp(max=T - 1)].float().view(B, -1, KH, H // KH, D).permute(0, 2, 1, 3, 4).reshape(B, KH, -1, D)
    where = table[:, j // page].clamp(min=0).long()
    ks = _keys(s, "k", where, j % page).permute(0, 2, 3, 1)
    vs = _keys(s, "v", where, j % page).permute(0, 2, 1, 3)
    pos = (kv - n)[:, None] + i
    end = torch.minimum((pos // bs + 1) * bs, kv[:, None])
    sees = (j < end[:, :, None]).repeat_interleave(H // KH, dim=1)[:, None]
    scores = torch.where(sees, qs @ ks / math.sqrt(D), -math.inf)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    o = (p @ vs / p.sum(dim=-1, keepdim=True)).view(B, KH, -1, H // KH, D).permute(0, 2, 1, 3, 4).reshape(B, -1, H, D)
    out = q.new_empty((T + 1, H, D))
    out[token] = o.to(q.dtype)
    return out[:T]


def _select(s):
    q, table, starts, kv, bounds = s["q"], s["page_table"], s["q_starts"], s["kv_lens"], s["bounds"]
    T, H, _ = q.shape
    B, KH, page, bs, width = table.shape[0], s["kv_heads"], s["page"], s["bs"], table.shape[1]
    # The bounds of the pages that hold tokens of the chunk, over the keys there are.
    c = kv - (starts[1:] - starts[:-1])
    i = torch.arange(s["max_q"] // page + 2, device=q.device)
    col = torch.minimum((c // page)[:, None] + i, ((kv - 1) // page)[:, None])
    slot = torch.arange(page, device=q.device)
    where = table.gather(1, col).long()
    keys = _keys(s, "k", where[..., None], slot)  # (seqs, pages, slots, KH, 64)
    there = (col[..., None] * page + slot < kv[:, None, None])[..., None, None]
    low = torch.where(there, keys, math.inf).amin(dim=2)
    high = torch.where(there, keys, -math.inf).amax(dim=2)
    bounds[where] = torch.stack([low, high], dim=3).to(BF)
    # No key k of a page has a larger q . k than sum_d max(q_d low_d, q_d high_d). In 64 bits: near the border the order counts.
    block, last, own_first, _ = _blocks(s)
    box = bounds[table.clamp(min=0).long()].double()  # (seqs, width, KH, 2, 64)
    box = torch.cat([box[..., 1, :], box[..., 0, :]], dim=-1).permute(0, 2, 3, 1).contiguous()
    i = torch.arange(s["max_q"], device=q.device)
    n = starts[1:] - starts[:-1]
    token = torch.where(i < n[:, None], starts[:-1, None] + i, T)
    qs = q[token.clamp(max=T - 1)].double().view(B, -1, KH, H // KH, D).permute(0, 2, 1, 3, 4)
    qs = torch.cat([qs.clamp(min=0), qs.clamp(max=0)], dim=-1).reshape(B, KH, -1, 2 * D)
    score = (qs @ box).view(B, KH, s["max_q"], H // KH, width).amax(dim=3).transpose(1, 2)
    rank = score.new_full((B, block["count"] + 1, KH, width), -math.inf)
    of = torch.where(i < n[:, None], (c[:, None] + i) // bs - (c // bs)[:, None], block["count"])
    rank.scatter_reduce_(1, of[:, :, None, None].expand(score.shape), score, "amax")
    rank = rank[:, :-1]
    at = torch.arange(width, device=q.device)
    rank = torch.where(((at < 1) | (at >= own_first[..., None] - 1))[:, :, None], math.inf, rank)
    rank = torch.where((at < last[..., None])[:, :, None] & (table >= 0)[:, None, None], rank, -math.inf)
    return bounds, _lists(rank, s["top"])[block["seq"], block["of"]]


def _sparse(s):
    q, table, starts = s["q"], s["page_table"], s["q_starts"]
    T, H, _ = q.shape
    B, KH, page, bs, top = table.shape[0], s["kv_heads"], s["page"], s["bs"], s["top"]
    G = H // KH
    block, _, _, end = _blocks(s)
    # The queries of each block side by side, and its list: that of its first token.
    c = s["kv_lens"] - (starts[1:] - starts[:-1])
    begin = (c // bs)[:, None] * bs + torch.arange(block["count"], device=q.device) * bs
    pos = begin[..., None] + torch.arange(min(bs, s["max_q"]), device=q.device)
    if bs > s["max_q"]:  # a block wider than any chunk: the chunk's tokens
        pos = pos - begin[..., None] + torch.maximum(begin, c[:, None])[..., None]
    mine = (pos >= c[:, None, None]) & (pos < end[..., None]) & (pos < (begin + bs)[..., None])
    token = torch.where(mine, (starts[:-1] - c)[:, None, None] + pos, T)
    first = token.amin(dim=2).clamp(max=T - 1)
    qs = q[token.clamp(max=T - 1)].float().view(B, block["count"], -1, KH, G, D).permute(0, 1, 3, 2, 4, 5).flatten(3, 4)
    cols = s["columns"][first].long()  # (seqs, blocks, KH, top)
    slot = torch.arange(page, device=q.device)
    key = (cols[..., None] * page + slot).flatten(3)
    sees = ((cols >= 0)[..., None].expand(*cols.shape, page).flatten(3)) & (key < end[:, :, None, None])
    where = torch.arange(B, device=q.device)[:, None, None, None], cols.clamp(min=0)
    where = table[where].long().clamp(min=0)[..., None].expand(*cols.shape, page).flatten(3)
    head = torch.arange(KH, device=q.device)[:, None]
    slot = slot.repeat(top)

    def gather(name):
        pages, scales = s[name + "_pages"], s[name + "_scales"]
        if scales is None:
            return pages[where, head, slot].float()
        return pages.view(torch.int8)[where, head, slot].view(pages.dtype).float() * scales[where, head, slot // BLOCK][..., None]

    scores = qs @ gather("k").transpose(-1, -2).contiguous() / math.sqrt(D)
    scores = torch.where(sees[:, :, :, None], scores, -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(most), 0.0, most))
    o = p @ gather("v") / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    o = o.unflatten(3, (-1, G)).permute(0, 1, 3, 2, 4, 5).reshape(*token.shape, H, D)
    out = q.new_empty((T + 1, H, D))
    out[token] = o.to(q.dtype)
    return out[:T]


def work(case):
    lens = _lengths(case)
    H, KH, page = case["heads"], case["kv_heads"], case["page"]
    tokens = sum(n for n, _ in lens)
    columns = sum(-(-(n + c) // page) for n, c in lens)
    table = columns * 4 + 8 * len(lens)
    # of a key or value of one head, its share of the scale with it
    el = 2 * D if case["type"] == "bf16" else D + 4 / BLOCK
    if case["kind"] == "append":
        # the projection, the queries, the codes; then the pages of the pool and their values
        pool = (columns + 5) * page
        moved = tokens * (H + 2 * KH) * D * 2 + tokens * H * D * 2 + 2 * tokens * KH * el
        rope = min(tokens, max(n + c for n, c in lens)) * D * 4
        return {"bytes": moved + rope + table + 2 * pool * KH * (el + 2 * D),
                "flops": 6 * tokens * (H + KH) * D // 2 + 2 * (2 * tokens + pool) * KH * D}
    bs, pairs, keys, spans, fresh = case["bs"], 0, 0, 0, 0
    for n, c in lens:
        fresh += (n + c - 1) // page - c // page + 1
        keys += 0 if case["kind"] == "sparse" else n + c
        # a block's tokens see the same keys
        for first in range(c // bs * bs, n + c, bs):
            end = min(first + bs, n + c)
            rows, seen = end - max(first, c), end
            spans += 1
            if case["kind"] == "sparse":
                seen = min(case["top"] * page, end)
                keys += seen
            pairs += rows * (-(-end // page) if case["kind"] == "select" else seen)
    if case["kind"] == "select":
        return {"bytes": fresh * KH * (page * el + 4 * D) + tokens * H * D * 2 + columns * KH * 4 * D
                + tokens * KH * case["top"] * 4 + table,
                "flops": 4 * D * H * pairs + 2 * fresh * KH * page * D}
    if case["kind"] == "sparse":  # blocks of one sequence may read the same page: at most all of its keys count
        keys = min(keys, sum(n + c for n, c in lens))
        table += spans * KH * case["top"] * 4
    return {"bytes": 2 * tokens * H * D * 2 + 2 * keys * KH * el + table, "flops": 4 * D * H * pairs}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "cache8": _exact_attention, "select": _exact_select,
            "sparse": _exact_sparse}[case["kind"]](case, s)


def _stored(pages, scales):
    """What a pool stands for, in 64 bits."""
    x = pages.to(F64) if pages.dtype != torch.float8_e4m3fn else pages.float().to(F64)
    if scales is not None:
        x = (x.unflatten(2, (-1, BLOCK)) * scales.to(F64)[..., None, None]).flatten(2, 3)
    return x


def _exact_append(case, s):
    H, KH, page, kind = case["heads"], case["kv_heads"], case["page"], case["type"]
    stored = [_stored(s["k_pages"], s["k_scales"]), _stored(s["v_pages"], s["v_scales"])]
    grids = [s["k_scales"].to(F64), s["v_scales"].to(F64)]
    qs, at = [], 0

    def rounded(x, step):  # to the multiples of the scale, or to its e4m3 values
        if kind == "int8":
            return torch.round(x / step) * step
        return (x / step).float().to(torch.float8_e4m3fn).float().to(F64) * step

    for b, (n, c) in enumerate(_lengths(case)):
        x = s["qkv"][at:at + n].to(F64).view(n, H + 2 * KH, 2, D // 2)
        z = torch.complex(x[:, :, 0], x[:, :, 1])
        turn = torch.complex(s["cos"][c:c + n].to(F64), s["sin"][c:c + n].to(F64))[:, None]
        turned = z[:, :H + KH] * turn
        turned = torch.cat([turned.real, turned.imag], dim=-1)
        qs.append(turned[:, :H])
        ids = s["page_table"][b].tolist()
        for p0 in range(c // BLOCK * BLOCK, c + n, BLOCK):
            lo, hi = max(p0, c), min(p0 + BLOCK, c + n)
            page_id, slot = ids[p0 // page], p0 % page
            for fresh, pool, grid in zip((turned[:, H:], x[:, H + KH:].reshape(n, KH, D)), stored, grids):
                new = fresh[lo - c:hi - c].transpose(0, 1)
                most = new.abs().amax(dim=(1, 2))
                if kind == "int8":
                    step = (most / 127).clamp(min=SMALLEST)
                else:
                    step = torch.exp2(torch.ceil(torch.log2(most / 448))).clamp(min=SMALLEST)
                if p0 < c:
                    old = grid[page_id, :, slot // BLOCK]
                    step = old * torch.exp2(torch.ceil(torch.log2(step / old)).clamp(min=0))
                    kept = pool[page_id, :, slot:slot + lo - p0]
                    pool[page_id, :, slot:slot + lo - p0] = rounded(kept, step[:, None, None])
                # what lies behind the last token keeps its codes, which mean nothing to the sequence
                behind = pool[page_id, :, slot + hi - p0:slot + BLOCK]
                ratio = (step / grid[page_id, :, slot // BLOCK])[:, None, None]
                if p0 < c:
                    pool[page_id, :, slot + hi - p0:slot + BLOCK] = rounded(behind, step[:, None, None])
                else:
                    pool[page_id, :, slot + hi - p0:slot + BLOCK] = behind * ratio
                pool[page_id, :, slot + lo - p0:slot + hi - p0] = rounded(new, step[:, None, None])
                grid[page_id, :, slot // BLOCK] = step
        at += n
    return torch.cat(qs), stored[0], stored[1]


def _exact_attention(case, s):
    H, KH, page, bs = case["heads"], case["kv_heads"], case["page"], case["bs"]
    k_all, v_all = _stored(s["k_pages"], s["k_scales"]), _stored(s["v_pages"], s["v_scales"])
    out, at = [], 0
    for b, (n, c) in enumerate(_lengths(case)):
        kv = n + c
        ids = s["page_table"][b, : -(-kv // page)].tolist()
        k = torch.cat([k_all[p] for p in ids], dim=1)[:, :kv]  # (KH, kv, D)
        v = torch.cat([v_all[p] for p in ids], dim=1)[:, :kv]
        q = s["q"][at:at + n].to(F64)
        o = torch.empty((n, H, D), dtype=F64, device=q.device)
        for r0 in range(0, n, 256):
            rows = torch.arange(r0, min(n, r0 + 256), device=q.device)
            mine = torch.div(c + rows, bs, rounding_mode="floor")
            hidden = torch.div(torch.arange(kv, device=q.device), bs, rounding_mode="floor") > mine[:, None]
            for h in range(H):
                w = q[rows, h] @ k[h * KH // H].t() * 0.125
                w = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1)
                o[rows, h] = w @ v[h * KH // H]
        out.append(o)
        at += n
    return torch.cat(out)


def _exact_select(case, s):
    H, KH, page, bs, top = case["heads"], case["kv_heads"], case["page"], case["bs"], case["top"]
    bounds = s["bounds"].to(F64)
    columns = torch.full((s["tokens"], KH, top), -1, dtype=torch.int32, device=bounds.device)
    at = 0
    for b, (n, c) in enumerate(_lengths(case)):
        kv, ids = n + c, s["page_table"][b].tolist()
        for col in range(c // page, -(-kv // page)):
            p = ids[col]
            scales = None if s["k_scales"] is None else s["k_scales"][p:p + 1]
            keys = _stored(s["k_pages"][p:p + 1], scales)[0][:, :min(page, kv - col * page)]
            bounds[p] = torch.stack([keys.min(dim=1).values, keys.max(dim=1).values], dim=1)
        rounded = bounds[torch.tensor(ids[:-(-kv // page)], device=bounds.device)].to(BF).to(F64)  # (cols, KH, 2, 64)
        for first in range(c // bs * bs, kv, bs):
            lo, end = max(first, c), min(first + bs, kv)
            cols = -(-end // page)
            forced = [i for i in range(cols) if i < 1 or i >= first // page - 1]
            q = s["q"][at + lo - c:at + end - c].to(F64).view(end - lo, KH, H // KH, D)
            for h in range(KH):
                score = torch.maximum(q[:, h, :, None] * rounded[:cols, h, 0], q[:, h, :, None] * rounded[:cols, h, 1])
                score = score.sum(dim=-1).amax(dim=(0, 1)).tolist()
                order = sorted(range(cols), key=lambda i: (i not in forced, -score[i], i))[:top]
                found = torch.tensor(sorted(order), dtype=torch.int32, device=columns.device)
                columns[at + lo - c:at + end - c, h, :len(order)] = found
        at += n
    return bounds, columns


def _exact_sparse(case, s):
    H, KH, page, bs = case["heads"], case["kv_heads"], case["page"], case["bs"]
    k_all, v_all = _stored(s["k_pages"], s["k_scales"]), _stored(s["v_pages"], s["v_scales"])
    out = torch.zeros(s["q"].shape, dtype=F64, device=s["q"].device)
    lists, table, at = s["columns"].tolist(), s["page_table"].tolist(), 0
    for b, (n, c) in enumerate(_lengths(case)):
        for first in range(c // bs * bs, n + c, bs):
            lo, end = max(first, c), min(first + bs, n + c)
            q = s["q"][at + lo - c:at + end - c].to(F64).view(end - lo, KH, H // KH, D)
            for h in range(KH):
                cols = [i for i in lists[at + lo - c][h] if i >= 0]
                ids = torch.tensor([table[b][i] for i in cols], device=out.device)
                key = (torch.tensor(cols, device=out.device)[:, None] * page
                       + torch.arange(page, device=out.device)).flatten()
                k, v = k_all[ids, h].flatten(0, 1)[key < end], v_all[ids, h].flatten(0, 1)[key < end]
                w = torch.softmax(q[:, h] @ k.t() * 0.125, dim=-1)
                out[at + lo - c:at + end - c].view(end - lo, KH, H // KH, D)[:, h] = w @ v
        at += n
    return out
