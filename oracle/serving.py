"""CPU definitions, in float64, of the ragged serving operators: attention of
packed chunks over a paged cache (all of it, or the pages of lists), the rotary
embedding written into pages, in bf16 or as 8-bit codes with scales, the pages that a
query selects, and adjusted logits. Loops over sequences, tokens and pages; used by the
tests."""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def keys_of(pages, table_row, kv, page_size):
    """(kv_heads, kv, 64) keys of one sequence and which of them exist."""
    P, KH, _, D = pages.shape
    out = torch.zeros((KH, kv, D), dtype=F64)
    there = torch.zeros(kv, dtype=torch.bool)
    for j0 in range(0, kv, page_size):
        page = int(table_row[j0 // page_size]) if j0 // page_size < len(table_row) else -1
        n = min(page_size, kv - j0)
        if 0 <= page < P:
            out[:, j0:j0 + n] = pages[page, :, :n].to(F64)
            there[j0:j0 + n] = True
    return out, there


def pool_values(pages, scales=None):
    """What pages stand for: (pages, kv_heads, page_size, 64) float64."""
    if scales is None:
        return pages.to(F64)
    x = pages.float().to(F64)
    return (x.unflatten(2, (-1, 16)) * scales.to(F64)[..., None, None]).flatten(2, 3)


def paged_attention(q, k_pages, v_pages, table, q_starts, kv_lens, block_size, out=None, columns=None):
    """(tokens, heads, 64) float64; rows of no sequence keep `out`'s values (0). `columns`
    (tokens, kv_heads, top): the pages that a block's first token names for it, as many entries
    as the sequence has columns."""
    T, H, D = q.shape
    KH, page = k_pages.shape[1], k_pages.shape[2]
    o = torch.zeros((T, H, D), dtype=F64) if out is None else out.to(F64).clone()
    for b in range(table.shape[0]):
        s, e, kv = int(q_starts[b]), int(q_starts[b + 1]), int(kv_lens[b])
        if e <= s:
            continue
        k, there = keys_of(k_pages, table[b], kv, page)
        v, _ = keys_of(v_pages, table[b], kv, page)
        pos = kv - (e - s) + torch.arange(e - s)
        j = torch.arange(kv)
        # (position // block) of a position before 0 is negative: it sees nothing
        all_seen = (j[None] // block_size <= pos[:, None] // block_size) & there[None] & (pos[:, None] >= 0)
        if columns is not None:  # the first token of each one's block
            leader = torch.stack([(pos // block_size == x // block_size).nonzero()[0, 0] for x in pos])
        for h in range(H):
            sees = all_seen
            if columns is not None:
                listed = columns[s + leader, h * KH // H][:, :-(-kv // page)]  # (tokens, entries)
                sees = all_seen & (listed[:, :, None] == (j // page)[None, None]).any(dim=1)
            w = q[s:e, h].to(F64) @ k[h * KH // H].t() / D ** 0.5
            w = w.masked_fill(~sees, -torch.inf)
            top = w.amax(dim=1, keepdim=True) if kv else torch.zeros(e - s, 1, dtype=F64)
            p = torch.exp(w - torch.where(torch.isinf(top), 0.0, top))
            total = p.sum(dim=1, keepdim=True)
            o[s:e, h] = torch.where(total > 0, p @ v[h * KH // H] / total.clamp(min=1e-300), 0.0)
    return o


def paged_attention_inputs(qkv, heads, sin, cos, k_pages, v_pages, table, q_starts, kv_lens):
    """(q, k_pages, v_pages) in float64; rows and slots not written are nan / as given."""
    T = qkv.shape[0]
    P, KH, page, D = k_pages.shape
    q = torch.full((T, heads, D), torch.nan, dtype=F64)
    kp, vp = k_pages.to(F64).clone(), v_pages.to(F64).clone()
    for b in range(table.shape[0]):
        s, e, kv = int(q_starts[b]), int(q_starts[b + 1]), int(kv_lens[b])
        for t in range(s, e):
            pos = kv - (e - t)
            at = min(max(pos, 0), sin.shape[0] - 1)
            x = qkv[t].to(F64).view(heads + 2 * KH, D)
            sn, cs = sin[at].to(F64), cos[at].to(F64)
            x1, x2 = x[:heads + KH, :D // 2], x[:heads + KH, D // 2:]
            y = torch.cat([x1 * cs - x2 * sn, x1 * sn + x2 * cs], dim=-1)
            q[t] = y[:heads]
            if pos < 0 or pos // page >= table.shape[1]:
                continue
            p = int(table[b, pos // page])
            if 0 <= p < P:
                kp[p, :, pos % page] = y[heads:]
                vp[p, :, pos % page] = x[heads + KH:]
    return q, kp, vp


def needed_scale(top, dtype):
    """The scale of a block whose values reach `top`."""
    if top == 0:
        return 2.0 ** -100
    s = top / 127 if dtype == torch.int8 else 2.0 ** math.ceil(math.log2(top / 448))
    return max(s, 2.0 ** -100)


def codes_of(x, dtype):
    """Values in units of the scale to codes."""
    if dtype == torch.int8:
        return torch.round(x).clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).float().to(dtype)


def paged_attention_inputs8(qkv, heads, sin, cos, k_pages, v_pages, k_scales, v_scales, table, q_starts, kv_lens):
    """(q, keys, values): the rotated queries and, as {(page, head, slot): 64 float64}, what the new keys and
    values are before they are encoded; (k_pages, v_pages, k_scales, v_scales) as they
    are afterwards."""
    KH, page = k_pages.shape[1], k_pages.shape[2]
    blank = torch.full(k_pages.shape, torch.nan, dtype=F64)
    q, kx, vx = paged_attention_inputs(qkv, heads, sin, cos, blank, blank, table, q_starts, kv_lens)
    codes = [k_pages.clone(), v_pages.clone()]
    scales = [k_scales.clone(), v_scales.clone()]
    new = [{}, {}]
    for b in range(table.shape[0]):
        n, kv = int(q_starts[b + 1]) - int(q_starts[b]), int(kv_lens[b])
        c = kv - n
        for p0 in range(c // 16 * 16, kv if n > 0 else c // 16 * 16, 16):
            at = int(table[b, p0 // page]) if 0 <= p0 // page < table.shape[1] and p0 >= 0 else -1
            if not 0 <= at < k_pages.shape[0]:
                continue
            slot = p0 % page
            lo, hi = max(c, p0) - p0, min(kv, p0 + 16) - p0
            for which, x in enumerate((kx, vx)):
                for h in range(KH):
                    mine = x[at, h, slot + lo:slot + hi]
                    scale = needed_scale(float(mine.abs().max()), k_pages.dtype)
                    block = codes[which][at, h, slot:slot + 16]
                    old = float(scales[which][at, h, slot // 16])
                    if p0 < c and 2.0 ** -100 <= old < math.inf:
                        grow = max(0, math.ceil(math.log2(scale / old)))
                        scale = old * 2.0 ** grow
                        if grow > 0:
                            block[:] = codes_of(block.double() * 2.0 ** -grow, k_pages.dtype)
                    block[lo:hi] = codes_of(mine / scale, k_pages.dtype)
                    scales[which][at, h, slot // 16] = scale
                    for r in range(lo, hi):
                        new[which][at, h, slot + r] = x[at, h, slot + r]
    return q, new[0], new[1], codes[0], codes[1], scales[0], scales[1]


def page_bounds(values, bounds, table, q_starts, kv_lens):
    """The bounds of the pages that the chunks' tokens are in, from the keys' values (float64)."""
    out, page = bounds.clone(), values.shape[2]
    for b in range(table.shape[0]):
        n, kv = int(q_starts[b + 1]) - int(q_starts[b]), int(kv_lens[b])
        for col in range(max(kv - n, 0) // page, -(-kv // page) if n > 0 else 0):
            at = int(table[b, col])
            if 0 <= at < values.shape[0]:
                keys = values[at, :, :min(page, kv - col * page)]
                out[at] = torch.stack([keys.amin(dim=1), keys.amax(dim=1)], dim=1).to(out.dtype)
    return out


def select_pages(q, bounds, table, q_starts, kv_lens, block_size, page, top, first=1, recent=1):
    """(tokens, kv_heads, top) columns; -2 in rows of no sequence."""
    T, H, _ = q.shape
    KH = bounds.shape[1]
    out = torch.full((T, KH, top), -2, dtype=torch.int32)
    box = bounds.to(F64)
    for b in range(table.shape[0]):
        s, e, kv = int(q_starts[b]), int(q_starts[b + 1]), int(kv_lens[b])
        pos = kv - (e - s) + torch.arange(e - s)
        for blk in torch.unique(pos // block_size).tolist():
            t = s + (pos // block_size == blk).nonzero()[:, 0]
            cols = -(-min((blk + 1) * block_size, kv) // page) if blk >= 0 else 0
            own = max(blk * block_size, 0) // page
            rows = q[t].to(F64)
            for h in range(KH):
                mine = rows[:, h * H // KH:(h + 1) * H // KH].reshape(-1, 1, q.shape[2])
                rank = []
                for col in range(cols):
                    at = int(table[b, col])
                    if not 0 <= at < bounds.shape[0]:
                        continue
                    if col < first or col >= own - recent:
                        rank.append((-math.inf, col))
                    else:
                        score = torch.where(mine > 0, mine * box[at, h, 1], mine * box[at, h, 0]).sum(dim=-1)
                        rank.append((-float(score.max()), col))
                taken = sorted(c for _, c in sorted(rank)[:top])
                out[t, h] = torch.tensor(taken + [-1] * (top - len(taken)), dtype=torch.int32)
    return out


def adjust_logits(logits, tokens=None, lengths=None, repetition=1.0, frequency=0.0, presence=0.0, bias=None,
                  allowed=None, fill=-1e6):
    """float64 of (batch, rows, vocab) logits."""
    B, R, V = logits.shape
    x = logits.to(F64).clone()

    def of(v, b):
        return float(v[b]) if torch.is_tensor(v) else float(torch.tensor(v, dtype=torch.float32))

    for b in range(B):
        if tokens is not None:
            n = tokens.shape[1] if lengths is None else min(max(int(lengths[b]), 0), tokens.shape[1])
            count = {}
            for t in tokens[b, :n].tolist():
                if 0 <= t < V:
                    count[t] = count.get(t, 0) + 1
            for t, c in count.items():
                r = of(repetition, b)
                x[b, :, t] = torch.where(x[b, :, t] > 0, x[b, :, t] / r, x[b, :, t] * r)
                x[b, :, t] -= of(frequency, b) * c + of(presence, b)
        if bias is not None:
            x[b] += (bias if bias.dim() == 1 else bias[b]).to(F64)
        # finite terms: in the type's range
        top = torch.finfo(logits.dtype).max
        x[b] = torch.where(torch.isfinite(x[b]), x[b].clamp(-top, top), x[b])
        if allowed is not None:
            for r in range(R):
                words = allowed if allowed.dim() == 1 else allowed[b] if allowed.dim() == 2 else allowed[b, r]
                v = torch.arange(V)
                x[b, r][((words[v // 32] >> (v % 32)) & 1) == 0] = fill
    return x
