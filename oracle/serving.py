"""CPU definitions, in float64, of the ragged serving operators: attention of
packed chunks over a paged cache, the rotary embedding written into pages, and
adjusted logits. Loops over sequences, tokens and pages; used by the tests."""
from __future__ import annotations

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


def paged_attention(q, k_pages, v_pages, table, q_starts, kv_lens, block_size, out=None):
    """(tokens, heads, 64) float64; rows of no sequence keep `out`'s values (0)."""
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
        sees = (j[None] // block_size <= pos[:, None] // block_size) & there[None] & (pos[:, None] >= 0)
        for h in range(H):
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
