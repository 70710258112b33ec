"""Inputs and tolerances of the ragged serving operators' tests."""
from __future__ import annotations

import torch

from oracle import serving as orc

BF = torch.bfloat16
D = 64
HALF = 2.0 ** -8   # a rounding to bf16, relative: half of torch.finfo(bfloat16).eps


def paged_case(lens, heads, kv_heads, page, seed=0, spare=3, poison=True, q_scale=1.0, extra_tokens=0, width_more=2):
    """CPU tensors of a batch of (chunk, context) lengths: a pool whose pages are
    taken in random order, nan in every slot that no sequence's keys fill, -1 in
    the unused table entries."""
    g = torch.Generator().manual_seed(seed)
    kv = [n + c for n, c in lens]
    used = [-(-x // page) for x in kv]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g).tolist()
    width = max(used + [1]) + width_more
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    shape = (pages, kv_heads, page, D)
    k = torch.randn(shape, generator=g).to(BF)
    v = torch.randn(shape, generator=g).to(BF)
    filled = torch.zeros(pages, page, dtype=torch.bool)
    for b, x in enumerate(kv):
        for i in range(used[b]):
            p = order.pop()
            table[b, i] = p
            filled[p, :min(page, x - i * page)] = True
    if poison:
        k.masked_fill_(~filled[:, None, :, None], torch.nan)
        v.masked_fill_(~filled[:, None, :, None], torch.nan)
    starts = torch.tensor([sum(n for n, _ in lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32)
    T = int(starts[-1]) + extra_tokens
    q = (torch.randn((T, heads, D), generator=g) * q_scale).to(BF)
    return {"q": q, "k": k, "v": v, "table": table, "starts": starts, "kv": torch.tensor(kv, dtype=torch.int32),
            "max_q": max([n for n, _ in lens] + [0]), "max_kv": max(kv + [0]), "total": sum(kv)}


def attention_reference(c, bs):
    """The definition's output and the bound on a kernel's distance from it.

    A kernel rounds each probability to bf16 (relative HALF, so sum p |v| HALF in
    the numerator) and the result once (|o| HALF). Scores are fp32 sums of 64
    exact products: off by at most 64 * 2^-24 * sum |q k| / 8 < 2^-12 for the
    rows of these tests (|q| |k| up to 64 * 8), which changes p / sum p by
    twice that, relatively; fp32 exponentials, sums and merges are far below."""
    ref = orc.paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["kv"], bs)
    size = orc.paged_attention(c["q"], c["k"], c["v"].abs(), c["table"], c["starts"], c["kv"], bs)
    return ref, 1.01 * HALF * (ref.abs() + size) + 2.0 ** -11 * size


def worst(got, ref, tol):
    """Largest |got - ref| / tol; every got must be finite where ref is."""
    got = got.double().cpu()
    assert torch.isfinite(got).all(), "not finite"
    over = (got - ref).abs() / tol.clamp(min=1e-30)
    return float(over.max()) if over.numel() else 0.0
