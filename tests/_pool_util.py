"""Inputs and tolerances of the tests of 8-bit pools and selected pages."""
from __future__ import annotations

import torch

from _serving_util import BF, D, attention_reference, paged_case
from oracle import serving as orc

I8, E4 = torch.int8, torch.float8_e4m3fn


def pool_case(lens, heads, kv_heads, page, dtype, seed=0, **kw):
    """A paged_case whose pools hold `dtype`. The codes of slots that no sequence's keys
    fill are nan (e4m3) or -128 (int8, which no value has), the scales of blocks without keys nan."""
    c = paged_case(lens, heads, kv_heads, page, seed=seed, **kw)
    c["k_scales"] = c["v_scales"] = None
    if dtype == BF:
        return c
    g = torch.Generator().manual_seed(seed + 1)
    for name in ("k", "v"):
        x = c[name].double()
        there = ~torch.isnan(x)
        x = torch.where(there, x, 0.0) * torch.exp2(torch.randint(-3, 3, x.shape[:2], generator=g).double())[..., None, None]
        blocks = x.unflatten(2, (-1, 16))
        top = blocks.abs().amax(dim=(3, 4)).clamp(min=1e-9)
        scales = (top / 127 if dtype == I8 else torch.exp2(torch.ceil(torch.log2(top / 448)))).float()
        codes = orc.codes_of(blocks / scales[..., None, None].double(), dtype).flatten(2, 3)
        raw = codes.view(torch.uint8)
        raw[~there] = 0x80 if dtype == I8 else 0x7F
        scales[~there.unflatten(2, (-1, 16)).any(dim=4).any(dim=3)] = torch.nan
        c[name], c[name + "_scales"] = codes, scales
    return c


def values_of(c):
    """The case with the values of its pools in float64, slots without keys 0."""
    d = dict(c)
    for name in ("k", "v"):
        x = orc.pool_values(c[name], c[name + "_scales"])
        if c[name].dtype == I8:
            x = torch.where(c[name] == -128, 0.0, x)
        d[name] = torch.nan_to_num(x, nan=0.0)
    return d


def pool_reference(c, bs, columns=None):
    """As attention_reference, over the values of the pool: codes are exact operands and the
    scales' products (2^-24 relative to a score, to a probability) are far below its terms."""
    v = values_of(c)
    if columns is None:
        return attention_reference(v, bs)
    args = v["table"], v["starts"], v["kv"], bs
    ref = orc.paged_attention(v["q"], v["k"], v["v"], *args, columns=columns)
    size = orc.paged_attention(v["q"], v["k"], v["v"].abs(), *args, columns=columns)
    return ref, 1.01 * 2.0 ** -8 * (ref.abs() + size) + 2.0 ** -11 * size


def lists(c, kv_heads, page, bs, top, seed, own=True):
    """Lists of columns for each token (of each block's first one, the others' are noise): random ones, the
    block's own among them, in any order, some short, entries that name no column behind
    and between them."""
    g = torch.Generator().manual_seed(seed)
    T = c["q"].shape[0]
    out = torch.randint(-5, 50, (T, kv_heads, top), generator=g, dtype=torch.int32)
    for b in range(c["table"].shape[0]):
        s, e, kv = int(c["starts"][b]), int(c["starts"][b + 1]), int(c["kv"][b])
        seen = set()
        for t in range(s, e):
            pos = kv - (e - t)
            if pos // bs in seen:
                continue
            seen.add(pos // bs)
            cols = -(-min((pos // bs + 1) * bs, kv) // page) if pos >= 0 else 0
            for h in range(kv_heads):
                take = torch.randperm(max(cols, 1), generator=g)[:min(cols, top)].tolist()
                if own and cols and cols - 1 not in take:
                    take[0] = cols - 1
                if len(take) > 2 and float(torch.rand((), generator=g)) < 0.3:
                    take = take[:len(take) // 2]
                if len(take) < top and float(torch.rand((), generator=g)) < 0.5:
                    take.insert(len(take) // 2, -1 if t % 2 else 1 << 29)  # names none; 2^29 lies past every table
                out[t, h] = torch.tensor(take + [-1] * (top - len(take)), dtype=torch.int32)
    return out


def step_of(x, scale, dtype):
    """Spacing of the values of codes around x, at that scale."""
    if dtype == I8:
        return scale * torch.ones_like(x)
    e = torch.floor(torch.log2((x / scale).abs().clamp(min=2.0 ** -6)))
    return scale * torch.exp2(e - 3)


def code_error(got, want, scale, dtype):
    """Largest |got - want| in half steps around it: at most 1 + 2^-8 for a value rounded to its
    code once after fp32 arithmetic (of want up to 448 or 127 steps, the rotation's and the division's roundings, at
    most 4 * 2^-24 of it, are below 2^-8 half steps; a rotated key's terms may be larger than
    their sum, so tests pass their size)."""
    return float(((got - want).abs() / (0.5 * step_of(torch.maximum(got.abs(), want.abs()), scale, dtype))).max())


__all__ = ["BF", "D", "E4", "I8", "code_error", "lists", "pool_case", "pool_reference", "step_of", "values_of"]
