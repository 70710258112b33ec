"""GPU parity of 8-bit paged caches and of attention over selected pages against their
definitions in float64 (oracle/serving.py)."""
from __future__ import annotations

import pytest
import torch

from _pool_util import BF, D, E4, I8, code_error, lists, pool_case, pool_reference, step_of, values_of
from _serving_util import HALF, worst
from kernels.kv_cache import rope_tables
from kernels.paged import (PagedKVCache, page_bounds, page_values, paged_attention, paged_attention_inputs,
                           paged_attention_inputs8, paged_attention_pool, select_pages)
from oracle import serving as orc

TYPES = [pytest.param(I8, id="int8"), pytest.param(E4, id="e4m3")]
POOLS = [pytest.param(BF, id="bf16"), *TYPES]


def on(c, dev):
    return {k: t.to(dev) if torch.is_tensor(t) else t for k, t in c.items()}


def attend(d, bs, columns=None, **kw):
    kw = {"max_q": d["max_q"], "max_kv": d["max_kv"], "total_kv": d["total"], **kw}
    return paged_attention_pool(d["q"], d["k"], d["v"], d["table"], d["starts"], d["kv"], bs, k_scales=d["k_scales"],
                                v_scales=d["v_scales"], columns=columns, **kw)


def same(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))


CASES = [
    # (chunk, context) of each sequence, heads, KV heads, page, block
    ([(1, 0)], 1, 1, 16, 1),
    ([(1, 599)], 12, 12, 16, 1),
    ([(1, 1), (1, 31), (1, 32), (1, 33), (1, 2047)], 4, 4, 32, 1),
    ([(16, 3584)], 12, 12, 64, 16),
    ([(16, 0), (16, 5), (16, 1000), (3, 77), (0, 50), (1, 1), (0, 0), (16, 496)], 2, 2, 64, 16),
    ([(4, 64), (4, 1020), (4, 300)], 3, 3, 16, 4),
    ([(32, 1504), (32, 0), (32, 31), (17, 300)], 4, 4, 64, 32),
    ([(65, 100), (64, 7)], 2, 2, 256, 64),
    ([(130, 70), (1, 300), (257, 0), (64, 64), (128, 128)], 2, 2, 16, 16),
    ([(300, 900), (7, 2000), (129, 1)], 2, 2, 64, 7),
    ([(513, 0), (128, 640)], 1, 1, 1024, 32),
    ([(32, 500), (8, 100), (1, 64)], 12, 4, 16, 32),
    ([(1, 700), (2, 30), (16, 256)], 16, 2, 64, 16),
    ([(40, 333), (90, 12)], 12, 1, 64, 8),
    ([(7, 100), (50, 200)], 6, 2, 64, 1 << 30),
    ([(1024, 0), (900, 100)], 12, 12, 64, 16),  # few, long items: four sets of waves
    ([(2049, 0), (0, 40)], 12, 6, 16, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("cut", ["whole", "many"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,heads,kv_heads,page,bs", CASES)
def test_attention_matches_definition(cuda, record_error, lens, heads, kv_heads, page, bs, dtype, cut):
    print(f"8-bit attention {lens} {heads}/{kv_heads} page {page} bs {bs} {dtype} {cut}", flush=True)
    c = pool_case(lens, heads, kv_heads, page, dtype, seed=len(lens) + page)
    ref, tol = pool_reference(c, bs)
    total = 0 if cut == "many" else len(lens) * max(c["max_kv"], 1)
    o = attend(on(c, cuda), bs, total_kv=total)
    assert o.shape == c["q"].shape and o.dtype == BF
    record_error("8-bit attention / bound", worst(o, ref, tol), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seqs,chunk", [(65, 1), (130, 16), (70, 40)])
def test_many_sequences_and_bad_entries(cuda, record_error, dtype, seqs, chunk):
    """More sequences than a wave has lanes, table entries that are no page, lengths and starts out of range."""
    g = torch.Generator().manual_seed(seqs)
    lens = [(int(n), int(x)) for n, x in zip(torch.randint(0, chunk + 1, (seqs,), generator=g),
                                             torch.randint(0, 300, (seqs,), generator=g))]
    lens[3], lens[seqs - 1] = (0, 0), (chunk, 700)
    c = pool_case(lens, 2, 1, 16, dtype, seed=seqs)
    c["table"][5, 0], c["table"][seqs - 1, 7], c["table"][seqs - 1, 40] = -1, 1 << 30, -7
    ref, tol = pool_reference(c, 16)
    for total in (0, 10 ** 7):
        record_error("8-bit attention / bound", worst(attend(on(c, cuda), 16, total_kv=total, max_q=chunk), ref, tol), 1.0)
    d = on(c, cuda)
    d["kv"] = torch.full_like(d["kv"], 1 << 30)  # cut to max_kv; pages past the sequence's are not there
    d["starts"][-1] = 1 << 30
    out = attend(d, 16, max_kv=c["max_kv"])
    torch.cuda.synchronize()
    assert out.shape == c["q"].shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_pools_and_results(cuda, record_error, dtype):
    """Slots outside heads, K and V in one tensor, out= with rows behind the last sequence."""
    c = pool_case([(16, 300), (5, 40)], 4, 2, 32, dtype, seed=7, extra_tokens=3)
    ref, tol = pool_reference(c, 16)
    d = on(c, cuda)
    both = torch.empty((c["k"].shape[0], 32, 2, 2, D), device=cuda, dtype=dtype)
    both[:, :, 0].view(torch.uint8).copy_(d["k"].view(torch.uint8).transpose(1, 2))
    both[:, :, 1].view(torch.uint8).copy_(d["v"].view(torch.uint8).transpose(1, 2))
    d["k"], d["v"] = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    out = torch.full((24, 8, D), 9.0, device=cuda, dtype=BF)[:, ::2]
    got = attend(d, 16, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[21:] == 9.0).all()
    record_error("8-bit attention / bound", worst(out[:21], ref[:21], tol[:21]), 1.0)


@pytest.mark.gpu
def test_one_pool_in_three_types(cuda):
    """Values that every type holds exactly (multiples of a scale up to 15). int8 and e4m3 agree to the bit: one arithmetic over
    the same codes and scales. The bf16 kernels divide by the running maximum itself, the others by one that may lag behind it,
    so other numbers P are rounded to bf16: each result is then within its own bound (a half step, 2^-8, of each P v and of the
    result: pool_reference) of the exact one, and the two within the sum of both bounds."""
    c = pool_case([(16, 500), (1, 77)], 4, 2, 16, BF, seed=9, poison=False)
    g = torch.Generator().manual_seed(0)
    d = on(c, cuda)
    for name in ("k", "v"):
        x = torch.randint(-15, 16, c[name].shape, generator=g).to(cuda)
        d[name] = (x * 0.25).to(BF)
        c[name] = d[name].cpu()
        for dtype in (I8, E4):
            d[f"{name}_{dtype}"] = x.to(torch.float32).to(dtype)
    _, tol = pool_reference(c, 16)
    want = attend(d, 16).double().cpu()
    shape = (c["k"].shape[0], 2, 1)
    got = []
    for dtype in (I8, E4):
        e = {**d, "k": d[f"k_{dtype}"], "v": d[f"v_{dtype}"], "k_scales": torch.full(shape, 0.25, device=cuda),
             "v_scales": torch.full(shape, 0.25, device=cuda)}
        got.append(attend(e, 16))
    assert torch.equal(*got)
    assert ((got[0].double().cpu() - want).abs() <= 2 * tol).all()


# -- the pages' inputs ---------------------------------------------------------

INPUTS = [
    # (chunk, context), heads, KV heads, page
    ([(1, 0)], 1, 1, 16),
    ([(1, 15), (1, 16), (1, 17), (1, 100)], 4, 2, 32),
    ([(16, 0), (16, 16), (16, 5), (0, 7), (3, 14), (2, 15), (33, 47)], 2, 2, 16),
    ([(70, 3), (100, 0), (31, 33)], 12, 4, 64),
    ([(257, 11)], 3, 3, 1024),
]


def inputs_case(lens, heads, kv_heads, page, dtype, seed):
    c = pool_case(lens, heads, kv_heads, page, dtype, seed=seed)
    g = torch.Generator().manual_seed(seed + 5)
    T = c["q"].shape[0]
    c["qkv"] = (torch.randn((T, (heads + 2 * kv_heads) * D), generator=g)
                * torch.exp2(torch.randint(-4, 5, (T, 1), generator=g).float())).to(BF)
    # blocks that only new tokens fill have had another sequence's scales
    for name in ("k_scales", "v_scales"):
        c[name] = torch.where(torch.isnan(c[name]), 3.0, c[name])
    return c


def check_inputs(c, heads, tables, got, dtype):
    """New values within half a step of what was encoded, scales and the other codes as defined."""
    q, k, v, ks, vs = got
    sin, cos = tables
    want = orc.paged_attention_inputs8(c["qkv"], heads, sin, cos, c["k"], c["v"], c["k_scales"], c["v_scales"], c["table"],
                                       c["starts"], c["kv"])
    there = ~torch.isnan(want[0])
    wq = torch.nan_to_num(want[0])
    size = wq.abs() + 2.0 ** -12 * c["qkv"].abs().max().double()  # fp32 sums of two products, far below a bf16 rounding
    assert float(((q.cpu().double() - wq).abs()[there] / (HALF * size[there])).max()) <= 1.01
    errors = []
    for new, codes, scales, wcodes, wscales in ((want[1], k, ks, want[3], want[5]), (want[2], v, vs, want[4], want[6])):
        codes, scales = codes.cpu(), scales.cpu()
        # of the maximum of fp32 sums: a few of its last bits; powers of two exactly
        assert torch.allclose(scales.double(), wscales.double(), rtol=2.0 ** -20 if dtype == I8 else 0, atol=0)
        touched = torch.zeros(codes.shape[:3], dtype=torch.bool)
        for (p, h, s), x in new.items():
            touched[p, h, s] = True
        if new:
            at = torch.tensor(list(new))
            x = torch.stack(list(new.values()))
            scale = scales[at[:, 0], at[:, 1], at[:, 2] // 16].double()[:, None]
            value = orc.pool_values(codes, scales)[at[:, 0], at[:, 1], at[:, 2]]
            errors.append(code_error(value, x, scale, dtype))
        # nan codes, behind a sequence's keys in a block whose scale grew, stand for nothing and may become anything
        rest = ~touched[..., None] & ~torch.isnan(wcodes.float())
        assert torch.equal(codes.view(torch.uint8)[rest], wcodes.view(torch.uint8)[rest])
    return max(errors, default=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,heads,kv_heads,page", INPUTS)
def test_inputs_match_definition(cuda, record_error, lens, heads, kv_heads, page, dtype):
    print(f"8-bit inputs {lens} {heads}/{kv_heads} page {page} {dtype}", flush=True)
    c = inputs_case(lens, heads, kv_heads, page, dtype, seed=page)
    tables = rope_tables(D, 512)
    d = on(c, cuda)
    q = paged_attention_inputs8(d["qkv"], heads, *(t.to(cuda) for t in tables), d["k"], d["v"], d["k_scales"], d["v_scales"],
                                d["table"], d["starts"], d["kv"])
    # half a step, and the rotation's fp32 roundings: terms of up to 2^5 * 4 sigma against steps of
    # 2^-8 of the block's largest value leave less than 2^-8 of a half step
    record_error("8-bit inputs / half step", check_inputs(c, heads, tables, (q, d["k"], d["v"], d["k_scales"], d["v_scales"]),
                                                          dtype), 1 + 2.0 ** -8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_one_at_a_time(cuda, record_error, dtype):
    """Growing values: every token raises its block's scale; the earlier ones end within a step."""
    tables = [t.to(cuda) for t in rope_tables(D, 64)]
    T, page = 48, 32
    g = torch.Generator().manual_seed(2)
    x = (torch.randn((T, 3 * D), generator=g) * torch.exp2(torch.arange(T) % 16 / 4.0)[:, None]).to(BF).to(cuda)
    k = torch.zeros((3, 1, page, D), device=cuda).to(dtype)
    v, ks = k.clone(), torch.zeros((3, 1, 2), device=cuda)
    vs = ks.clone()
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=cuda)
    for t in range(T):
        paged_attention_inputs8(x[t:t + 1], 1, *tables, k, v, ks, vs, table, torch.tensor([0, 1], dtype=torch.int32, device=cuda),
                                torch.tensor([t + 1], dtype=torch.int32, device=cuda))
    got = page_values(k, v, ks, vs)[1][[2, 0], 0].reshape(-1, D)[:T].cpu().double()
    want = x[:, 2 * D:].cpu().double()
    scale = vs[[2, 0], 0].reshape(-1)[torch.arange(T) // 16].cpu().double()[:, None]
    # page_values rounds to bf16: a relative HALF of up to 127 steps, or of a code that bf16 holds: nothing
    if dtype == I8:
        record_error("growing blocks / step", float((((got - want).abs() - HALF * got.abs()) / scale).max()), 1.0)
    else:
        # A growth is exact for codes that stay normal. One that becomes subnormal is rounded to the multiples of
        # 2^-9 scale, which at least double from growth to growth: halves of them, and the half step of the
        # first rounding, which is no larger, add up to 1/2 (1 + 1/2 + 1/4 + ...) < 1 of the last.
        step = step_of(torch.maximum(got.abs(), want.abs()), scale, E4)
        record_error("growing blocks / step", float(((got - want).abs() / step).max()), 1.0)
    assert (vs[1] == 0).all() and (ks[1] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-33, 3e37, 3.3e38])
def test_extreme_values(cuda, dtype, size):
    tables = [t.to(cuda) for t in rope_tables(D, 64)]
    x = torch.full((20, 3 * D), size, dtype=BF, device=cuda)
    x[:, ::3] *= -0.5
    k = torch.zeros((2, 1, 32, D), device=cuda).to(dtype)
    v, ks = k.clone(), torch.zeros((2, 1, 2), device=cuda)
    vs = ks.clone()
    one = torch.tensor([[1]], dtype=torch.int32, device=cuda)
    paged_attention_inputs8(x, 1, *tables, k, v, ks, vs, one, torch.tensor([0, 20], dtype=torch.int32, device=cuda),
                            torch.tensor([20], dtype=torch.int32, device=cuda))
    assert torch.isfinite(vs).all() and (vs[1] >= 2.0 ** -100).all()
    got = (v[1, 0, :20].float().double() * vs[1, 0].double().repeat_interleave(16)[:20, None]).cpu()
    want = x[:, 2 * D:].cpu().double()
    assert float((got - want).abs().max()) <= float(0.51 * step_of(want.abs().max(), vs[1].max().cpu().double(), dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_inputs_write_nothing_elsewhere(cuda, dtype):
    """Positions before 0, entries that are no page, positions past the table: q comes, no page or scale changes; rows behind
    the last sequence stay."""
    tables = [t.to(cuda) for t in rope_tables(D, 40)]
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn((60, 3 * D), generator=g).to(BF).to(cuda)
    k = torch.randint(0, 100, (4, 1, 16, D), generator=g).to(torch.uint8).to(cuda).view(dtype)
    v, ks = k.clone(), torch.rand((4, 1, 1), generator=g).to(cuda)
    vs = ks.clone()
    before = [t.clone() for t in (k, v, ks, vs)]
    table = torch.tensor([[-1, 4], [1 << 30, -5], [0, 1], [2, 3]], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 10, 20, 30, 50], dtype=torch.int32, device=cuda)
    lens = torch.tensor([20, 32, 0, 100], dtype=torch.int32, device=cuda)
    out = torch.full((60, 1, D), 5.0, dtype=BF, device=cuda)
    paged_attention_inputs8(qkv, 1, *tables, k, v, ks, vs, table, starts, lens, out=out)
    for a, b in zip((k, v, ks, vs), before):
        assert same(a, b)
    assert (out[50:] == 5.0).all() and (out[:50] != 5.0).any(dim=-1).all()
    # as the bf16 pages' queries, which clamp positions to the tables the same way
    pages = torch.zeros((4, 1, 16, D), dtype=BF, device=cuda)
    want = paged_attention_inputs(qkv, 1, *tables, pages, pages.clone(), table, starts, lens)
    assert torch.equal(out[:50], want[:50])


@pytest.mark.gpu
def test_page_values(cuda):
    g = torch.Generator().manual_seed(4)
    for dtype in (I8, E4):
        raw = torch.randint(0, 256, (7, 3, 48 // 16 * 32, 2 * D), generator=g, dtype=torch.uint8)
        raw[(raw & 0x7F) == 0x7F] = 0  # e4m3's nan
        pages = raw.to(cuda).view(dtype)[:, :, :32]
        k, v = pages[..., :D], pages[..., D:]
        ks, vs = torch.rand((7, 3, 2), generator=g).to(cuda), torch.rand((7, 3, 2), generator=g).to(cuda) * 1e-5
        got = page_values(k, v, ks, vs)
        for x, codes, scales in zip(got, (k, v), (ks, vs)):
            want = (codes.float().unflatten(2, (2, 16)) * scales[..., None, None]).flatten(2, 3).to(BF)
            assert torch.equal(x, want)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 16, 40, 150])
@pytest.mark.parametrize("dtype", POOLS)
def test_pages_past_32_bit_offsets(cuda, dtype, chunk):
    """A step of every operator over pages whose element offsets pass 2^32, beside the first ones, against the same step
    over a small pool, to the bit."""
    lens, heads, kv_heads, page, bs, top = [(chunk, 200), (chunk, 90)], 4, 2, 64, 16, 5
    tables = [t.to(cuda) for t in rope_tables(D, 512)]
    g = torch.Generator().manual_seed(chunk)
    need = [-(-(n + x) // page) for n, x in lens]
    n = sum(need)
    far = (1 << 32) // (kv_heads * page * D) + 100
    table = torch.full((2, max(need)), -1, dtype=torch.int32)
    for b, ids in enumerate(torch.randperm(n, generator=g).split(need)):
        table[b, :need[b]] = ids
    starts = torch.tensor([0, chunk, 2 * chunk], dtype=torch.int32, device=cuda)
    kv = torch.tensor([a + b for a, b in lens], dtype=torch.int32, device=cuda)
    before = torch.tensor([0, 200, 290], dtype=torch.int32, device=cuda), torch.tensor([200, 90], dtype=torch.int32, device=cuda)
    first = torch.randn((290, (heads + 2 * kv_heads) * D), generator=g).to(BF).to(cuda)
    qkv = torch.randn((2 * chunk, (heads + 2 * kv_heads) * D), generator=g).to(BF).to(cuda)

    def step(pages, table):
        k, v = (torch.empty((pages, kv_heads, page, D), device=cuda, dtype=dtype) for _ in range(2))
        bounds = torch.empty((pages, kv_heads, 2, D), device=cuda, dtype=BF)
        scales = [torch.empty((pages, kv_heads, page // 16), device=cuda) for _ in range(2)] if dtype != BF else [None] * 2
        ids = torch.cat([t[t >= 0] for t in table]).long()
        for t in (k, v, *scales):  # slots that no call writes
            if t is not None:
                t.view(torch.uint8)[ids] = 0
        for x, s, e in ((first, *before), (qkv, starts, kv)):
            if dtype == BF:
                q = paged_attention_inputs(x, heads, *tables, k, v, table, s, e)
            else:
                q = paged_attention_inputs8(x, heads, *tables, k, v, *scales, table, s, e)
            page_bounds(k, bounds, table, s, e, x.shape[0], scales[0])
        columns = select_pages(q, bounds, table, starts, kv, bs, page, top, chunk)
        batch = q, k, v, table, starts, kv, bs, chunk
        o = paged_attention_pool(*batch, k_scales=scales[0], v_scales=scales[1])
        listed = paged_attention_pool(*batch, k_scales=scales[0], v_scales=scales[1], columns=columns)
        values = [x[ids] for x in (page_values(k, v, *scales) if dtype != BF and chunk == 16 else ())]
        return [q, o, columns, listed, bounds[ids], k.view(torch.uint8)[ids], v.view(torch.uint8)[ids], *values] + \
            [t[ids] for t in scales if t is not None]

    small = step(n, table.to(cuda))
    large = step(far, torch.where(table >= n // 2, table + far - n, table).to(cuda))
    assert all(same(a.contiguous(), b.contiguous()) for a, b in zip(small, large))


# -- lists of pages --------------------------------------------------------------

LISTED = [
    # (chunk, context), heads, KV heads, page, block, top
    ([(1, 0)], 1, 1, 16, 1, 1),
    ([(1, 999), (1, 3), (1, 500)], 12, 4, 16, 1, 9),
    ([(16, 3000)], 4, 4, 64, 16, 12),
    ([(16, 0), (16, 5), (16, 1000), (3, 77), (0, 50), (1, 1), (0, 0), (16, 496)], 2, 2, 64, 16, 5),
    ([(40, 700), (7, 60), (33, 0)], 4, 2, 32, 16, 7),
    ([(50, 301), (3, 1000)], 6, 2, 16, 7, 20),
    ([(32, 1000), (90, 31)], 12, 4, 32, 32, 70),
    ([(20, 200), (5, 4)], 12, 1, 16, 4, 66),
    ([(100, 50)], 2, 2, 128, 1 << 30, 2),
    ([(9, 900)], 2, 1, 1024, 1, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", POOLS)
@pytest.mark.parametrize("lens,heads,kv_heads,page,bs,top", LISTED)
def test_listed_pages_match_definition(cuda, record_error, lens, heads, kv_heads, page, bs, top, dtype):
    print(f"listed pages {lens} {heads}/{kv_heads} page {page} bs {bs} top {top} {dtype}", flush=True)
    c = pool_case(lens, heads, kv_heads, page, dtype, seed=len(lens) + page)
    for own in (True, False):  # without its own page a token may see nothing: 0
        columns = lists(c, kv_heads, page, bs, top, seed=page + own, own=own)
        ref, tol = pool_reference(c, bs, columns)
        wide = torch.full((c["q"].shape[0], kv_heads, top + 3), 1, dtype=torch.int32, device=cuda)
        wide[:, :, :top] = columns.to(cuda)
        for given in (columns.to(cuda), wide[:, :, :top]):
            record_error("listed pages / bound", worst(attend(on(c, cuda), bs, given), ref, tol), 1.0)


@pytest.mark.gpu
def test_lists_in_other_layouts(cuda):
    """One list for all tokens (stride 0), the front of longer lists, KV heads first."""
    c = pool_case([(16, 900), (7, 300)], 4, 2, 32, I8, seed=3)
    d = on(c, cuda)
    g = torch.Generator().manual_seed(1)
    one = torch.stack([torch.randperm(20, generator=g)[:12].sort().values for _ in range(2)]).to(torch.int32).to(cuda)
    T = d["q"].shape[0]
    want = attend(d, 16, one.expand(T, 2, 12).contiguous())
    assert torch.equal(attend(d, 16, one.expand(T, 2, 12)), want)
    longer = torch.full((T, 2, 40), 3, dtype=torch.int32, device=cuda)
    longer[:, :, :12] = one
    assert torch.equal(attend(d, 16, longer[:, :, :12]), want)
    heads_first = one[:, None].expand(2, T, 12).contiguous().transpose(0, 1)
    assert torch.equal(attend(d, 16, heads_first), want)


@pytest.mark.gpu
def test_empty_lists_and_all_pages(cuda, record_error):
    c = pool_case([(16, 300), (16, 20)], 2, 2, 32, BF, seed=6)
    d = on(c, cuda)
    none = torch.full((32, 2, 4), -1, dtype=torch.int32, device=cuda)
    assert (attend(d, 16, none) == 0).all()
    every = torch.arange(12, dtype=torch.int32, device=cuda).expand(32, 2, 12)
    ref, tol = pool_reference(c, 16)
    record_error("listed pages / bound", worst(attend(d, 16, every.contiguous()), ref, tol), 1.0)
    record_error("listed pages / bound", worst(attend(d, 16, every), ref, tol), 1.0)  # one list for all, strides 0


@pytest.mark.gpu
@pytest.mark.parametrize("kv,n", [(5, 40), (0, 20), (33, 50)])
def test_listed_pages_with_tokens_before_the_first_position(cuda, record_error, kv, n):
    """A length below the chunk's: those tokens see nothing, and are 0."""
    c = pool_case([(n, 0)], 2, 1, 16, BF, seed=8)
    c["kv"][0] = kv
    c["max_kv"] = max(kv, 1)
    columns = torch.tensor([0, 1, 2], dtype=torch.int32).expand(n, 1, 3).contiguous()
    for bs in (1, 4, 16):
        ref, tol = pool_reference(c, bs, columns)
        o = attend(on(c, cuda), bs, columns.to(cuda))
        assert (o[:n - kv] == 0).all()
        record_error("listed pages / bound", worst(o, ref, tol), 1.0)


# -- bounds and selection ----------------------------------------------------------


def bounded(c, kv_heads):
    """Bounds of all pages from the keys that fill them (elsewhere 0)."""
    x = values_of(c)["k"]
    there = (x != 0).any(dim=-1, keepdim=True)
    low = torch.where(there, x, torch.inf).amin(dim=2)
    high = torch.where(there, x, -torch.inf).amax(dim=2)
    return torch.nan_to_num(torch.stack([low, high], dim=2), posinf=0.0, neginf=0.0).to(BF)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", POOLS)
@pytest.mark.parametrize("lens,kv_heads,page", [([(1, 0)], 1, 16), ([(1, 31), (1, 32), (40, 3), (0, 9), (16, 16)], 3, 32),
                                                ([(300, 77), (5, 1000)], 2, 64), ([(700, 900)], 1, 1024),
                                                ([(3, k) for k in range(70)], 2, 16)])
def test_bounds_match_definition(cuda, lens, kv_heads, page, dtype):
    c = pool_case(lens, kv_heads, kv_heads, page, dtype, seed=page)
    if len(lens) > 1:
        c["table"][1, 0] = -1
    start = torch.randn((c["k"].shape[0], kv_heads, 2, D), generator=torch.Generator().manual_seed(1)).to(BF)
    want = orc.page_bounds(orc.pool_values(c["k"], c["k_scales"]).float().to(BF).double(), start, c["table"], c["starts"], c["kv"])
    d = on(c, cuda)
    got = start.to(cuda)
    assert page_bounds(d["k"], got, d["table"], d["starts"], d["kv"], c["q"].shape[0], d["k_scales"]) is got
    assert torch.equal(got.cpu(), want)


SELECT = [
    # (chunk, context), heads, KV heads, page, block, top, first, recent
    ([(1, 0)], 1, 1, 16, 1, 3, 1, 1),
    ([(1, 999), (1, 3), (1, 500)], 12, 4, 16, 1, 9, 1, 1),
    ([(16, 3000), (16, 100), (5, 7)], 4, 4, 64, 16, 12, 1, 1),
    ([(40, 700), (7, 60), (33, 0), (0, 8)], 4, 2, 32, 16, 4, 0, 0),
    ([(50, 301), (3, 1000)], 6, 2, 16, 7, 21, 2, 3),
    ([(40, 500)], 16, 1, 16, 32, 11, 1, 0),
    ([(1, 8300)], 2, 1, 16, 1, 64, 1, 1),     # over 512 columns
    ([(2, 25000), (1, 17000)], 1, 1, 16, 1, 100, 1, 1),  # over 1536
    ([(1, 32800), (5, 40000), (3, 90)], 1, 1, 16, 4, 130, 1, 1),  # over 2048
    ([(1, 140000)], 1, 1, 16, 1, 2000, 1, 1),  # over 8192
    ([(100, 50)], 2, 2, 128, 1 << 30, 4, 1, 1),
]


def pick(d, bounds, bs, page, top, first=1, recent=1, **kw):
    kw = {"max_q": d["max_q"], "max_kv": d["max_kv"], **kw}
    return select_pages(d["q"], bounds, d["table"], d["starts"], d["kv"], bs, page, top, first=first, recent=recent, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["random", "equal", "near", "zero", "wide", "huge", "tiny", "subnormal"])
@pytest.mark.parametrize("lens,heads,kv_heads,page,bs,top,first,recent", SELECT)
def test_selection_matches_definition(cuda, lens, heads, kv_heads, page, bs, top, first, recent, kind):
    """Columns to the last one, also where scores are equal, or differ by less than fp32 sums do."""
    print(f"select {lens} {heads}/{kv_heads} page {page} bs {bs} top {top} {kind}", flush=True)
    c = pool_case(lens, heads, kv_heads, page, BF, seed=page + top)
    bounds = bounded(c, kv_heads)
    g = torch.Generator().manual_seed(top)
    if kind == "equal":  # few different pages
        bounds = bounds[torch.randint(0, 3, (bounds.shape[0],), generator=g)]
    elif kind == "near":  # one page's bounds, a last bit off in one channel
        bounds = bounds[:1].expand_as(bounds).clone()
        at = torch.randint(0, D, (bounds.shape[0],), generator=g)
        raw = bounds.view(torch.int16)
        raw[torch.arange(bounds.shape[0]), :, 1, at] += torch.randint(-1, 2, (bounds.shape[0], 1), generator=g).to(torch.int16)
    elif kind == "zero":
        c["q"].zero_()
    elif kind == "wide":  # terms of either sign and very different sizes that nearly cancel
        big = torch.exp2(torch.randint(-6, 7, (D,), generator=g).float())
        bounds = (bounds[:1].float() * big + torch.randn(bounds.shape, generator=g) * 2.0 ** -6).to(BF)
    elif kind == "huge":  # fp32 sums overflow
        bounds, c["q"] = (bounds.float() * 2.0 ** 64).to(BF), (c["q"].float() * 2.0 ** 62).to(BF)
    elif kind == "tiny":  # products about fp32's smallest
        bounds, c["q"] = (bounds.float() * 2.0 ** -66).to(BF), (c["q"].float() * 2.0 ** -62).to(BF)
    elif kind == "subnormal":  # bf16's smallest, few bits of them
        bounds, c["q"] = (bounds.float() * 2.0 ** -130).to(BF), (c["q"].float() * 2.0 ** 100).to(BF)
    c["table"][0, 0] = -1 if len(lens) > 1 else c["table"][0, 0]
    want = orc.select_pages(c["q"], bounds, c["table"], c["starts"], c["kv"], bs, page, top, first, recent)
    d = on(c, cuda)
    out = torch.full((c["q"].shape[0], kv_heads, top), -2, dtype=torch.int32, device=cuda)
    got = pick(d, bounds.to(cuda), bs, page, top, first, recent, out=out)
    assert got is out or got.data_ptr() == out.data_ptr()
    assert torch.equal(out.cpu(), want)


@pytest.mark.gpu
def test_selection_of_many_sequences(cuda):
    g = torch.Generator().manual_seed(5)
    lens = [(int(n), int(x)) for n, x in zip(torch.randint(0, 5, (150,), generator=g), torch.randint(0, 400, (150,), generator=g))]
    c = pool_case(lens, 2, 2, 16, BF, seed=5, extra_tokens=4)
    c["kv"][7] = 1  # fewer keys than tokens
    bounds = bounded(c, 2)
    want = orc.select_pages(c["q"], bounds, c["table"], c["starts"], c["kv"], 4, 16, 6)
    d = on(c, cuda)
    out = torch.full((c["q"].shape[0], 2, 6), -2, dtype=torch.int32, device=cuda)
    pick(d, bounds.to(cuda), 4, 16, 6, out=out, max_q=5)
    assert torch.equal(out.cpu(), want)
    assert (out[-4:] == -2).all()


@pytest.mark.gpu
def test_selected_pages_hold_the_weight(cuda):
    """What the selection is for: with a few keys that a query looks for, the listed pages give the dense result."""
    c = pool_case([(16, 4000)], 4, 2, 32, BF, seed=12, poison=False)
    d = on(c, cuda)
    page = int(c["table"][0, 40])
    d["q"][:, :2] = d["q"][:1, :1]  # the group of KV head 0 asks for one direction
    d["k"][page, 0, 5] = (3.0 * d["q"][0, 0].float()).to(BF)
    bounds = torch.zeros((c["k"].shape[0], 2, 2, D), dtype=BF, device=cuda)
    everything = torch.tensor([0, 4016], dtype=torch.int32, device=cuda)
    page_bounds(d["k"], bounds, d["table"], everything, d["kv"], 4016)
    columns = pick(d, bounds, 16, 32, 8)
    assert (columns[:, 0] == 40).any(dim=-1).all()
    near = attend(d, 16, columns)[:, :2].float()
    full = attend(d, 16)[:, :2].float()
    assert float((near - full).norm() / full.norm()) < 0.02


# -- together ------------------------------------------------------------------------


def model_step(batch, qkv, heads, tables, layer, bs, top, final):
    q = batch.attention_inputs(qkv, heads, *tables, layer)
    if final:
        batch.update_bounds(layer)
    return batch.attention(q, layer, bs, top=top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", POOLS)
def test_cache_steps(cuda, record_error, dtype):
    """Prompts, drafts that are overwritten and single tokens through the cache, all pages or selected ones, against
    the definitions over what the pool then holds."""
    heads, kv_heads, page, bs, top = 4, 2, 16, 4, 6
    tables = [t.to(cuda) for t in rope_tables(D, 512)]
    cache = PagedKVCache(2, 60, kv_heads, page, device=cuda, dtype=dtype, bounds=True)
    g = torch.Generator().manual_seed(1)
    a, b = cache.add(), cache.add()

    def step(seqs, tokens, top, commit):
        batch = cache.batch(seqs, tokens)
        for layer in range(2):
            qkv = torch.randn((sum(tokens), (heads + 2 * kv_heads) * D), generator=g).to(BF).to(cuda)
            o = model_step(batch, qkv, heads, tables, layer, bs, top, commit)
            q = batch.attention_inputs(qkv, heads, *tables, layer)  # the same again: changes nothing
            c = {"q": q.cpu(), "k": cache.k_pages[layer].cpu(), "v": cache.v_pages[layer].cpu(), "table": batch.page_table.cpu(),
                 "starts": batch.q_starts.cpu(), "kv": batch.kv_lens.cpu()}
            c["k_scales"], c["v_scales"] = (None if s is None else s.cpu() for s in cache.scales(layer))
            columns = None
            if top is not None:
                columns = orc.select_pages(c["q"], cache.bounds[layer].cpu(), c["table"], c["starts"], c["kv"], bs, page, top)
            ref, tol = pool_reference(c, bs, columns)
            record_error("cache step / bound", worst(o, ref, tol), 1.0)
        if commit:
            batch.commit()

    step([a, b], [200, 33], None, True)
    for k in range(3):
        step([b, a], [4, 4], top, False)
    step([b, a], [4, 4], top, True)
    for k in range(5):
        step([a], [1], top, True)
    step([b, a], [70, 21], top, True)
    cache.free(a)
    c = cache.add()
    step([c, b], [100, 4], top, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", POOLS)
def test_captured_step(cuda, dtype):
    """Two captures of a whole step in one pool, replayed in turn with other lengths and inputs, against eager calls."""
    heads, page, bs, top, seqs = 4, 16, 16, 5, 3
    tables = [t.to(cuda) for t in rope_tables(D, 1024)]
    cache = PagedKVCache(2, 200, heads, page, device=cuda, dtype=dtype, bounds=True)
    ids = [cache.add() for _ in range(seqs)]
    g = torch.Generator().manual_seed(2)
    first = cache.batch(ids, [600, 500, 400])
    for layer in range(2):
        qkv = torch.randn((1500, 3 * heads * D), generator=g).to(BF).to(cuda)
        first.attention_inputs(qkv, heads, *tables, layer)
        first.update_bounds(layer)
    first.commit()
    batch = cache.batch(ids, [bs] * seqs)
    qkv = torch.randn((bs * seqs, 3 * heads * D), generator=g).to(BF).to(cuda)
    state = [cache.k_pages, cache.v_pages, cache.bounds] + ([] if dtype == BF else [cache.k_scales, cache.v_scales])
    kept = [t.clone() for t in state]

    def run(layer):
        return model_step(batch, qkv, heads, tables, layer, bs, top, True)

    def reset():
        for t, k in zip(state, kept):
            t.view(torch.uint8).copy_(k.view(torch.uint8))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(0), run(1)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, pool = [], [], torch.cuda.graph_pool_handle()
    for layer in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(run(layer))
        graphs.append(graph)
    lens = batch.kv_lens.clone()
    for k in range(3):
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF))
        batch.kv_lens.copy_(lens - torch.tensor([17 * k, 0, 16 * k], device=cuda, dtype=torch.int32))
        reset()
        want = [run(0).clone(), run(1).clone()]
        after = [t.clone() for t in state]
        reset()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), k
        assert all(same(t, w) for t, w in zip(state, after)), k


@pytest.mark.gpu
def test_calls_on_other_streams(cuda):
    """Two streams with work of their own at once: workspaces are each call's own."""
    c = pool_case([(1, 3000), (1, 2000)], 8, 8, 16, I8, seed=3)
    d = on(c, cuda)
    bounds = bounded(c, 8).to(cuda)
    want = pick(d, bounds, 1, 16, 40), attend(d, 1), None
    want = (want[0], want[1], attend(d, 1, want[0]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 4:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            columns = pick(d, bounds, 1, 16, 40)
            got.append((columns, attend(d, 1), attend(d, 1, columns)))
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a, b) for a, b in zip(x, want))


@pytest.mark.gpu
def test_custom_ops_and_compile(cuda):
    import kernels.ops  # noqa: F401
    c = pool_case([(4, 300), (4, 77)], 4, 2, 16, I8, seed=4)
    d = on(c, cuda)
    bounds = bounded(c, 2).to(cuda)
    batch = d["table"], d["starts"], d["kv"]

    def f(q):
        torch.ops.bd3.page_bounds(d["k"], bounds, *batch, 8, d["k_scales"])
        columns = torch.ops.bd3.select_pages(q, bounds, *batch, 4, 16, 6, 4, d["max_kv"])
        return torch.ops.bd3.paged_attn_pool(q, d["k"], d["v"], *batch, 4, 4, d["max_kv"], d["total"], d["k_scales"],
                                             d["v_scales"], columns) + 1

    want = attend(d, 4, pick(d, page_bounds(d["k"], bounds.clone(), *batch, 8, d["k_scales"]), 4, 16, 6)) + 1
    assert torch.equal(f(d["q"]), want)
    assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(d["q"]), want)
    tables = [t.to(cuda) for t in rope_tables(D, 512)]
    qkv = torch.randn(8, 8 * D, device=cuda, dtype=BF)
    x, y = ([t.clone() for t in (d["k"], d["v"], d["k_scales"], d["v_scales"])] for _ in range(2))
    q = torch.ops.bd3.paged_qkv_rope8(qkv, 4, *tables, *x, *batch)
    assert torch.equal(q, paged_attention_inputs8(qkv, 4, *tables, *y, *batch))
    assert all(same(a, b) for a, b in zip(x, y))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,top", [(I8, None), (E4, None), (BF, 8), (I8, 8)])
def test_serving_with_a_smaller_cache(cuda, dtype, top):
    """The serving loop over 8-bit pages and selected ones: its first logits beside the eager backbone's."""
    from perf.e2e_sampling import Cfg, backbone_eager, init_params, serve
    cfg = Cfg(vocab=1001, mask=1000, max_seq=512, d=256, heads=4, layers=4, d_ff=512, bs=16)
    p = init_params(cfg, 0, cuda)
    tables = rope_tables(64, cfg.max_seq, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(0)
    prompts = [torch.randint(0, cfg.mask, (16 * n,), generator=g, device=cuda) for n in (1, 13, 0, 5)]
    n_blocks = [2, 1, 2, 1]
    got = []

    def check(before, block, logits):
        with torch.no_grad():
            cache = [None] * cfg.layers
            if len(before):
                pos = torch.arange(len(before), device=cuda)
                causal = (pos[None, :] // cfg.bs) <= (pos[:, None] // cfg.bs)
                backbone_eager(cfg, p, tables, before[None], cache, True, mask=causal)
            want = backbone_eager(cfg, p, tables, block[None], cache, False)[0].float()
            got.append(float((want - logits.float()).norm() / want.norm()))

    def go(check=None):
        with torch.no_grad():
            return serve(cfg, p, tables, prompts, n_blocks, 3, 14, page_size=32, seed=3, check=check, cache_dtype=dtype, top=top)

    out = go(check)
    # 224 tokens are 7 pages of 32: 8 hold all of them. Keys and values are off by 2^-4 (e4m3) of themselves at most, 2^-8 of their
    # block's largest (int8); averaged over 64 channels and the keys, logits keep far more
    assert len(got) == sum(n_blocks) and max(got) <= (2.0 ** -4 if dtype == E4 else 2.0 ** -5)
    for t, prompt, n in zip(out, prompts, n_blocks):
        assert len(t) == len(prompt) + 16 * n and torch.equal(t[:len(prompt)], prompt)
    assert all(torch.equal(a, b) for a, b in zip(out, go()))


# -- refusals of the calls ------------------------------------------------------------


@pytest.mark.gpu
def test_refusals(cuda):
    c = pool_case([(4, 60)], 2, 2, 16, I8, seed=1)
    d = on(c, cuda)
    batch = d["table"], d["starts"], d["kv"]
    kw = dict(max_q=4, max_kv=64)

    def attention(**over):
        e = {**d, **over}
        return paged_attention_pool(e["q"], e["k"], e["v"], *batch, 4, **kw, k_scales=e["k_scales"], v_scales=e["v_scales"],
                                    columns=e.get("columns"), out=e.get("out"))

    bad = [(dict(k_scales=None), "need scales"), (dict(k_scales=d["k_scales"][:1]), "scales must be"),
           (dict(k_scales=d["k_scales"].double()), "scales must be"), (dict(k_scales=d["k_scales"].cpu()), "one device"),
           (dict(v=d["v"].view(E4)), "one dtype"), (dict(k=d["k"][..., :32], v=d["v"][..., :32]), "64"),
           (dict(k=d["k"].view(torch.uint8), v=d["v"].view(torch.uint8)), "bf16 inputs only"),
           (dict(k=d["k"].to(BF), v=d["v"].to(BF)), "take none"),
           (dict(columns=torch.zeros(4, 2, 3, device=cuda)), "columns must be"),
           (dict(columns=torch.zeros(3, 2, 3, device=cuda, dtype=torch.int32)), "columns must be"),
           (dict(columns=torch.zeros(4, 1, 3, device=cuda, dtype=torch.int32)), "columns must be"),
           (dict(columns=torch.zeros(4, 2, 0, device=cuda, dtype=torch.int32)), "columns must be"),
           (dict(columns=torch.zeros(4, 2, 3, dtype=torch.int32)), "one device"),
           (dict(out=d["q"]), "overlap")]
    for over, text in bad:
        with pytest.raises(AssertionError, match=text):
            attention(**over)
    # results over the scales or the lists
    scales = torch.rand(4 * 2 * D // 2, device=cuda)
    out = scales.view(BF).view(4, 2, D)
    n = d["k_scales"].numel()
    with pytest.raises(AssertionError, match="overlap"):
        attention(out=out, v_scales=scales[:n].view(d["k_scales"].shape))
    with pytest.raises(AssertionError, match="overlap"):
        attention(out=out, columns=scales.view(torch.int32)[:24].view(4, 2, 3))
    with pytest.raises(AssertionError, match="need scales"):
        paged_attention(d["q"], d["k"], d["v"], *batch, 4, **kw)

    tables = [t.to(cuda) for t in rope_tables(D, 64)]
    qkv = torch.zeros((4, 6 * D), dtype=BF, device=cuda)

    def inputs(**over):
        e = {**d, **over}
        return paged_attention_inputs8(qkv, 2, *tables, e["k"], e["v"], e["k_scales"], e["v_scales"], *batch)

    for over, text in [(dict(v=d["k"]), "overlap"), (dict(v_scales=d["k_scales"]), "overlap"),
                       (dict(k=d["k"][:1].expand(d["k"].shape)), "twice|overlap"), (dict(k_scales=d["k_scales"][:1]), "scales"),
                       (dict(k_scales=d["k_scales"].transpose(0, 1)), "scales must be"),
                       (dict(k=d["k"].view(E4)), "one dtype")]:
        with pytest.raises(AssertionError, match=text):
            inputs(**over)
    with pytest.raises(AssertionError, match="need scales"):
        paged_attention_inputs(qkv, 2, *tables, d["k"], d["v"], *batch)
    with pytest.raises(AssertionError, match="int8 or float8"):
        page_values(d["k"].to(BF), d["v"].to(BF), d["k_scales"], d["v_scales"])

    bounds = torch.zeros((c["k"].shape[0], 2, 2, D), dtype=BF, device=cuda)
    for b, text in [(bounds[1:], "bounds must"), (bounds.float(), "bounds must"), (bounds.transpose(0, 1), "bounds must"),
                    (bounds.cpu(), "one device")]:
        with pytest.raises(AssertionError, match=text):
            page_bounds(d["k"], b, *batch, 4, d["k_scales"])
    for b, over, text in [(bounds.float(), {}, "bounds must"), (bounds[:, :, :1], {}, "bounds must"), (bounds, dict(top=2), "always taken"),
                          (bounds, dict(top=0), "top"), (bounds, dict(first=-1), "first"),
                          (bounds, dict(out=torch.zeros(4, 2, 5, device=cuda, dtype=torch.int64)), "out must"),
                          (bounds, dict(out=torch.zeros(4, 2, 6, device=cuda, dtype=torch.int32)), "out must")]:
        with pytest.raises(AssertionError, match=text):
            select_pages(d["q"], b, *batch, 4, 16, **{"top": 5, "max_q": 4, **over})
    torch.cuda.synchronize()
