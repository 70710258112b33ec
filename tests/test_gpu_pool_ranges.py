"""Lengths and starts out of range, and lists past the places that are read, against the definitions over what counts of them."""
from __future__ import annotations

import pytest
import torch

from _pool_util import BF, D, E4, I8, lists, pool_reference
from _serving_util import worst
from kernels.paged import page_bounds, paged_attention_pool, select_pages
from oracle import serving as orc

POOLS = [pytest.param(BF, id="bf16"), pytest.param(I8, id="int8"), pytest.param(E4, id="e4m3")]


def full_case(dtype, seqs, chunk, heads, kv_heads, page, max_kv, seed, pages=40):
    """A pool whose every slot holds a value, tables whose every entry is a page."""
    g = torch.Generator().manual_seed(seed)
    width = -(-max_kv // page) + 1
    c = {"table": torch.randint(0, pages, (seqs, width), generator=g, dtype=torch.int32), "k_scales": None, "v_scales": None}
    for name in ("k", "v"):
        x = torch.randn((pages, kv_heads, page, D), generator=g)
        if dtype == BF:
            c[name] = x.to(BF)
        else:
            c[name] = (x * 30).clamp(-127, 127).round().to(I8) if dtype == I8 else (x * 8).to(E4)
            c[name + "_scales"] = torch.exp2(torch.rand((pages, kv_heads, page // 16), generator=g) * 3 - 5)
    n = torch.randint(0, chunk + 1, (seqs,), generator=g)
    n[0], n[-1] = chunk, chunk
    c["starts"] = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(torch.int32)
    c["kv"] = (n + torch.randint(0, max_kv - chunk + 1, (seqs,), generator=g)).to(torch.int32)
    c["q"] = torch.randn((int(c["starts"][-1]), heads, D), generator=g).to(BF)
    return c


def attend(c, dev, bs, max_q, max_kv, total, columns=None):
    d = {k: t.to(dev) if torch.is_tensor(t) else t for k, t in c.items()}
    return paged_attention_pool(d["q"], d["k"], d["v"], d["table"], d["starts"], d["kv"], bs, max_q, max_kv, total,
                                k_scales=d["k_scales"], v_scales=d["v_scales"],
                                columns=None if columns is None else columns.to(dev))


def out_of_range(c, most):
    """The case with such lengths and starts; c's own become what they count as."""
    given = dict(c)
    given["kv"] = c["kv"].clone()
    given["kv"][::3] = 1 << 30
    given["kv"][2::7] = most + 1
    given["kv"][1::5] = -3
    given["kv"][-1] = 2 ** 31 - 1
    given["starts"] = c["starts"].clone()
    given["starts"][0], given["starts"][-1] = -(1 << 30), 1 << 30
    c["kv"] = given["kv"].clamp(0, most)
    return given


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", POOLS)
@pytest.mark.parametrize("seqs,chunk,heads,kv_heads", [(65, 1, 2, 1), (130, 16, 2, 1), (70, 40, 2, 1), (3, 40, 2, 2), (3, 500, 1, 1),
                                                       (66, 450, 1, 1)])
def test_lengths_and_starts_out_of_range(cuda, record_error, dtype, seqs, chunk, heads, kv_heads):
    """Lengths count as max_kv at most and 0 at least, starts as those of tokens that are there."""
    bs, page, max_kv = 16, 16, chunk + 299
    print(f"out of range {seqs} x {chunk} {heads}/{kv_heads} {dtype}", flush=True)
    c = full_case(dtype, seqs, chunk, heads, kv_heads, page, max_kv, seed=seqs + chunk)
    given = out_of_range(c, max_kv)
    ref, tol = pool_reference(c, bs)
    for total in (0, seqs * max_kv):
        record_error("bounded batch / bound", worst(attend(given, cuda, bs, chunk, max_kv, total), ref, tol), 1.0)
    columns = lists({**c, "max_kv": max_kv}, kv_heads, page, bs, 9, seed=seqs)
    ref, tol = pool_reference(c, bs, columns)
    record_error("bounded lists / bound", worst(attend(given, cuda, bs, chunk, max_kv, seqs * max_kv, columns), ref, tol), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", POOLS)
@pytest.mark.parametrize("seqs,chunk", [(5, 1), (70, 40), (3, 300)])
def test_bounds_and_selections_of_such_batches(cuda, dtype, seqs, chunk):
    """page_bounds takes the table's keys as the most of a sequence, select_pages max_kv."""
    page, most = 16, 16 * (-(-(chunk + 299) // 16))
    pages = seqs * (most // page)
    c = full_case(dtype, seqs, chunk, 2, 1, page, most, seed=seqs, pages=pages)
    c["table"] = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).to(torch.int32).view(seqs, -1)
    given = out_of_range(c, most)
    T = c["q"].shape[0]
    start = torch.randn((pages, 1, 2, D), generator=torch.Generator().manual_seed(1)).to(BF)
    want = orc.page_bounds(orc.pool_values(c["k"], c["k_scales"]).float().to(BF).double(), start, c["table"], c["starts"], c["kv"])
    d = {k: t.to(cuda) if torch.is_tensor(t) else t for k, t in given.items()}
    bounds = page_bounds(d["k"], start.to(cuda), d["table"], d["starts"], d["kv"], T, d["k_scales"])
    assert torch.equal(bounds.cpu(), want)
    out = torch.full((T, 1, 8), -2, dtype=torch.int32, device=cuda)
    select_pages(d["q"], bounds, d["table"], d["starts"], d["kv"], 16, page, 8, chunk, most, out=out)
    assert torch.equal(out.cpu(), orc.select_pages(c["q"], want, c["table"], c["starts"], c["kv"], 16, page, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", POOLS)
@pytest.mark.parametrize("chunk", [1, 16, 48])
def test_lists_are_read_as_far_as_the_sequence_has_columns(cuda, record_error, dtype, chunk):
    """Three columns: the first three places are read, whatever stands there. A column behind them is not."""
    page, max_kv, bs = 16, 48, 48
    c = full_case(dtype, 2, chunk, 2, 1, page, max_kv, seed=chunk)
    c["starts"], c["kv"] = torch.tensor([0, chunk, 2 * chunk], dtype=torch.int32), torch.tensor([48, 48], dtype=torch.int32)
    c["q"] = torch.cat([c["q"][:chunk], c["q"][:chunk]])
    for row in ([-1, -1, 0, 1, 2], [2, -1, 1, 0, -1], [-1, -1, -1, 0, 1], [0, 1, 2, -1, -1], [1, 7, 1 << 29, 0, 2], [-1, 2, -5, 2, 2]):
        columns = torch.tensor(row, dtype=torch.int32).expand(2 * chunk, 1, 5).contiguous()
        ref, tol = pool_reference(c, bs, columns)
        read = torch.tensor(row[:3] + [-1, -1], dtype=torch.int32).expand(2 * chunk, 1, 5).contiguous()
        assert torch.equal(pool_reference(c, bs, read)[0], ref), "the definition"
        o = attend(c, cuda, bs, chunk, max_kv, 96, columns)
        record_error("lists' places / bound", worst(o, ref, tol), 1.0)
        assert (o == 0).all() == (row[:3] == [-1, -1, -1])
