"""The selection of pages does not depend on bounds that it does not rank: those of the columns always taken, of pages that
no column names, of columns without a page."""
from __future__ import annotations

import pytest
import torch

from _pool_util import BF, D
from kernels import _native
from kernels.paged import select_pages

KINDS = [pytest.param(x, id=str(x)) for x in (float("inf"), float("-inf"), float("nan"), 3e38, -3e38)]


def case(seqs, heads, kv_heads, columns, page, top, dev, seed=0):
    """A token of each sequence over `columns` pages of its own; page 0 belongs to none, one entry in the middle of a
    sequence's table is no page."""
    g = torch.Generator().manual_seed(seed)
    table = 1 + torch.arange(seqs * columns, dtype=torch.int32).view(seqs, columns)
    table[:, columns // 3] = -1
    middle = torch.randn((seqs * columns + 1, kv_heads, 1, D), generator=g)
    bounds = torch.cat([middle - 1, middle + 1], dim=2).to(BF)
    q = torch.randn((seqs, heads, D), generator=g).to(BF)
    starts = torch.arange(seqs + 1, dtype=torch.int32)
    kv = torch.full((seqs,), columns * page - 3, dtype=torch.int32)
    return dict(q=q.to(dev), bounds=bounds.to(dev), table=table.to(dev), starts=starts.to(dev), kv=kv.to(dev), page=page, top=top)


def poisoned(c, value):
    """Bounds of the first column, the last two (the token's own and the one before), and page 0."""
    bounds = c["bounds"].clone()
    bounds[0] = value
    for col in (0, -1, -2):
        bounds[c["table"][:, col].long()] = value
    return bounds


def pick(c, bounds):
    return select_pages(c["q"], bounds, c["table"], c["starts"], c["kv"], 1, c["page"], c["top"], 1)


def summed_again(c, bounds):
    """By the C entry point with a workspace of the caller's: the columns whose scores were summed in 64 bits."""
    lib = _native.lib()
    (T, H, _), KH, B, width = c["q"].shape, bounds.shape[1], c["table"].shape[0], c["table"].shape[1]
    kv = width * c["page"]
    need = lib.bd3_select_pages_workspace_bytes(B, T, KH, c["page"], kv, 1)
    assert need > 0, "a launch that scores, and one that chooses"
    ws = torch.full((need // 8 + 1,), 7.0, dtype=torch.float64, device=bounds.device)
    out = torch.full((T, KH, c["top"]), -2, dtype=torch.int32, device=bounds.device)
    st = (_native.ctypes.c_int64 * 3)(c["q"].stride(0), c["q"].stride(1), c["table"].stride(0))
    rc = lib.bd3_select_pages(c["q"].data_ptr(), bounds.data_ptr(), c["table"].data_ptr(), c["starts"].data_ptr(),
                              c["kv"].data_ptr(), out.data_ptr(), B, T, H, KH, D, bounds.shape[0], c["page"], width, 1, kv, 1,
                              c["top"], 1, 1, st, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, _native.last_error()
    padded = -(-width // 16) * 16
    return out, (ws[:T * KH * padded] != 7.0).view(T, KH, padded)


@pytest.mark.gpu
@pytest.mark.parametrize("value", KINDS)
@pytest.mark.parametrize("columns", [300, 1000, 2500, 9000])
def test_unranked_bounds_put_no_column_in_doubt(cuda, columns, value):
    """Two launches, whose sums lie in the workspace: the same columns are summed again as without them (where the border's
    scores lie close; all of them if the bound of the errors took such bounds in)."""
    c = case(2, 4, 2, columns, 16, 40, cuda, seed=columns)
    want, clean = summed_again(c, c["bounds"])
    assert torch.equal(want, pick(c, c["bounds"]))
    got, again = summed_again(c, poisoned(c, value))
    assert torch.equal(got, want)
    assert int((again != clean).sum()) == 0


def us(f, calls=20):
    for _ in range(3):
        f()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(calls):
        f()
    end.record()
    end.synchronize()
    return begin.elapsed_time(end) / calls * 1e3


@pytest.mark.gpu
@pytest.mark.parametrize("value", KINDS)
def test_unranked_bounds_cost_nothing(cuda, value):
    """One launch, whose sums stay in the workgroup: the time tells (15 to 20 us; above 300 if every column is summed again)."""
    c = case(24, 8, 8, 1000, 16, 40, cuda, seed=1)
    bad = poisoned(c, value)
    want = pick(c, c["bounds"])
    assert torch.equal(pick(c, bad), want)
    clean = us(lambda: pick(c, c["bounds"]))
    print(f"clean {clean:.1f} us, with {value} {us(lambda: pick(c, bad)):.1f}", flush=True)
    assert us(lambda: pick(c, bad)) < 4 * clean + 20
