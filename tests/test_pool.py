"""8-bit pools and selected pages without a GPU: definitions, the cache, and every
refusal of the C ABI and the Python calls."""
from __future__ import annotations

import ctypes
import inspect

import pytest
import torch

from _pool_util import BF, D, E4, I8, lists, pool_case, values_of
from kernels import _native
from kernels.kv_cache import rope_tables
from kernels.paged import (PagedKVCache, page_bounds, page_values, paged_attention, paged_attention_inputs8,
                           paged_attention_pool, select_pages)
from oracle import serving as orc


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        import __graft_entry__
        __graft_entry__.build()
    return _native.lib()


@pytest.mark.parametrize("dtype,scale", [(I8, 10.0 / 127), (E4, 2.0 ** -5)])
def test_encoding_by_hand(dtype, scale):
    """10 needs 10 / 127, or 2^-5: 448 * 2^-5 = 14, 448 * 2^-6 = 7."""
    assert orc.needed_scale(10.0, dtype) == scale
    assert orc.needed_scale(0.0, dtype) == orc.needed_scale(1e-35, dtype) == 2.0 ** -100
    assert orc.needed_scale(448.0, E4) == 1.0 and orc.needed_scale(448.001, E4) == 2.0
    x = orc.codes_of(torch.tensor([0.5, 1.5, 2.5, 126.6, -300.0], dtype=torch.float64), I8)
    assert x.tolist() == [0, 2, 2, 127, -127]


def test_inputs_definition_keeps_earlier_tokens():
    """A later, larger token makes the block's scale grow by a power of two; the earlier ones stay within a step."""
    sin, cos = rope_tables(D, 64)
    k = torch.zeros(2, 1, 16, D, dtype=I8)
    v, ks, vs = k.clone(), torch.zeros(2, 1, 1), torch.zeros(2, 1, 1)
    table, g = torch.tensor([[1]], dtype=torch.int32), torch.Generator().manual_seed(0)
    x = torch.randn(16, 3 * D, generator=g).to(BF) * torch.exp2(torch.arange(16.0) / 3)[:, None].to(BF)
    for t in range(16):
        _, _, _, k, v, ks, vs = orc.paged_attention_inputs8(x[t:t + 1], 1, sin, cos, k, v, ks, vs, table,
                                                            torch.tensor([0, 1]), torch.tensor([t + 1]))
    got = orc.pool_values(v, vs)[1, 0]
    assert float((got - x[:, 2 * D:].double()).abs().max() / vs[1]) < 1.0
    assert float(vs[0]) == 0.0


def test_selected_definition():
    """With every column listed it is the dense attention; lists of one page see that page."""
    c = pool_case([(5, 60), (2, 3)], 2, 1, 16, BF, seed=3)
    v = values_of(c)
    args = v["q"], v["k"], v["v"], v["table"], v["starts"], v["kv"], 4
    every = torch.arange(5, dtype=torch.int32).expand(7, 1, 5)
    assert torch.equal(orc.paged_attention(*args, columns=every), orc.paged_attention(*args))
    one = orc.paged_attention(*args, columns=torch.full((7, 1, 1), 0, dtype=torch.int32))
    page = int(v["table"][0, 0])
    want = torch.softmax(v["q"][0, 0].double() @ v["k"][page, 0].t() / 8, dim=-1) @ v["v"][page, 0]
    assert torch.allclose(one[0, 0], want)


def test_select_definition_by_hand():
    q = torch.zeros(1, 1, D, dtype=BF)
    q[0, 0, 0], q[0, 0, 1] = 2.0, -1.0
    bounds = torch.zeros(6, 1, 2, D, dtype=BF)
    for p, (lo, hi) in enumerate([(1, 1), (-3, 5), (0, 4), (0, 4), (1, 2), (0, 0)]):
        bounds[p, 0, 0, 0], bounds[p, 0, 1, 0] = lo, hi
    table = torch.tensor([[0, 1, 2, 3, 4, 5]], dtype=torch.int32)
    args = q, bounds, table, torch.tensor([0, 1]), torch.tensor([96]), 1, 16
    # scores 2, 10, 8, 8, 4, 0; column 5 is the query's own
    assert orc.select_pages(*args, 3, first=0, recent=0).tolist() == [[[1, 2, 5]]]
    assert orc.select_pages(*args, 3, first=1, recent=0).tolist() == [[[0, 1, 5]]]
    assert orc.select_pages(*args, 4, first=0, recent=1).tolist() == [[[1, 2, 4, 5]]]
    assert orc.select_pages(*args, 8).tolist() == [[[0, 1, 2, 3, 4, 5, -1, -1]]]


def test_bounds_are_bounds():
    c = values_of(pool_case([(40, 30)], 2, 2, 32, BF, seed=4))
    b = orc.page_bounds(c["k"], torch.zeros(c["k"].shape[0], 2, 2, D, dtype=BF), c["table"], c["starts"], c["kv"])
    page = int(c["table"][0, 1])
    q = c["q"][0, 0].double()
    best = torch.maximum(q * b[page, 0, 0].double(), q * b[page, 0, 1].double()).sum()
    assert float((c["k"][page, 0] @ q).max()) <= float(best)
    assert (b[int(c["table"][0, 0])] != 0).any(), "the chunk begins in the first page"


def test_signatures():
    def params(f):
        return list(inspect.signature(f).parameters)
    pool, batch = ["k_pages", "v_pages"], ["page_table", "q_starts", "kv_lens"]
    assert params(paged_attention_pool) == params(paged_attention) + ["k_scales", "v_scales", "columns"]
    assert params(paged_attention_inputs8) == ["qkv", "n_heads", "sin_table", "cos_table", *pool, "k_scales", "v_scales",
                                               *batch, "out"]
    assert params(page_values) == [*pool, "k_scales", "v_scales"]
    assert params(page_bounds) == ["k_pages", "bounds", *batch, "tokens", "k_scales"]
    assert params(select_pages) == ["q", "bounds", *batch, "block_size", "page_size", "top", "max_q", "max_kv", "first",
                                    "recent", "out"]


def test_cache_of_any_type():
    for dtype in (BF, I8, E4):
        cache = PagedKVCache(2, 10, 3, 32, device="cpu", dtype=dtype, bounds=True)
        assert cache.k_pages.dtype == cache.v_pages.dtype == dtype and cache.bounds.shape == (2, 10, 3, 2, D)
        if dtype == BF:
            assert cache.scales(1) == (None, None)
        else:
            assert cache.scales(1)[0].shape == (10, 3, 2) and cache.scales(1)[0].dtype == torch.float32
    assert PagedKVCache(1, 1, 1, device="cpu").bounds is None
    with pytest.raises(AssertionError, match="bfloat16, int8 or float8_e4m3fn"):
        PagedKVCache(1, 1, 1, device="cpu", dtype=torch.float16)
    cache = PagedKVCache(1, 4, 1, device="cpu")
    batch = cache.batch([cache.add()], [3])
    with pytest.raises(AssertionError, match="bounds=True"):
        batch.update_bounds(0)
    with pytest.raises(AssertionError, match="bounds=True"):
        batch.attention(torch.zeros(3, 1, D, dtype=BF), 0, 16, top=4)


def test_custom_ops_fake_shapes():
    import kernels.ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        k = torch.empty(9, 2, 32, 64, dtype=I8)
        s = torch.empty(9, 2, 2)
        i = torch.empty(3, dtype=torch.int32)
        q = torch.ops.bd3.paged_qkv_rope8(torch.empty(7, 8 * 64, dtype=BF), 4, torch.empty(9, 32), torch.empty(9, 32), k, k,
                                          s, s, i[None], i, i)
        assert q.shape == (7, 4, 64) and q.dtype == BF
        bounds = torch.empty(9, 2, 2, 64, dtype=BF)
        torch.ops.bd3.page_bounds(k, bounds, i[None], i, i, 7, s)
        columns = torch.ops.bd3.select_pages(q, bounds, i[None], i, i, 16, 32, 5, 4)
        assert columns.shape == (7, 2, 5) and columns.dtype == torch.int32
        o = torch.ops.bd3.paged_attn_pool(q, k, k, i[None], i, i, 16, 4, k_scales=s, v_scales=s, columns=columns)
        assert o.shape == q.shape and o.dtype == BF


def test_cpu_tensors_raise(lib):
    c = pool_case([(4, 8)], 2, 2, 16, I8)
    batch = c["table"], c["starts"], c["kv"]
    with pytest.raises(AssertionError, match="CUDA"):
        paged_attention_pool(c["q"], c["k"], c["v"], *batch, 4, max_q=4, k_scales=c["k_scales"], v_scales=c["v_scales"])
    with pytest.raises(AssertionError, match="CUDA"):
        paged_attention_inputs8(torch.zeros(4, 6 * D, dtype=BF), 2, torch.zeros(9, 32), torch.zeros(9, 32), c["k"], c["v"],
                                c["k_scales"], c["v_scales"], *batch)
    with pytest.raises(AssertionError, match="CUDA"):
        page_values(c["k"], c["v"], c["k_scales"], c["v_scales"])
    bounds = torch.zeros(c["k"].shape[0], 2, 2, D, dtype=BF)
    with pytest.raises(AssertionError, match="CUDA"):
        page_bounds(c["k"], bounds, *batch, 4, c["k_scales"])
    with pytest.raises(AssertionError, match="CUDA"):
        select_pages(c["q"], bounds, *batch, 4, 16, 4, 4)


def test_lists_helper():
    c = pool_case([(9, 70), (4, 0)], 2, 2, 16, BF)
    out = lists(c, 2, 16, 4, 4, seed=1)
    assert out.shape == (13, 2, 4) and out.dtype == torch.int32


# -- the C ABI: every refusal comes before any HIP call ------------------------

P = 4096  # a pointer that is never followed
AST = [256, 64, 2048, 1024, 64, 2048, 1024, 64, 256, 64, 4, 20, 10]
RST = [512, 256, 64, 2048, 1024, 64, 2048, 1024, 64, 4]


def at(i, value, base):
    st = list(base)
    st[i] = value
    return st


def i64(st):
    return None if st is None else (ctypes.c_int64 * len(st))(*st)


BATCH = dict(table=P, starts=P, lens=P, seqs=2, tokens=8, heads=4, kv_heads=2, head_dim=64, pages=9, page=16, width=4)


def attn(lib, **kw):
    a = dict(BATCH, q=P, k=P, v=P, ks=P, vs=P, pool=1, o=P, columns=P, top=5, max_q=4, max_kv=64, total=100, bs=16, st=AST,
             scale=0.125, ws=None, ws_bytes=0)
    a.update(kw)
    return lib.bd3_paged_attn_pool(
        a["q"], a["k"], a["v"], a["ks"], a["vs"], a["pool"], a["o"], a["table"], a["starts"], a["lens"], a["columns"], a["top"],
        a["seqs"], a["tokens"], a["heads"], a["kv_heads"], a["head_dim"], a["pages"], a["page"], a["width"], a["max_q"],
        a["max_kv"], a["total"], a["bs"], i64(a["st"]), a["scale"], a["ws"], a["ws_bytes"], None)


def rope(lib, **kw):
    a = dict(BATCH, qkv=P, sin=P, cos=P, max_pos=64, q=P, k=P, v=P, ks=P, vs=P, pool=2, st=RST)
    a.update(kw)
    return lib.bd3_paged_qkv_rope8(
        a["qkv"], a["sin"], a["cos"], a["max_pos"], a["q"], a["k"], a["v"], a["ks"], a["vs"], a["pool"], a["table"], a["starts"],
        a["lens"], a["seqs"], a["tokens"], a["heads"], a["kv_heads"], a["head_dim"], a["pages"], a["page"], a["width"],
        i64(a["st"]), None)


def values(lib, **kw):
    a = dict(k=P, v=P, ks=P, vs=P, pool=1, ko=P, vo=P, pages=9, kv_heads=2, page=16, head_dim=64,
             st=[2048, 1024, 64, 2048, 1024, 64])
    a.update(kw)
    return lib.bd3_page_values(a["k"], a["v"], a["ks"], a["vs"], a["pool"], a["ko"], a["vo"], a["pages"], a["kv_heads"],
                               a["page"], a["head_dim"], i64(a["st"]), None)


def bounds_call(lib, **kw):
    a = dict(BATCH, k=P, ks=P, pool=1, bounds=P, st=[2048, 1024, 64, 4])
    a.update(kw)
    return lib.bd3_page_bounds(a["k"], a["ks"], a["pool"], a["bounds"], a["table"], a["starts"], a["lens"], a["seqs"], a["tokens"],
                               a["kv_heads"], a["head_dim"], a["pages"], a["page"], a["width"], i64(a["st"]), None)


def select(lib, **kw):
    a = dict(BATCH, q=P, bounds=P, out=P, max_q=4, max_kv=64, bs=16, top=4, first=1, recent=1, st=[256, 64, 4], ws=P,
             ws_bytes=1 << 30)
    a.update(kw)
    return lib.bd3_select_pages(a["q"], a["bounds"], a["table"], a["starts"], a["lens"], a["out"], a["seqs"], a["tokens"],
                                a["heads"], a["kv_heads"], a["head_dim"], a["pages"], a["page"], a["width"], a["max_q"],
                                a["max_kv"], a["bs"], a["top"], a["first"], a["recent"], i64(a["st"]), a["ws"], a["ws_bytes"],
                                None)


SHAPES = [(dict(kv_heads=0), "multiple"), (dict(head_dim=128), "head_dim"), (dict(pages=0), "at least one page"),
          (dict(page=24), "power of two"), (dict(page=8), "power of two"), (dict(page=2048), "power of two"),
          (dict(width=1 << 27), "2^30"), (dict(table=None), "page_table"), (dict(starts=None), "q_starts"),
          (dict(lens=None), "kv_lens"), (dict(st=None), "strides is NULL"), (dict(seqs=-1), ">= 0"), (dict(tokens=-1), ">= 0")]
POOL = [(dict(pool=3), "pool_type"), (dict(pool=-1), "pool_type"), (dict(ks=None), "8-bit pools have scales"),
        (dict(ks=P + 2), "4-byte aligned"), (dict(k=None), "k_pages"), (dict(k=P + 8), "k_pages")]


@pytest.mark.parametrize("kw,text", SHAPES + POOL + [
    (dict(pool=0), "bf16 pools none"), (dict(v=P + 8), "v_pages"), (dict(vs=None), "8-bit pools have scales"),
    (dict(heads=3), "multiple"), (dict(q=None), "q must"), (dict(o=P + 2), "o must"), (dict(bs=0), "block_size"),
    (dict(top=0), "top"), (dict(max_q=-1), "max_q"), (dict(max_kv=65), "exceeds"), (dict(scale=0.0), "scale"),
    (dict(st=at(4, 72, AST)), "multiple of 16"), (dict(st=at(5, 8, AST)), "multiple of 16"),
    (dict(st=at(7, 1 << 24, AST)), "slot strides"), (dict(st=at(11, -1, AST)), "columns"), (dict(st=at(12, -1, AST)), "columns"),
    (dict(columns=P + 1), "columns"), (dict(seqs=1 << 20, tokens=1 << 30, max_q=4096, bs=1), "too large"),
    (dict(columns=None, seqs=1 << 20, tokens=1 << 30, max_q=1 << 20), "too large")])
def test_attention_refusals(lib, kw, text):
    assert attn(lib, **kw) == _native.BD3_EINVAL
    assert text in _native.last_error()


@pytest.mark.parametrize("kw,text", SHAPES + POOL + [
    (dict(pool=0), "pool_type"), (dict(vs=P + 1), "4-byte aligned"), (dict(v=None), "v_pages"), (dict(heads=3), "multiple"),
    (dict(qkv=P + 2), "qkv"), (dict(q=None), "q_out"), (dict(sin=None), "sin_table"), (dict(max_pos=0), "max_pos"),
    (dict(st=at(5, 72, RST)), "multiple of 16"), (dict(st=at(9, -1, RST)), "page_table stride"),
    (dict(tokens=1 << 28, heads=64), "too large"), (dict(seqs=1 << 26, tokens=1 << 26, heads=2), "too large")])
def test_inputs_refusals(lib, kw, text):
    assert rope(lib, **kw) == _native.BD3_EINVAL
    assert text in _native.last_error()


@pytest.mark.parametrize("kw,text", POOL + [
    (dict(pool=0), "pool_type"), (dict(v=P + 8), "v_pages"), (dict(vs=None), "scales"), (dict(ko=None), "k_out"),
    (dict(vo=P + 8), "v_out"), (dict(pages=-1), "pages"), (dict(kv_heads=0), "kv_heads"), (dict(page=8), "power of two"),
    (dict(head_dim=32), "head_dim"), (dict(st=None), "strides is NULL"), (dict(pages=1 << 24), "too large"),
    (dict(st=[2048, 1024, 64, 2048, 1000, 64]), "multiple of")])
def test_values_refusals(lib, kw, text):
    assert values(lib, **kw) == _native.BD3_EINVAL
    assert text in _native.last_error()


@pytest.mark.parametrize("kw,text", SHAPES + POOL + [
    (dict(pool=0), "bf16 pools none"), (dict(bounds=None), "bounds"), (dict(bounds=P + 8), "bounds"),
    (dict(st=[2048, 1024, 72, 4]), "multiple of 16"), (dict(st=[2048, 1024, 64, -1]), "page_table stride"),
    (dict(seqs=1 << 30, tokens=1 << 30), "too large")])
def test_bounds_refusals(lib, kw, text):
    assert bounds_call(lib, **kw) == _native.BD3_EINVAL
    assert text in _native.last_error()


@pytest.mark.parametrize("kw,text", SHAPES + [
    (dict(heads=3), "multiple"), (dict(bs=0), "block_size"), (dict(max_q=-1), "max_q"), (dict(max_kv=65), "exceeds"),
    (dict(first=-1), "first"), (dict(recent=-1), "recent"), (dict(top=2), "always taken"), (dict(top=3, bs=17), "always taken"),
    (dict(top=0, max_kv=0), "top"), (dict(q=None), "q must"), (dict(bounds=P + 2), "bounds"), (dict(out=None), "out"),
    (dict(out=P + 2), "out"), (dict(st=[256, 60, 4]), "q stride"), (dict(st=[256, 64, -1]), "page_table stride"),
    (dict(ws_bytes=100, width=2049, max_kv=2049 * 16), "too small"), (dict(ws=None, width=2049, max_kv=2049 * 16), "workspace must"),
    (dict(ws=P + 4, width=2049, max_kv=2049 * 16), "workspace must"), (dict(seqs=1 << 24, tokens=1 << 24, bs=1), "too large"),
    (dict(seqs=1 << 12, tokens=1 << 12, bs=1, width=1 << 18, max_kv=1 << 22, top=9), "too large")])
def test_select_refusals(lib, kw, text):
    assert select(lib, **kw) == _native.BD3_EINVAL
    assert text in _native.last_error()


def test_no_work_is_no_launch(lib):
    for f, which in ((attn, ("seqs", "tokens", "max_q")), (rope, ("seqs", "tokens")), (bounds_call, ("seqs", "tokens")),
                     (select, ("seqs", "tokens", "max_q")), (values, ("pages",))):
        for name in which:
            assert f(lib, **{name: 0}) == 0, (f, name)


def test_workspaces(lib):
    size = lib.bd3_paged_attn_pool_workspace_bytes
    assert size(1, 2, 8, 4, 2, 16, 4, 64, 100, 16, 0) == 0
    assert size(1, 2, 8, 4, 2, 16, 4, 64, 100, 16, 5) == 0
    # the bf16 pool without lists is bd3_paged_attn's
    for args in ((1, 16, 12, 12, 16, 8192, 8192), (8, 128, 12, 4, 16, 4000, 9000)):
        assert size(0, *args[:4], 16, *args[4:], 16, 0) == lib.bd3_paged_attn_workspace_bytes(*args)
    # lists: cut by their keys, not by the cache's
    assert size(0, 1, 1, 12, 12, 16, 1, 1 << 20, 1 << 20, 1, 4) == 0
    need = size(0, 1, 1, 12, 12, 64, 1, 1 << 20, 1 << 20, 1, 128)
    assert 0 < need <= 12 * 64 * 260 + 512
    assert attn(lib, seqs=1, tokens=1, heads=12, kv_heads=12, page=64, width=1 << 14, max_q=1, max_kv=1 << 20, total=1 << 20,
                bs=1, top=128, ws=P, ws_bytes=need - 1) == _native.BD3_EINVAL
    assert "too small" in _native.last_error()
    for bad in ((1, 0, 8, 4, 2, 16, 4, 64, 100, 16, 0), (1, 2, 8, 4, 2, 16, 4, 64, 100, 0, 5), (1, 2, 8, 4, 2, 0, 4, 64, 100, 16, 5),
                (1, 2, 8, 4, 2, 16, 4, 64, 100, 16, -1)):
        assert size(*bad) == 0
    size = lib.bd3_select_pages_workspace_bytes
    for bad in ((0, 8, 2, 16, 64, 16), (2, 0, 2, 16, 64, 16), (2, 8, 0, 16, 64, 16), (2, 8, 2, 8, 64, 16), (2, 8, 2, 16, 0, 16),
                (2, 8, 2, 16, (1 << 30) + 1, 16), (2, 8, 2, 16, 1 << 20, 0)):
        assert size(*bad) == 0
    assert size(200, 200, 2, 16, 2048 * 16, 16) == 0  # a workgroup's LDS
    assert size(200, 200, 2, 16, 2048 * 16 + 1, 16) > 0
    assert size(1, 1, 4, 16, 256 * 16, 1) == 0 and size(1, 1, 4, 16, 1000 * 16, 1) > 0  # few items, spread over the CUs


def test_selection_without_room_for_the_columns_always_taken(lib):
    """first + recent + those a block can lie in, unless the table has fewer."""
    # an absent q shows that `top` was accepted
    for bs, page in ((1, 16), (16, 16), (17, 16), (7, 64), (7, 16), (64, 64), (65, 64), (32, 16), (48, 32), (200, 16)):
        kw = dict(bs=bs, page=page, width=1024, max_kv=1024 * page, q=None)
        own = max((a + bs - 1) // page - a // page + 1 for a in range(0, bs * page, bs))
        assert select(lib, **kw, top=2 + own - 1) == _native.BD3_EINVAL and "always taken" in _native.last_error()
        assert select(lib, **kw, top=2 + own) == _native.BD3_EINVAL and "q must" in _native.last_error()
    assert select(lib, bs=1 << 30, top=4, q=None) == _native.BD3_EINVAL and "q must" in _native.last_error()
