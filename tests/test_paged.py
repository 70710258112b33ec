"""The ragged serving operators without a GPU: their definitions against dense
torch, the cache's bookkeeping, and every refusal of the C ABI and the Python
calls."""
from __future__ import annotations

import ctypes
import inspect

import pytest
import torch

from _serving_util import BF, D, paged_case
from kernels import _native
from kernels.paged import PagedKVCache, paged_attention, paged_attention_inputs
from kernels.sampling import adjust_logits
from oracle import serving as orc


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        import __graft_entry__
        __graft_entry__.build()
    return _native.lib()


def test_attention_definition_against_dense():
    c = paged_case([(8, 24), (3, 0), (0, 9), (20, 13)], 4, 2, 16, seed=1)
    got = orc.paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["kv"], 8)
    for b, (n, ctx) in enumerate([(8, 24), (3, 0), (0, 9), (20, 13)]):
        if n == 0:
            continue
        kv = n + ctx
        ids = c["table"][b, :-(-kv // 16)].long()
        k = c["k"][ids].permute(1, 0, 2, 3).reshape(2, -1, D)[:, :kv].double().repeat_interleave(2, dim=0)
        v = c["v"][ids].permute(1, 0, 2, 3).reshape(2, -1, D)[:, :kv].double().repeat_interleave(2, dim=0)
        s = int(c["starts"][b])
        q = c["q"][s:s + n].transpose(0, 1).double()
        pos = torch.arange(ctx, kv)
        mask = torch.arange(kv)[None] // 8 <= pos[:, None] // 8
        want = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=mask)
        assert torch.allclose(got[s:s + n].transpose(0, 1), want, atol=1e-12)


def test_inputs_definition_against_complex_rotation():
    from kernels.kv_cache import rope_tables
    c = paged_case([(5, 18), (17, 0)], 2, 1, 16, seed=2, poison=False)
    qkv = torch.randn(22, 4 * D).to(BF)
    sin, cos = rope_tables(D, 64)
    q, k, v = orc.paged_attention_inputs(qkv, 2, sin, cos, c["k"], c["v"], c["table"], c["starts"], c["kv"])
    x = qkv.double().view(22, 4, 2, 32)
    pos = torch.cat([torch.arange(18, 23), torch.arange(17)])
    z = torch.complex(x[:, :3, 0], x[:, :3, 1]) * torch.complex(cos[pos].double(), sin[pos].double())[:, None]
    z = torch.cat([z.real, z.imag], -1)
    assert torch.allclose(q, z[:, :2])
    for t, (b, p) in enumerate([(0, p) for p in range(18, 23)] + [(1, p) for p in range(17)]):
        page = int(c["table"][b, p // 16])
        assert torch.allclose(k[page, :, p % 16], z[t, 2:])
        assert torch.equal(v[page, :, p % 16], qkv[t].double().view(4, D)[3:])


def test_logits_definition_by_hand():
    x = torch.tensor([[[2.0, -2.0, 1.0, 4.0]]])
    got = orc.adjust_logits(x, torch.tensor([[0, 1, 1, 9, -1, 3]]), torch.tensor([5]), 2.0, 0.5, 0.25,
                            bias=torch.tensor([0.0, 0.0, 1.0, 0.0]), allowed=torch.tensor([0b0111]), fill=-9.0)
    assert got.tolist() == [[[1.0 - 0.75, -4.0 - 1.25, 2.0, -9.0]]]


def test_signatures():
    def params(f):
        return list(inspect.signature(f).parameters)
    batch = ["k_pages", "v_pages", "page_table", "q_starts", "kv_lens"]
    assert params(paged_attention) == ["q", *batch, "block_size", "max_q", "max_kv", "total_kv", "out"]
    assert params(paged_attention_inputs) == ["qkv", "n_heads", "sin_table", "cos_table", *batch, "out"]
    assert params(adjust_logits) == ["logits", "tokens", "lengths", "repetition", "frequency", "presence", "bias",
                                     "allowed", "fill", "out"]


def test_cache_bookkeeping():
    cache = PagedKVCache(2, 10, 2, 16, device="cpu")
    a, b = cache.add(), cache.add()
    batch = cache.batch([a, b], [20, 1])
    assert batch.q_starts.tolist() == [0, 20, 21] and batch.kv_lens.tolist() == [20, 1]
    assert (batch.max_q, batch.max_kv, batch.total_kv, batch.tokens) == (20, 20, 21, 21)
    assert batch.page_table.shape == (2, 2) and batch.page_table[1, 1] == -1
    assert cache.free_pages == 7
    again = cache.batch([a, b], [20, 1])  # not committed: the same pages
    assert torch.equal(again.page_table, batch.page_table) and cache.free_pages == 7
    again.commit()
    assert cache.length(a) == 20 and cache.length(b) == 1
    with pytest.raises(AssertionError, match="moved on"):
        batch.commit()
    assert cache.length(a) == 20
    step = cache.batch([b, a], [15, 13])  # in any order; a needs a third page, b none
    assert cache.free_pages == 6 and step.kv_lens.tolist() == [16, 33]
    pages = step.page_table.flatten().tolist()
    assert len({p for p in pages if p >= 0}) == 4
    with pytest.raises(RuntimeError, match="6 free pages, the batch needs 7"):
        cache.batch([a, b], [1, 16 * 7])
    assert cache.free_pages == 6
    cache.free(a)
    assert cache.free_pages == 9
    with pytest.raises(AssertionError, match="moved on"):
        step.commit()
    assert cache.length(b) == 1, "nothing is committed of a batch that is refused"
    with pytest.raises(AssertionError, match="unknown"):
        cache.batch([a], [1])
    with pytest.raises(AssertionError, match="occurs once"):
        cache.batch([b, b], [1, 1])
    with pytest.raises(AssertionError, match=">= 0"):
        cache.batch([b], [-1])
    with pytest.raises(AssertionError, match="page_size"):
        PagedKVCache(1, 1, 1, 24, device="cpu")
    empty = cache.batch([], [])
    assert empty.page_table.shape == (0, 1) and empty.max_q == 0


def test_custom_ops_fake_shapes():
    import kernels.ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        k = torch.empty(9, 2, 16, 64, dtype=BF)
        i = torch.empty(3, dtype=torch.int32)
        q = torch.ops.bd3.paged_qkv_rope(torch.empty(7, 8 * 64, dtype=BF), 4, torch.empty(9, 32), torch.empty(9, 32), k, k,
                                         i[None], i, i)
        assert q.shape == (7, 4, 64) and q.dtype == BF
        o = torch.ops.bd3.paged_attn(q, k, k, i[None], i, i, 16, 4)
        assert o.shape == q.shape and o.dtype == BF


def test_cpu_tensors_raise(lib):
    c = paged_case([(4, 8)], 2, 2, 16)
    with pytest.raises(AssertionError, match="CUDA"):
        paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["kv"], 4, max_q=4)
    with pytest.raises(AssertionError, match="CUDA"):
        paged_attention_inputs(torch.zeros(4, 6 * D, dtype=BF), 2, torch.zeros(9, 32), torch.zeros(9, 32), c["k"], c["v"],
                               c["table"], c["starts"], c["kv"])
    with pytest.raises(AssertionError, match="CUDA"):
        adjust_logits(torch.zeros(2, 2, 8))


# -- the C ABI: every refusal comes before any HIP call ------------------------

P = 4096  # a pointer that is never followed


def attn(lib, **kw):
    a = dict(q=P, k=P, v=P, o=P, table=P, starts=P, lens=P, seqs=2, tokens=8, heads=4, kv_heads=2, head_dim=64, pages=9,
             page=16, width=4, max_q=4, max_kv=64, total=100, bs=16, st=[256, 64, 2048, 1024, 64, 2048, 1024, 64, 256, 64, 4],
             scale=0.125, ws=None, ws_bytes=0)
    a.update(kw)
    st = None if a["st"] is None else (ctypes.c_int64 * 11)(*a["st"])
    return lib.bd3_paged_attn(a["q"], a["k"], a["v"], a["o"], a["table"], a["starts"], a["lens"], a["seqs"], a["tokens"],
                              a["heads"], a["kv_heads"], a["head_dim"], a["pages"], a["page"], a["width"], a["max_q"],
                              a["max_kv"], a["total"], a["bs"], st, a["scale"], a["ws"], a["ws_bytes"], None)


def rope(lib, **kw):
    a = dict(qkv=P, sin=P, cos=P, max_pos=64, q=P, k=P, v=P, table=P, starts=P, lens=P, seqs=2, tokens=8, heads=4,
             kv_heads=2, head_dim=64, pages=9, page=16, width=4, st=[512, 256, 64, 2048, 1024, 64, 2048, 1024, 64, 4])
    a.update(kw)
    st = None if a["st"] is None else (ctypes.c_int64 * 10)(*a["st"])
    return lib.bd3_paged_qkv_rope(a["qkv"], a["sin"], a["cos"], a["max_pos"], a["q"], a["k"], a["v"], a["table"],
                                  a["starts"], a["lens"], a["seqs"], a["tokens"], a["heads"], a["kv_heads"], a["head_dim"],
                                  a["pages"], a["page"], a["width"], st, None)


def at(i, value, base):
    st = list(base)
    st[i] = value
    return st


AST = [256, 64, 2048, 1024, 64, 2048, 1024, 64, 256, 64, 4]
RST = [512, 256, 64, 2048, 1024, 64, 2048, 1024, 64, 4]
POOL = [(dict(heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "multiple"), (dict(head_dim=128), "head_dim"),
        (dict(pages=0), "at least one page"), (dict(width=0), "at least one page"), (dict(page=24), "power of two"),
        (dict(page=8), "power of two"), (dict(page=2048), "power of two"), (dict(width=1 << 27, page=16), "2^30"),
        (dict(table=None), "page_table"), (dict(starts=None), "q_starts"), (dict(lens=None), "kv_lens"),
        (dict(st=None), "strides is NULL"), (dict(seqs=-1), ">= 0"), (dict(tokens=-1), ">= 0"),
        (dict(k=None), "k_pages"), (dict(v=P + 8), "v_pages")]


@pytest.mark.parametrize("kw,text", POOL + [
    (dict(q=None), "q must"), (dict(o=P + 2), "o must"), (dict(bs=0), "block_size"), (dict(max_q=-1), "max_q"),
    (dict(max_kv=65), "exceeds"), (dict(total=-1), "total_kv"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(st=at(0, 4, AST)), "q stride"), (dict(st=at(4, 63, AST)), "k_pages stride"),
    (dict(st=at(7, 1 << 24, AST)), "slot strides"), (dict(st=at(9, -8, AST)), "o stride"),
    (dict(st=at(10, -1, AST)), "page_table stride"),
    (dict(seqs=1 << 20, tokens=1 << 30, max_q=4096), "too large"),
])
def test_attention_refusals(lib, kw, text):
    assert attn(lib, **kw) == _native.BD3_EINVAL
    assert text in _native.last_error()


@pytest.mark.parametrize("kw,text", POOL + [
    (dict(qkv=P + 2), "qkv"), (dict(q=None), "q_out"), (dict(sin=None), "sin_table"), (dict(cos=P + 4), "sin_table"),
    (dict(max_pos=0), "max_pos"), (dict(st=at(0, 513, RST)), "qkv stride"), (dict(st=at(9, -1, RST)), "page_table stride"),
    (dict(tokens=1 << 28, heads=64, kv_heads=2), "too large"),
])
def test_inputs_refusals(lib, kw, text):
    assert rope(lib, **kw) == _native.BD3_EINVAL
    assert text in _native.last_error()


def test_no_work_is_no_launch(lib):
    for kw in (dict(seqs=0), dict(tokens=0), dict(max_q=0)):
        assert attn(lib, **kw) == 0
    for kw in (dict(seqs=0), dict(tokens=0)):
        assert rope(lib, **kw) == 0


def test_workspace(lib):
    size = lib.bd3_paged_attn_workspace_bytes
    assert size(2, 8, 4, 2, 4, 64, 100) == 0  # nothing to cut
    need = size(1, 16, 12, 12, 16, 8192, 8192)
    assert need > 0 and need % 4 == 0
    kw = dict(seqs=1, heads=12, kv_heads=12, tokens=16, max_q=16, width=512, max_kv=8192, total=8192)
    assert attn(lib, **kw, ws=P, ws_bytes=need - 1) == _native.BD3_EINVAL and "too small" in _native.last_error()
    assert attn(lib, **kw, ws=None, ws_bytes=need) == _native.BD3_EINVAL and "aligned" in _native.last_error()
    for bad in ((0, 16, 12, 12, 16, 8192, 1), (1, 0, 12, 12, 16, 8192, 1), (1, 16, 0, 0, 16, 8192, 1),
                (1, 16, 12, 12, 0, 8192, 1), (1, 16, 12, 12, 16, -1, 1), (1, 16, 12, 12, 16, (1 << 30) + 1, 1),
                (1, 16, 12, 12, 16, 8192, -1)):
        assert size(*bad) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), ">= 0"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 30) + 1), "vocab"), (dict(fp32=2), "logits_fp32"), (dict(x=None), "non-NULL"),
    (dict(out=P + 1), "aligned to their elements"), (dict(tokens=P + 4), "8 bytes"), (dict(pen=[0.0, 0, 0]), "repetition"),
    (dict(pen=[float("inf"), 0, 0]), "repetition"), (dict(pen=[1.0, float("nan"), 0]), "frequency"), (dict(pen=None), "penalties"),
    (dict(fill=float("-inf")), "fill"), (dict(fill=-3.4e38), "fill"), (dict(st=[-1] + [0] * 7), "stride[0]"), (dict(st=None), "strides"),
    (dict(batch=1 << 22, vocab=1 << 20), "too large")])
def test_logits_refusals(lib, kw, text):
    a = dict(x=P, fp32=0, out=P, batch=2, rows=3, vocab=100, tokens=P, history=5, lens=None, pen=[1.0, 0.0, 0.0],
             fill=-1e6, st=[300, 100, 300, 100, 5, 0, 0, 0])
    a.update(kw)
    pen = None if a["pen"] is None else (ctypes.c_float * 3)(*a["pen"])
    st = None if a["st"] is None else (ctypes.c_int64 * 8)(*a["st"])
    assert lib.bd3_adjust_logits(a["x"], a["fp32"], a["out"], a["batch"], a["rows"], a["vocab"], a["tokens"], a["history"],
                                 a["lens"], pen, None, None, None, None, None, a["fill"], st, None) == _native.BD3_EINVAL
    assert text in _native.last_error()


@pytest.mark.parametrize("kw", [dict(history=(1 << 31) - 1), dict(history=(1 << 30) + 1), dict(rows=(1 << 31) - 1, vocab=1),
                                dict(rows=(1 << 30) + 1, vocab=1), dict(rows=1 << 30, vocab=1)])
def test_logits_sizes_whose_indices_would_wrap(lib, kw):
    """Indices into the history and the rows are 32 bits wide and run up to a
    workgroup's worth past the last one."""
    a = dict(batch=1, rows=3, vocab=100, history=5)
    a.update(kw)
    pen, st = (ctypes.c_float * 3)(1.0, 0.0, 0.0), (ctypes.c_int64 * 8)(300, 100, 300, 100, 5, 0, 0, 0)
    assert lib.bd3_adjust_logits(P, 0, P, a["batch"], a["rows"], a["vocab"], P, a["history"], None, pen, None, None, None,
                                 None, None, -1e6, st, None) == _native.BD3_EINVAL
    assert "2^30" in _native.last_error() or "too large" in _native.last_error()


def test_attention_rows_beyond_32_bits(lib):
    """max_q * heads / kv_heads rows of 2^32 and more do not fit the tile numbers."""
    kw = dict(seqs=1, tokens=1 << 30, heads=1 << 24, kv_heads=1, max_q=1 << 30, total=64)
    assert attn(lib, **kw) == _native.BD3_EINVAL
    assert "too large" in _native.last_error()
    assert lib.bd3_paged_attn_workspace_bytes(1, 1 << 30, 1 << 24, 1, 1 << 30, 64, 64) == 0
    assert lib.bd3_paged_attn_workspace_bytes(1, 1 << 30, 1 << 24, 1, 1 << 30, 1 << 20, 1 << 20) == 0


def test_totals_beyond_the_bound_are_the_bound(lib):
    size = lib.bd3_paged_attn_workspace_bytes
    for seqs, tokens, heads, kv_heads, max_q, max_kv in ((1, 16, 12, 12, 16, 8192), (2, 32, 12, 12, 16, 8192)):
        most = size(seqs, tokens, heads, kv_heads, max_q, max_kv, seqs * max_kv)
        assert most > 0
        for total in (seqs * max_kv + 1, 1 << 40, 2 ** 63 - 1):
            assert size(seqs, tokens, heads, kv_heads, max_q, max_kv, total) == most


def test_partials_follow_the_tokens(lib):
    """Scratch memory goes by the query rows that there are, a row of 64 outputs and
    an LSE for each and range, not by the longest chunk in every sequence: a prompt
    chunk beside many single tokens took gigabytes."""
    for singles, chunk, heads, kv_heads, max_kv, total in (
            (63, 2048, 12, 12, 8192, 64 * 600), (63, 2048, 12, 12, 8192, 64 * 4000), (127, 2048, 12, 12, 32768, 128 * 600),
            (31, 200, 12, 12, 8192, 32 * 600), (47, 2000, 12, 12, 8192, 50000), (127, 2048, 32, 8, 32768, 1 << 19),
            (255, 2048, 32, 8, 16384, 1 << 19), (0, 1 << 17, 12, 12, 1 << 20, 1 << 20)):
        tokens, ranges = singles + chunk, 65
        need = lib.bd3_paged_attn_workspace_bytes(singles + 1, tokens, heads, kv_heads, chunk, max_kv, total)
        assert need <= min(tokens * heads * ranges * 260, (256 << 20) + 256), (singles, chunk, need)
    # and it is what the rows of the ranges take
    need = lib.bd3_paged_attn_workspace_bytes(1, 16, 12, 12, 16, 8192, 8192)
    assert need % (16 * 12 * 260) < 256 and need // (16 * 12 * 260) in range(2, 66)


def test_batches_are_refused_by_what_they_launch(lib):
    """A long chunk beside many short ones: what counts is the tiles that the tokens
    make, not the longest chunk's in every sequence. (An absent q shows that the
    sizes were accepted, before anything could be launched.)"""
    for singles, chunk, heads, kv_heads, max_kv in ((255, 16384, 32, 32, 16384), (511, 8192, 32, 8, 16384),
                                                    (4095, 32768, 64, 8, 1 << 17), (8191, 1024, 16, 2, 1024)):
        for total in (0, max_kv + 100 * singles, (singles + 1) * max_kv):
            kw = dict(seqs=singles + 1, tokens=singles + chunk, heads=heads, kv_heads=kv_heads, max_q=chunk,
                      width=max_kv // 16, max_kv=max_kv, total=total)
            assert attn(lib, **kw, q=None) == _native.BD3_EINVAL
            assert "q must" in _native.last_error(), (singles, chunk, _native.last_error())
    # and products that would wrap are still refused
    big = (1 << 31) - 1
    for kw in (dict(seqs=big, tokens=big, max_q=1), dict(seqs=big, tokens=big, heads=big, kv_heads=big, max_q=1),
               dict(seqs=1 << 20, tokens=1 << 30, max_q=4096), dict(seqs=1 << 24, tokens=1 << 24, heads=64, kv_heads=64),
               dict(seqs=1, tokens=1 << 28, heads=4, kv_heads=2, max_q=1 << 28)):
        assert attn(lib, **kw, q=None) == _native.BD3_EINVAL
        assert "too large" in _native.last_error(), kw
        n = {**dict(seqs=2, tokens=8, heads=4, kv_heads=2, max_q=4), **kw}
        assert lib.bd3_paged_attn_workspace_bytes(n["seqs"], n["tokens"], n["heads"], n["kv_heads"], n["max_q"], 64, 100) == 0


def test_at_most_64_ranges(lib):
    """Of a sequence, as rounded: 16540 keys are 65 ranges of about 256."""
    size = lib.bd3_paged_attn_workspace_bytes
    for max_kv in (16383, 16384, 16511, 16512, 16540, 16639, 16640, 33100, 66200, 1 << 20):
        for total in (max_kv // 10, max_kv):
            assert size(1, 1, 1, 1, 1, max_kv, total) <= 64 * 260 + 256, max_kv


def test_repetitions_without_a_reciprocal(lib):
    """1 / 1e-39 is infinite in fp32: x / repetition would be, however small x is."""
    st = (ctypes.c_int64 * 8)(300, 100, 300, 100, 5, 0, 0, 0)
    for r in (1e-39, 1e-44, 2.0 ** -127):
        pen = (ctypes.c_float * 3)(r, 0.0, 0.0)
        assert pen[0] > 0
        assert lib.bd3_adjust_logits(None, 0, None, 2, 3, 100, P, 5, None, pen, None, None, None, None, None, -1e6, st,
                                     None) == _native.BD3_EINVAL
        assert "repetition" in _native.last_error()
    pen = (ctypes.c_float * 3)(2.0 ** -126, 0.0, 0.0)
    assert lib.bd3_adjust_logits(None, 0, None, 2, 3, 100, P, 5, None, pen, None, None, None, None, None, -1e6, st,
                                 None) == _native.BD3_EINVAL
    assert "non-NULL" in _native.last_error()
