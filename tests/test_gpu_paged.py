"""GPU parity of the paged attention and its inputs against their definitions in
float64 (oracle/serving.py), over chunk and cache lengths, head layouts, pages,
strides, bad table entries and lengths, streams and graphs."""
from __future__ import annotations

import pytest
import torch

from _serving_util import BF, D, HALF, attention_reference, paged_case, worst
from kernels.BlockSparseDecodeAttention import block_sparse_decode_attention
from kernels.kv_cache import rope_tables
from kernels.paged import PagedKVCache, paged_attention, paged_attention_inputs
from oracle import serving as orc


def on(c, dev):
    return {k: t.to(dev) if torch.is_tensor(t) else t for k, t in c.items()}


def attend(d, bs, **kw):
    kw = {"max_q": d["max_q"], "max_kv": d["max_kv"], "total_kv": d["total"], **kw}
    return paged_attention(d["q"], d["k"], d["v"], d["table"], d["starts"], d["kv"], bs, **kw)


CASES = [
    # (chunk, context) of each sequence, heads, KV heads, page, block
    ([(1, 0)], 1, 1, 16, 1),
    ([(1, 599)], 12, 12, 16, 1),
    ([(1, 1), (1, 31), (1, 32), (1, 33), (1, 2047)], 4, 4, 32, 1),
    ([(16, 3584)], 12, 12, 64, 16),
    ([(16, 0), (16, 5), (16, 1000), (3, 77), (0, 50), (1, 1), (0, 0), (16, 496)], 2, 2, 64, 16),
    ([(4, 64), (4, 1020), (4, 300)], 3, 3, 16, 4),
    ([(5, 13), (5, 250), (2, 7)], 6, 3, 16, 5),
    ([(32, 1504), (32, 0), (32, 31), (17, 300)], 4, 4, 64, 32),
    ([(33, 64), (64, 500), (48, 3)], 2, 2, 128, 16),
    ([(65, 100), (64, 7)], 2, 2, 256, 64),
    ([(130, 70), (1, 300), (257, 0), (64, 64), (128, 128)], 2, 2, 16, 16),
    ([(300, 900), (7, 2000), (129, 1)], 2, 2, 64, 7),
    ([(200, 333), (100, 0)], 2, 2, 32, 1),
    ([(513, 0), (128, 640)], 1, 1, 1024, 32),
    # grouped heads: 3, 8 and 12 query heads to a KV head
    ([(32, 500), (8, 100), (1, 64)], 12, 4, 16, 32),
    ([(1, 700), (2, 30), (16, 256)], 16, 2, 64, 16),
    ([(1, 1000), (1, 5)], 12, 1, 32, 1),
    ([(40, 333), (90, 12)], 12, 1, 64, 8),
    ([(7, 100), (50, 200)], 6, 2, 64, 1 << 30),
]


@pytest.mark.gpu
@pytest.mark.parametrize("cut", ["whole", "many"])
@pytest.mark.parametrize("lens,heads,kv_heads,page,bs", CASES)
def test_attention_matches_definition(cuda, record_error, lens, heads, kv_heads, page, bs, cut):
    print(f"paged attention {lens} {heads}/{kv_heads} page {page} bs {bs} {cut}", flush=True)
    c = paged_case(lens, heads, kv_heads, page, seed=len(lens) + page)
    ref, tol = attention_reference(c, bs)
    # total_kv 0 cuts the keys into as many ranges as the launch allows, a large one into few
    total = 0 if cut == "many" else len(lens) * max(c["max_kv"], 1)
    o = attend(on(c, cuda), bs, total_kv=total)
    assert o.shape == c["q"].shape and o.dtype == BF
    record_error("paged attention / bound", worst(o, ref, tol), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [64, 65, 130])
@pytest.mark.parametrize("chunk,heads,kv_heads", [(1, 2, 1), (16, 2, 2), (32, 1, 1), (70, 1, 1), (25, 6, 1)])
def test_many_sequences(cuda, record_error, seqs, chunk, heads, kv_heads):
    """More sequences than a wave has lanes; some without tokens, some without keys."""
    g = torch.Generator().manual_seed(seqs)
    lens = [(int(n), int(x)) for n, x in zip(torch.randint(0, chunk + 1, (seqs,), generator=g),
                                             torch.randint(0, 400, (seqs,), generator=g))]
    lens[3], lens[seqs - 1] = (0, 0), (chunk, 900)
    c = paged_case(lens, heads, kv_heads, 16, seed=seqs)
    ref, tol = attention_reference(c, 16)
    for total in (0, c["total"], 10 ** 7):
        o = attend(on(c, cuda), 16, total_kv=total, max_q=chunk)
        record_error("paged attention / bound", worst(o, ref, tol), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk,bound", [(16, 5), (32, 20), (64, 33), (300, 130)])
def test_tokens_beyond_max_q_are_left_out(cuda, record_error, chunk, bound):
    """A chunk longer than the bound: its first tokens as ever, the rest as they were."""
    c = paged_case([(chunk, 800), (3, 50)], 2, 2, 16, seed=8)
    ref, tol = attention_reference(c, 16)
    for total in (0, c["total"]):
        out = torch.full_like(c["q"], 7.0).to(cuda)
        attend(on(c, cuda), 16, out=out, max_q=bound, total_kv=total)
        assert (out[bound:chunk] == 7.0).all()
        kept = torch.cat([torch.arange(bound), torch.arange(chunk, chunk + 3)])
        record_error("paged attention / bound", worst(out[kept.to(cuda)], ref[kept], tol[kept]), 1.0)


@pytest.mark.gpu
def test_large_scores(cuda, record_error):
    """Scores of +-100: a row's weight sits on few keys, whichever range holds them."""
    c = paged_case([(16, 700), (1, 2000), (100, 100)], 2, 2, 64, seed=3, q_scale=8.0)
    ref, tol = attention_reference(c, 16)
    for total in (0, 6000):
        record_error("paged attention / bound", worst(attend(on(c, cuda), 16, total_kv=total), ref, tol), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 16, 40, 200])
def test_bounds_looser_than_the_batch(cuda, record_error, chunk):
    """max_q and max_kv above the batch's, defaults, out= with rows behind the last sequence."""
    c = paged_case([(chunk, 300), (1, 40)], 4, 2, 32, seed=chunk, extra_tokens=5)
    ref, tol = attention_reference(c, 16)
    T = int(c["starts"][-1])
    d = on(c, cuda)
    for kw in ({"max_q": 1000}, {"max_kv": None, "total_kv": None}, {"max_kv": 16 * 32, "max_q": chunk + 1}):
        if kw.get("max_kv") and kw["max_kv"] > c["table"].shape[1] * 32:
            kw["max_kv"] = c["table"].shape[1] * 32
        out = torch.full_like(d["q"], 7.0)
        got = attend(d, 16, out=out, **kw)
        assert got.data_ptr() == out.data_ptr()
        assert (out[T:] == 7.0).all(), "rows behind the last sequence were written"
        record_error("paged attention / bound", worst(out[:T], ref[:T], tol[:T]), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 16, 33, 150])
def test_entries_that_are_no_page(cuda, record_error, chunk):
    """Keys of table entries outside the pool are not seen; a sequence without any
    gives 0; nothing non-finite comes in from the pool."""
    c = paged_case([(chunk, 700), (chunk, 20), (chunk, 64)], 2, 2, 16, seed=chunk)
    c["table"][0, 3] = -1
    c["table"][0, 20] = c["k"].shape[0]
    c["table"][0, 21] = 2 ** 31 - 1
    c["table"][1, :] = -2 ** 31
    c["k"][0], c["v"][0] = torch.nan, torch.nan  # whatever page 0 holds does not come in
    c["table"][c["table"] == 0] = -5
    ref, tol = attention_reference(c, 16)
    for total in (0, 10 ** 6):
        o = attend(on(c, cuda), 16, total_kv=total)
        record_error("paged attention / bound", worst(o, ref, tol), 1.0)
        assert (o[chunk:2 * chunk] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 20, 100])
def test_lengths_that_do_not_fit(cuda, record_error, chunk):
    """Fewer keys than tokens: those before position 0 see nothing. Lengths below 0
    and past the bound, starts past the tokens."""
    c = paged_case([(chunk, 100), (chunk, 100), (chunk, 100)], 2, 2, 16, seed=5)
    c["kv"][0] = chunk // 2
    c["kv"][1] = -3
    cut = dict(c, kv=c["kv"].clone())
    c["kv"][2] = 10 ** 6
    cut["kv"][1], cut["kv"][2] = 0, c["max_kv"]
    ref, tol = attention_reference(cut, 4)
    o = attend(on(c, cuda), 4)
    record_error("paged attention / bound", worst(o, ref, tol), 1.0)
    assert (o[chunk:2 * chunk] == 0).all()
    c["starts"][3] = 10 ** 6  # cut to the tokens there are: the same chunk
    assert torch.equal(attend(on(c, cuda), 4), o)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[(1, 300), (1, 64)], [(16, 500), (16, 48)], [(32, 100)], [(200, 100), (70, 5)]])
def test_strides(cuda, lens):
    """Slot-major pools, a layer of a pool, q inside a wider tensor, a table inside a
    wider one, out in another order: the same bits as the plain layout's."""
    c = on(paged_case(lens, 4, 2, 32, seed=1), cuda)
    want = attend(c, 16)
    d = dict(c)
    d["k"] = c["k"].transpose(1, 2).contiguous().transpose(1, 2)
    pool = torch.full((3, *c["v"].shape), torch.nan, device=cuda, dtype=BF)
    pool[1] = c["v"]
    d["v"] = pool[1]
    wide = torch.full((c["q"].shape[0], 9, D), torch.nan, device=cuda, dtype=BF)
    wide[:, 3:7] = c["q"]
    d["q"] = wide[:, 3:7]
    table = torch.full((len(lens), c["table"].shape[1] + 5), 7, device=cuda, dtype=torch.int32)
    table[:, :-5] = c["table"]
    d["table"] = table[:, :-5]
    out = torch.zeros((4, c["q"].shape[0], D), device=cuda, dtype=BF).transpose(0, 1)
    assert torch.equal(attend(d, 16, out=out), want) and torch.equal(out, want)
    # rows that are not 16-byte aligned: q is copied
    odd = torch.empty((c["q"].shape[0], 4, D + 1), device=cuda, dtype=BF)
    odd[..., 1:] = c["q"]
    assert torch.equal(attend(dict(c, q=odd[..., 1:]), 16), want)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 16, 32, 130])
def test_pages_past_32_bit_offsets(cuda, record_error, chunk):
    """Pages whose element offsets pass 2^32, beside the first ones."""
    c = paged_case([(chunk, 200), (chunk, 90)], 2, 2, 64, seed=9, poison=False)
    d = on(c, cuda)
    n, per = c["k"].shape[0], 2 * 64 * D
    far = (1 << 32) // per + 100
    for name in ("k", "v"):
        pool = torch.empty((far, 2, 64, D), device=cuda, dtype=BF)
        pool[:n // 2] = d[name][:n // 2]
        pool[far - (n - n // 2):] = d[name][n // 2:]
        d[name] = pool
    t = d["table"]
    d["table"] = torch.where(t >= n // 2, t + far - n, t)
    ref, tol = attention_reference(c, 16)
    record_error("paged attention / bound", worst(attend(d, 16), ref, tol), 1.0)


@pytest.mark.gpu
def test_matches_rectangular_decode(cuda, record_error):
    """A batch of equal lengths against the decode attention over contiguous caches."""
    B, H, n, kv, page = 4, 12, 16, 560, 16
    c = paged_case([(n, kv - n)] * B, H, H, page, seed=2)
    d = on(c, cuda)
    ids = d["table"][:, :kv // page].long()
    k = d["k"][ids].permute(0, 2, 1, 3, 4).reshape(B, H, kv, D).contiguous()
    v = d["v"][ids].permute(0, 2, 1, 3, 4).reshape(B, H, kv, D).contiguous()
    q = d["q"].view(B, n, H, D).transpose(1, 2).contiguous()
    want = block_sparse_decode_attention(q, k, v, 16).transpose(1, 2).reshape(B * n, H, D)
    _, tol = attention_reference(c, 16)
    record_error("paged vs decode / bound", worst(attend(d, 16), want.double().cpu(), 2 * tol), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [16, 150])
def test_empty_batches(cuda, chunk):
    c = on(paged_case([(0, 40), (0, 0)], 2, 2, 16), cuda)
    out = torch.empty((0, 2, D), device=cuda, dtype=BF)
    assert attend(c, 16).shape == out.shape
    none = paged_attention(torch.empty(chunk, 2, D, device=cuda, dtype=BF), c["k"], c["v"], c["table"][:0],
                           torch.zeros(1, dtype=torch.int32, device=cuda), c["kv"][:0], 16, max_q=chunk)
    assert none.shape == (chunk, 2, D)
    # no keys at all: every token sees none
    d = on(paged_case([(chunk, 0)], 2, 2, 16), cuda)
    d["kv"].zero_()
    assert (attend(d, 16, max_kv=0, total_kv=0) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[(1, 3000), (1, 70)], [(16, 2500), (16, 90)], [(32, 2000), (32, 0)],
                                  [(200, 1500), (130, 0)]])
def test_attention_graph_follows_the_lengths(cuda, lens):
    """Captured once, replayed with other lengths, tables and queries: each replay
    equals the eager call with the same bounds, work between the replays."""
    c = on(paged_case(lens, 2, 2, 16, seed=4), cuda)
    bound = {"max_q": c["max_q"], "max_kv": c["max_kv"], "total_kv": 0}
    out = torch.zeros_like(c["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        attend(c, 16, out=out, **bound)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            attend(c, 16, out=out, **bound)
    torch.cuda.synchronize()
    g = torch.Generator(device=cuda).manual_seed(0)
    for rep in range(4):
        if rep:
            c["kv"].copy_(c["kv"] - 16 * rep * (c["kv"] > 1000).int())
            c["table"].copy_(c["table"].flip(0) if rep == 2 else c["table"])
            if rep == 2:
                c["kv"].copy_(c["kv"].flip(0))
            c["q"].copy_(torch.randn(c["q"].shape, generator=g, device=cuda))
        out.fill_(3.0)
        want = attend(c, 16, **bound)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), rep


@pytest.mark.gpu
def test_other_streams_and_repeats_agree(cuda):
    """Two streams at once and the same call again: equal bits (nothing depends on
    the order in which workgroups finish)."""
    c = on(paged_case([(16, 3000), (16, 100), (3, 900)], 12, 12, 64, seed=6), cuda)
    want = attend(c, 16, total_kv=0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs += [attend(c, 16, total_kv=0) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.gpu
def test_shared_prefix_pages(cuda, record_error):
    """Two sequences whose tables begin with the same pages."""
    c = paged_case([(16, 496), (16, 240)], 2, 2, 16, seed=12)
    c["table"][1, :15] = c["table"][0, :15]
    ref, tol = attention_reference(c, 16)
    record_error("paged attention / bound", worst(attend(on(c, cuda), 16), ref, tol), 1.0)


@pytest.mark.gpu
def test_compile_paged_no_graph_break(cuda):
    """The custom ops under torch.compile: the same bits, one graph, pages written."""
    import kernels.ops  # noqa: F401
    c = on(inputs_case([(16, 100), (5, 30)], 4, 2, 16, seed=1), cuda)
    batch = (c["table"], c["starts"], c["kv"])

    def layer(qkv, k, v):
        q = torch.ops.bd3.paged_qkv_rope(qkv * 2, 4, c["sin"], c["cos"], k, v, *batch)
        return torch.ops.bd3.paged_attn(q, k, v, *batch, 16, 16) + 1

    k1, v1, k2, v2 = c["k"].clone(), c["v"].clone(), c["k"].clone(), c["v"].clone()
    want = layer(c["qkv"], k1, v1)
    got = torch.compile(layer, backend="aot_eager", fullgraph=True, dynamic=True)(c["qkv"], k2, v2)
    assert torch.equal(got, want) and torch.equal(k1, k2) and torch.equal(v1, v2)
    assert not torch.equal(k1, c["k"])


@pytest.mark.gpu
def test_refusals(cuda):
    c = on(paged_case([(4, 20)], 4, 2, 16), cuda)
    ok = dict(q=c["q"], k=c["k"], v=c["v"], table=c["table"], starts=c["starts"], kv=c["kv"])

    def call(**kw):
        d = {**c, **ok, **kw}
        return paged_attention(d["q"], d["k"], d["v"], d["table"], d["starts"], d["kv"], 4, max_q=4,
                               out=kw.get("out"))

    for kw, text in [
            (dict(q=c["q"].float()), "bf16"), (dict(q=c["q"][:, :3]), "multiple"), (dict(k=c["k"].float()), "bf16"),
            (dict(v=c["v"][:-1]), "k_pages and v_pages"), (dict(k=c["k"][..., :32], v=c["v"][..., :32]), "64"),
            (dict(table=c["table"].long()), "int32"), (dict(table=c["table"][:, ::2]), "last stride 1"),
            (dict(starts=c["starts"][:1]), "q_starts"), (dict(kv=c["kv"].repeat(2)), "kv_lens"),
            (dict(kv=c["kv"].cpu()), "one device"), (dict(out=torch.empty(4, 4, 32, device=cuda, dtype=BF)), "out must"),
            (dict(out=torch.empty(4, 4, D, device=cuda)), "out must"),
            (dict(out=torch.empty(4, 1, D, device=cuda, dtype=BF).expand(4, 4, D)), "out must"),
            (dict(k=torch.empty(c["k"].numel() + 1, device=cuda, dtype=BF)[1:].view_as(c["k"])), "16-byte")]:
        with pytest.raises(AssertionError, match=text):
            call(**kw)
    with pytest.raises(AssertionError, match="exceeds"):
        paged_attention(c["q"], c["k"], c["v"], c["table"], c["starts"], c["kv"], 4, max_q=4, max_kv=10 ** 6)
    sin, cos = (t.to(cuda) for t in rope_tables(D, 64))
    qkv = torch.zeros(4, 8 * D, device=cuda, dtype=BF)
    with pytest.raises(AssertionError, match="no element may occur twice"):
        one = c["k"][:1].expand(3, -1, -1, -1)
        paged_attention_inputs(qkv, 4, sin, cos, one, one, c["table"], c["starts"], c["kv"])
    with pytest.raises(AssertionError, match="projection width"):
        paged_attention_inputs(qkv[:, :-D], 4, sin, cos, c["k"], c["v"], c["table"], c["starts"], c["kv"])
    with pytest.raises(AssertionError, match="RoPE tables"):
        paged_attention_inputs(qkv, 4, sin.double(), cos.double(), c["k"], c["v"], c["table"], c["starts"], c["kv"])


# ---------------------------------------------------------------------------
# attention inputs


def inputs_case(lens, heads, kv_heads, page, seed, extra_tokens=0):
    c = paged_case(lens, heads, kv_heads, page, seed=seed, poison=False, extra_tokens=extra_tokens)
    g = torch.Generator().manual_seed(seed + 1)
    c["qkv"] = (torch.randn(c["q"].shape[0], (heads + 2 * kv_heads) * D, generator=g) * 2).to(BF)
    c["sin"], c["cos"] = rope_tables(D, 4096)
    return c


def put(d, heads, **kw):
    return paged_attention_inputs(d["qkv"], heads, d["sin"], d["cos"], d["k"], d["v"], d["table"], d["starts"], d["kv"],
                                  **kw)


def check_inputs(c, d, q, heads, kv_heads):
    """q and k: one rounding to bf16 of an fp32 value off by at most 3 * 2^-24
    (|x1 c| + |x2 s|) <= 2^-22 max |x|; v is copied; other slots as they were."""
    rq, rk, rv = orc.paged_attention_inputs(c["qkv"], heads, c["sin"], c["cos"], c["k"], c["v"], c["table"], c["starts"],
                                            c["kv"])
    small = 2.0 ** -22 * 2 * float(c["qkv"].float().abs().max())
    T = int(c["starts"][-1])
    assert worst(q[:T], rq[:T], 1.001 * HALF * rq[:T].abs() + small) <= 1.0
    kd = d["k"].double().cpu()
    assert ((kd - rk).abs() <= 1.001 * HALF * rk.abs() * (rk != c["k"].double()) + small * (rk != c["k"].double())).all()
    assert torch.equal(d["v"].double().cpu(), rv)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads,kv_heads,page", [
    ([(1, 0)], 1, 1, 16), ([(16, 1000)], 12, 12, 64), ([(1, 5), (0, 7), (1, 64), (1, 2000)], 12, 4, 32),
    ([(32, 16), (5, 100), (0, 0), (64, 0), (17, 130)], 3, 3, 16), ([(300, 700), (1, 15), (200, 0)], 16, 2, 256),
    ([(2, 3)] * 150, 2, 1, 16), ([(3, 4090)], 2, 2, 16)])
def test_inputs_match_definition(cuda, lens, heads, kv_heads, page):
    print(f"paged inputs {lens[:5]} {heads}/{kv_heads} page {page}", flush=True)
    c = inputs_case(lens, heads, kv_heads, page, seed=page + heads, extra_tokens=3)
    d = on(c, cuda)
    out = torch.full_like(d["q"], 7.0)
    q = put(d, heads, out=out)
    assert q.data_ptr() == out.data_ptr()
    assert (out[int(c["starts"][-1]):] == 7.0).all(), "rows behind the last sequence were written"
    check_inputs(c, d, q, heads, kv_heads)


@pytest.mark.gpu
def test_inputs_bad_entries_write_nothing(cuda):
    c = inputs_case([(40, 100), (16, 0), (20, 300)], 4, 2, 16, seed=3)
    c["table"][0, 7] = -1
    c["table"][0, 8] = c["k"].shape[0]
    c["kv"][1] = 5        # 11 tokens before position 0
    c["kv"][2] = 10 ** 6  # past the table
    d = on(c, cuda)
    check_inputs(c, d, put(d, 4), 4, 2)


@pytest.mark.gpu
def test_inputs_strides_and_far_pages(cuda):
    c = on(inputs_case([(40, 100), (16, 0)], 4, 2, 16, seed=3), cuda)
    want_k, want_v = c["k"].clone(), c["v"].clone()
    want = put(dict(c, k=want_k, v=want_v), 4)
    d = dict(c)
    d["k"] = c["k"].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros((c["qkv"].shape[0], c["qkv"].shape[1] + 8), device=cuda, dtype=BF)
    wide[:, 8:] = c["qkv"]
    d["qkv"] = wide[:, 8:]
    n, far = c["v"].shape[0], (1 << 32) // (2 * 16 * D) + 10
    pool = torch.empty((far, 2, 16, D), device=cuda, dtype=BF)
    pool[far - n:] = c["v"]
    d["v"], d["table"] = pool, torch.where(c["table"] >= 0, c["table"] + far - n, -1).int()
    kp = torch.empty((far, 2, 16, D), device=cuda, dtype=BF)
    kp[far - n:] = d["k"]
    q = put(dict(d, k=kp), 4)
    assert torch.equal(q, want) and torch.equal(kp[far - n:], want_k) and torch.equal(pool[far - n:], want_v)


@pytest.mark.gpu
def test_cache_steps_equal_one_pass(cuda, record_error):
    """Prompts of different lengths through the cache in one pass, in chunks and
    in blocks with uncommitted steps between: the same keys, the same attention; a
    sequence that ends gives its pages to a new one."""
    H, KH, page, bs = 4, 2, 16, 8
    g = torch.Generator(device=cuda).manual_seed(1)
    sin, cos = (t.to(cuda) for t in rope_tables(D, 512))
    lens = [40, 96, 8]
    qkv = [torch.randn(n, (H + 2 * KH) * D, generator=g, device=cuda).to(BF) for n in lens]

    def once(parts):
        """attention outputs of each sequence, `parts` tokens at a time"""
        cache = PagedKVCache(2, 40, KH, page, device=cuda)
        cache.free(cache.add())
        seqs = [cache.add() for _ in lens]
        outs = [[] for _ in lens]
        at = [0] * len(lens)
        while any(a < n for a, n in zip(at, lens)):
            live = [i for i in range(len(lens)) if at[i] < lens[i]]
            take = [min(parts, lens[i] - at[i]) for i in live]
            # a step whose tokens are not kept, then the one that is
            for keep in (False, True):
                batch = cache.batch([seqs[i] for i in live], take)
                x = torch.cat([qkv[i][at[i]:at[i] + n] for i, n in zip(live, take)])
                if not keep:
                    x = x * 2
                for layer in (0, 1):
                    q = batch.attention_inputs(x, H, sin, cos, layer)
                    o = batch.attention(q, layer, bs)
            batch.commit()
            for i, piece in zip(live, o.split(take)):
                outs[i].append(piece)
            for i, n in zip(live, take):
                at[i] += n
        assert [cache.length(s) for s in seqs] == lens
        free = cache.free_pages
        cache.free(seqs[1])
        assert cache.free_pages == free + lens[1] // page
        return [torch.cat(o) for o in outs]

    whole, chunks, blocks = once(10 ** 6), once(24), once(bs)
    for a, b, c in zip(whole, chunks, blocks):
        # each within HALF (|o| + sum p |v|), |v| < 6, of the same value
        record_error("chunks vs whole", float((a - b).abs().max()), 2 * HALF * 12)
        record_error("blocks vs whole", float((a - c).abs().max()), 2 * HALF * 12)


@pytest.mark.gpu
def test_overlapping_tensors_are_refused(cuda):
    """What a workgroup writes while another still reads it has no defined result.
    Apart, the halves of one buffer are fine, and so are interleaved k and v pools."""
    c = on(paged_case([(4, 20)], 4, 2, 16), cuda)
    batch = (c["table"], c["starts"], c["kv"])
    flat = torch.zeros(2 * c["q"].numel(), device=cuda, dtype=BF)
    n = c["q"].numel()
    q = flat[:n].view_as(c["q"]).copy_(c["q"])
    want = paged_attention(c["q"], c["k"], c["v"], *batch, 4, max_q=4)
    for out in (q, flat[64:n + 64].view_as(q), c["k"].view(-1)[:n].view_as(q), c["v"].view(-1)[:n].view_as(q)):
        with pytest.raises(AssertionError, match="overlap"):
            paged_attention(q, c["k"], c["v"], *batch, 4, max_q=4, out=out)
    assert torch.equal(paged_attention(q, c["k"], c["v"], *batch, 4, max_q=4, out=flat[n:].view_as(q)), want)

    sin, cos = (t.to(cuda) for t in rope_tables(D, 64))
    buf = torch.ones(4 * 8 * D, device=cuda, dtype=BF)
    qkv = buf.view(4, 8 * D)

    def inputs(k, v, out=None):
        return paged_attention_inputs(qkv, 4, sin, cos, k, v, *batch, out=out)

    pool = torch.zeros(c["k"].numel() + 64, device=cuda, dtype=BF)
    k = pool[:-64].view_as(c["k"])
    for kw in (dict(k=k, v=k), dict(k=k, v=pool[64:].view_as(k)), dict(k=k, v=c["v"], out=buf[:n].view_as(q)),
               dict(k=k, v=c["v"], out=k.view(-1)[:n].view_as(q))):
        with pytest.raises(AssertionError, match="overlap"):
            inputs(**kw)
    both = torch.zeros(2, *c["k"].shape, device=cuda, dtype=BF)
    woven = torch.zeros(c["k"].shape[0], 2, *c["k"].shape[1:], device=cuda, dtype=BF)
    a, b = inputs(both[0], both[1]), inputs(woven[:, 0], woven[:, 1])
    assert torch.equal(a, b) and torch.equal(both, woven.transpose(0, 1)) and both.abs().sum() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("chunk,heads,kv_heads", [(1, 2, 2), (16, 4, 2), (50, 160, 40), (200, 2, 2)])
def test_any_total_is_a_hint(cuda, record_error, chunk, heads, kv_heads):
    """total_kv up to the largest integer: the launch it shapes stays that of the
    batch (2^63 - 1 wrapped the number of workgroups)."""
    c = paged_case([(chunk, 900), (1, 30)], heads, kv_heads, 16, seed=chunk)
    ref, tol = attention_reference(c, 16)
    d = on(c, cuda)
    for total in (2 * c["max_kv"], 1 << 40, 2 ** 63 - 1):
        record_error("paged attention / bound", worst(attend(d, 16, total_kv=total), ref, tol), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("singles,chunk,ctx,heads,kv_heads", [
    (90, 300, 900, 2, 2), (63, 700, 100, 4, 1), (70, 40, 1500, 2, 2), (130, 12, 1200, 6, 3), (5, 33, 3000, 2, 1)])
def test_a_chunk_beside_single_tokens(cuda, record_error, singles, chunk, ctx, heads, kv_heads):
    """A prompt chunk in the middle of sequences of one token, some without any: the
    keys of both in ranges, whose partials lie packed, rows of several sequences to a
    workgroup of the merge."""
    from kernels import _native
    g = torch.Generator().manual_seed(singles)
    lens = [(int(n), int(x)) for n, x in zip((torch.rand(singles, generator=g) < 0.8).int(),
                                             torch.randint(0, 1700, (singles,), generator=g))]
    lens.insert(singles // 2, (chunk, ctx))
    c = paged_case(lens, heads, kv_heads, 16, seed=singles, extra_tokens=4)
    T = int(c["starts"][-1])
    ref, tol = attention_reference(c, 16)
    d = on(c, cuda)
    cut = 0
    for total in (0, c["total"], 10 ** 7):
        out = torch.full_like(d["q"], 7.0)
        attend(d, 16, total_kv=total, out=out)
        record_error("paged attention / bound", worst(out[:T], ref[:T], tol[:T]), 1.0)
        assert (out[T:] == 7.0).all(), "rows behind the last sequence were written"
        cut += _native.lib().bd3_paged_attn_workspace_bytes(len(lens), T + 4, heads, kv_heads, c["max_q"], c["max_kv"],
                                                            total) > 0
    assert cut, "no call cut its keys"


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 16, 40, 200])
def test_partials_of_starts_that_do_not_ascend(cuda, chunk):
    """Starts that run backwards are no batch; the rows of sequences that still own
    tokens of their own come out as ever, and nothing else is touched."""
    c = paged_case([(chunk, 1500), (chunk, 900), (chunk, 1200)], 2, 2, 16, seed=chunk)
    d = on(c, cuda)
    want = attend(d, 16, total_kv=0)
    d["starts"] = torch.tensor([0, chunk, chunk - 1, -5], dtype=torch.int32, device=cuda)
    out = torch.full_like(d["q"], 7.0)
    attend(d, 16, total_kv=0, out=out)
    assert torch.equal(out[:chunk], want[:chunk])
    assert (out[chunk:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,chunk", [(16, 2, 1024), (4, 2, 100), (4, 2, 3)])
def test_thousands_of_sequences(cuda, record_error, heads, kv_heads, chunk):
    """One chunk among 8192 sequences, most without tokens in this step: the launch
    goes by the tokens."""
    g = torch.Generator().manual_seed(1)
    lens = [(int(n), int(x)) for n, x in zip((torch.rand(8191, generator=g) < 0.05).int(),
                                             torch.randint(0, 40, (8191,), generator=g))]
    lens.insert(5000, (chunk, 700))
    c = paged_case(lens, heads, kv_heads, 64, seed=1)
    ref, tol = attention_reference(c, 16)
    for total in (0, c["total"]):
        record_error("paged attention / bound", worst(attend(on(c, cuda), 16, total_kv=total), ref, tol), 1.0)


@pytest.mark.gpu
def test_results_over_the_batch_s_arrays_are_refused(cuda):
    """The table, starts and lengths, and RoPE tables, that a launch reads while it
    writes its result or the pages."""
    c = on(paged_case([(4, 20), (3, 2)], 4, 2, 16), cuda)
    n = c["q"].numel()
    buf = torch.zeros(n, device=cuda, dtype=BF)
    out = buf.view_as(c["q"])
    ints = buf.view(torch.int32)
    same = dict(table=c["table"], starts=c["starts"], kv=c["kv"])

    def inside(t):
        return ints[8:8 + t.numel()].view_as(t).copy_(t)

    sin, cos = (t.to(cuda) for t in rope_tables(D, 64))
    qkv = torch.zeros(c["q"].shape[0], 8 * D, device=cuda, dtype=BF)
    pool = torch.zeros(c["k"].numel(), device=cuda, dtype=BF).view_as(c["k"])
    for name in same:
        kw = {**same, name: inside(same[name])}
        batch = (kw["table"], kw["starts"], kw["kv"])
        with pytest.raises(AssertionError, match="overlap"):
            paged_attention(c["q"], c["k"], c["v"], *batch, 4, max_q=4, out=out)
        with pytest.raises(AssertionError, match="overlap"):
            paged_attention_inputs(qkv, 4, sin, cos, c["k"], c["v"], *batch, out=out)
        pool_ints = pool.view(-1).view(torch.int32)
        kw[name] = pool_ints[:same[name].numel()].view_as(same[name]).copy_(same[name])
        for k, v in ((pool, c["v"]), (c["k"], pool)):
            with pytest.raises(AssertionError, match="overlap"):
                paged_attention_inputs(qkv, 4, sin, cos, k, v, kw["table"], kw["starts"], kw["kv"])
    wide = torch.zeros(4 * c["k"].numel(), device=cuda, dtype=BF)
    pages = wide[:c["k"].numel()].view_as(c["k"])
    rope = wide.view(torch.float32)[:32].view(1, 32)
    for a, b in ((rope, cos[:1]), (sin[:1], rope)):
        with pytest.raises(AssertionError, match="overlap"):
            paged_attention_inputs(qkv, 4, a, b, pages, c["v"], *same.values())
    batch = tuple(same.values())
    assert torch.equal(paged_attention(c["q"], c["k"], c["v"], *batch, 4, max_q=4, out=out),
                       paged_attention(c["q"], c["k"], c["v"], *batch, 4, max_q=4))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2])
def test_rows_off_the_grid_are_copied(cuda, n):
    """Tokens of a wider tensor whose rows are not multiples of 16 bytes, one of them
    too (torch calls that one contiguous), and bases off the grid."""
    c = on(inputs_case([(n, 100)], 4, 2, 16, seed=1), cuda)
    want = attend(c, 16)
    wide = torch.zeros((n, c["q"].numel() // n + 3), device=cuda, dtype=BF)
    wide[:, :-3] = c["q"].view(n, -1)
    flat = torch.zeros(c["q"].numel() + 1, device=cuda, dtype=BF)
    flat[1:] = c["q"].view(-1)
    for q in (wide[:, :-3].view(n, 4, D), flat[1:].view(n, 4, D)):
        assert torch.equal(attend(dict(c, q=q), 16), want)
    k1, v1 = c["k"].clone(), c["v"].clone()
    rotated = put(dict(c, k=k1, v=v1), 4)
    wide = torch.zeros((n, 8 * D + 5), device=cuda, dtype=BF)
    wide[:, :-5] = c["qkv"]
    flat = torch.zeros(c["qkv"].numel() + 3, device=cuda, dtype=BF)
    flat[3:] = c["qkv"].view(-1)
    for qkv in (wide[:, :-5], flat[3:].view(n, -1)):
        k2, v2 = c["k"].clone(), c["v"].clone()
        assert torch.equal(put(dict(c, qkv=qkv, k=k2, v=v2), 4), rotated)
        assert torch.equal(k1, k2) and torch.equal(v1, v2)


@pytest.mark.gpu
@pytest.mark.parametrize("first,heads,kv_heads", [([1, 1, 16, 0, 1], 4, 4), ([30, 1, 1, 40, 2], 4, 2),
                                                  ([1, 300, 1, 7, 130], 2, 2)])
def test_attention_graph_follows_the_starts(cuda, first, heads, kv_heads):
    """Two captures in one memory pool, replayed in turn with tokens moved between the
    sequences, eager calls between: the merge finds each row's sequence on the device."""
    T, bound = sum(first), max(first)
    kv = [1500, 700, 2100, 40, 900]
    c = on(paged_case([(n, x - n if x > n else 0) for n, x in zip(first, kv)], heads, kv_heads, 16, seed=3, poison=False), cuda)
    kw = {"max_q": bound, "max_kv": c["max_kv"], "total_kv": 0}
    side, pool = torch.cuda.Stream(), torch.cuda.graph_pool_handle()
    outs = [torch.zeros_like(c["q"]) for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(c, 16, **kw)
        torch.cuda.synchronize()
        for graph, out in zip(graphs, outs):
            with torch.cuda.graph(graph, stream=side, pool=pool):
                attend(c, 16, out=out, **kw)
    torch.cuda.synchronize()
    for order in ([0, 1, 2, 3, 4], [4, 3, 2, 1, 0], [1, 4, 0, 2, 3], [2, 0, 3, 4, 1]):
        n = [first[i] for i in order]
        c["starts"].copy_(torch.tensor([sum(n[:b]) for b in range(6)], dtype=torch.int32))
        assert int(c["starts"][-1]) == T
        host = {k: t.cpu() if torch.is_tensor(t) else t for k, t in c.items()}
        ref, tol = attention_reference(host, 16)
        eager = attend(c, 16, **kw)
        for graph, out in zip(graphs, outs):
            out.fill_(5.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager), order
        assert worst(eager, ref, tol) <= 1.0
