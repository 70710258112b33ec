"""GPU parity of adjust_logits with its definition in float64 (oracle/serving.py),
and of the draw from adjusted logits."""
from __future__ import annotations

import pytest
import torch

from kernels.sampling import PhiloxStream, adjust_logits, subs_sample_step
from oracle import serving as orc

BF = torch.bfloat16


def case(B, R, V, dtype, history, penalties, bias, allowed, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, R, V, generator=g) * 3).to(dtype)
    kw = {}
    if history is not None:
        kw["tokens"] = (torch.rand(B, history, generator=g) ** 3 * V * 1.1 - 0.05 * V).long()  # some outside
        kw["lengths"] = torch.randint(0, history + 1, (B,), generator=g).to(torch.int32)
    if penalties == "scalar":
        kw.update(repetition=1.3, frequency=0.2, presence=-0.4)
    elif penalties == "each":
        kw.update(repetition=0.5 + torch.rand(B, generator=g), frequency=torch.rand(B, generator=g),
                  presence=torch.rand(B, generator=g) - 0.5)
    if bias:
        kw["bias"] = torch.randn(*((V,) if bias == 1 else (B, V)), generator=g)
    if allowed:
        words = -(-V // 32)
        kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, ((words,), (B, words), (B, R, words))[allowed - 1],
                                      generator=g).to(torch.int32)
    return x, kw


def bound(x, kw, ref):
    """One rounding to the logits' type plus at most eight fp32 roundings (2^-24 each)
    of the terms' magnitudes."""
    def top(v, neutral):
        return float(v.abs().max()) if torch.is_tensor(v) else abs(kw.get(v, neutral)) if isinstance(v, str) else abs(v)

    rep = kw.get("repetition", 1.0)
    low = float(rep.min()) if torch.is_tensor(rep) else rep
    size = float(x.float().abs().max()) * max(top(rep, 1), 1 / low)
    if "tokens" in kw:
        size += top(kw.get("frequency", 0.0), 0) * kw["tokens"].shape[1] + top(kw.get("presence", 0.0), 0)
    if "bias" in kw:
        size += float(kw["bias"].abs().max())
    u = torch.finfo(x.dtype).eps / 2
    return 1.001 * u * ref.abs() + 2.0 ** -21 * size


def dev(kw, d):
    return {k: v.to(d) if torch.is_tensor(v) else v for k, v in kw.items()}


def check(got, x, kw):
    ref = orc.adjust_logits(x, **kw)
    assert got.shape == x.shape and got.dtype == x.dtype
    err = (got.double().cpu() - ref).abs()
    assert (err <= bound(x, kw, ref)).all(), float((err / bound(x, kw, ref)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("B,R,V,history,penalties,bias,allowed", [
    (1, 1, 1, 3, "scalar", 1, 1), (1, 1, 7, 20, "each", 2, 3), (2, 3, 33, 5, "scalar", 0, 2),
    (3, 4, 2048, 100, "each", 1, 3), (2, 2, 2049, 1, "scalar", 2, 1), (1, 16, 5001, 700, "each", 0, 0),
    (4, 1, 4099, 64, "scalar", 0, 3), (2, 5, 10000, 3000, "each", 2, 2), (3, 2, 777, None, None, 2, 3),
    (2, 7, 2055, None, None, 0, 2), (2, 2, 500, 0, "scalar", 1, 0), (1, 2, 64, None, None, 0, 0),
    (1, 2, 50258, 2000, "scalar", 1, 1)])
def test_matches_definition(cuda, dtype, B, R, V, history, penalties, bias, allowed):
    print(f"adjust_logits {B} {R} {V} {dtype} {history} {penalties} {bias} {allowed}", flush=True)
    x, kw = case(B, R, V, dtype, history, penalties, bias, allowed, seed=V)
    xd = x.to(cuda)
    got = adjust_logits(xd, **dev(kw, cuda))
    check(got, x, kw)
    assert torch.equal(xd.cpu(), x), "the logits were changed"
    again = xd.clone()
    assert adjust_logits(again, **dev(kw, cuda), out=again).data_ptr() == again.data_ptr()
    assert torch.equal(again, got), "in place"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_strides_and_two_dims(cuda, dtype):
    """A slice of wider logits, rows that start at any element, broadcast and
    transposed arguments, (batch, vocab) logits, neighbours left alone."""
    x, kw = case(3, 4, 1001, dtype, 50, "each", 2, 2, seed=1)
    d = dev(kw, cuda)
    want = adjust_logits(x.to(cuda), **d)
    wide = torch.full((3, 6, 1013), 5.0, device=cuda, dtype=dtype)
    wide[:, 1:5, 3:1004] = x.to(cuda)
    view = wide[:, 1:5, 3:1004]
    assert torch.equal(adjust_logits(view, **d), want)
    out = torch.full((3, 6, 1013), 5.0, device=cuda, dtype=dtype)
    adjust_logits(view, **d, out=out[:, 1:5, 3:1004])
    assert torch.equal(out[:, 1:5, 3:1004], want)
    out[:, 1:5, 3:1004] = 5.0
    assert (out == 5.0).all(), "neighbours were written"
    d["bias"] = d["bias"].t().contiguous().t()
    d["allowed"] = d["allowed"][:, None].expand(-1, 4, -1)
    d["tokens"] = torch.cat([d["tokens"], d["tokens"]], dim=1)[:, :50]
    assert torch.equal(adjust_logits(x.to(cuda).transpose(1, 2).contiguous().transpose(1, 2), **d), want)
    flat, kf = case(5, 1, 300, dtype, 9, "scalar", 1, 2, seed=2)
    two = adjust_logits(flat[:, 0].to(cuda), **dev(kf, cuda))
    assert two.shape == (5, 300)
    check(two[:, None], flat, kf)
    again = flat[:, 0].to(cuda)
    assert adjust_logits(again, **dev(kf, cuda), out=again).shape == (5, 300)
    assert torch.equal(again, two)


@pytest.mark.gpu
def test_masked_values_do_not_matter(cuda):
    """nan and infinities where the mask forbids, the type's lowest value among the
    logits; a row that allows nothing is `fill` everywhere."""
    for dtype in (BF, torch.float32):
        x, kw = case(2, 3, 300, dtype, 40, "scalar", 1, 3, seed=4)
        kw["allowed"][1, 2] = 0
        v = torch.arange(300)
        yes = ((kw["allowed"][..., v // 32] >> (v % 32)) & 1).bool()
        clean = adjust_logits(x.to(cuda), **dev(kw, cuda))
        dirty = x.clone()
        dirty[~yes] = torch.tensor([torch.nan, torch.inf, -torch.inf]).to(dtype).repeat(int((~yes).sum()))[:int((~yes).sum())]
        assert torch.equal(adjust_logits(dirty.to(cuda), **dev(kw, cuda)), clean)
        assert (clean[1, 2] == torch.tensor(-1e6).to(dtype).item()).all()
        low = torch.full((1, 1, 40), torch.finfo(dtype).min, dtype=dtype)
        low[0, 0, 3] = 1.0
        got = adjust_logits(low.to(cuda), bias=torch.zeros(40, device=cuda), fill=-50.0)
        assert torch.equal(got.cpu(), low)


@pytest.mark.gpu
def test_zero_sizes(cuda):
    x = torch.empty((0, 4, 100), device=cuda)
    assert adjust_logits(x, bias=torch.zeros(100, device=cuda)).shape == (0, 4, 100)
    assert adjust_logits(torch.empty((3, 0, 100), device=cuda)).shape == (3, 0, 100)
    y = torch.randn(2, 2, 100, device=cuda)
    assert torch.equal(adjust_logits(y), y)
    none = torch.zeros(2, 5, dtype=torch.long, device=cuda)
    for n in (0, -7):
        got = adjust_logits(y, none, torch.full((2,), n, dtype=torch.int32, device=cuda), repetition=2.0, presence=1.0)
        assert torch.equal(got, y)
    over = adjust_logits(y, none, torch.full((2,), 99, dtype=torch.int32, device=cuda), presence=1.0)
    assert torch.equal(over, adjust_logits(y, none, presence=1.0))


@pytest.mark.gpu
def test_graph_and_draw(cuda):
    """Adjusted logits and the draw from them, captured and replayed with a longer
    history each time: no token that the grammar forbids is drawn."""
    B, R, V, MASK = 3, 8, 5000, 4999
    x, kw = case(B, R, V, BF, 64, "each", 1, 2, seed=7)
    kw["allowed"][:, 10:] = 0  # tokens 0 .. 319 at most
    d, xd = dev(kw, cuda), x.to(cuda)
    out = torch.empty_like(xd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        adjust_logits(xd, **d, out=out)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            adjust_logits(xd, **d, out=out)
    torch.cuda.synchronize()
    block = torch.full((B, R), MASK, device=cuda)
    v = torch.arange(V)
    yes = ((kw["allowed"][:, v // 32] >> (v % 32)) & 1).bool()
    for rep in range(4):
        d["lengths"].fill_(16 * rep)
        out.fill_(9.0)
        want = adjust_logits(xd, **d)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        drawn = subs_sample_step(out, block, MASK, 0.0, generator=PhiloxStream(rep)).cpu()
        assert all(yes[b, t] for b in range(B) for t in drawn[b].tolist())


@pytest.mark.gpu
def test_refusals(cuda):
    x = torch.zeros(2, 3, 100, device=cuda)
    t = torch.zeros(2, 5, dtype=torch.long, device=cuda)
    for args, kw, text in [
            ((x.half(),), {}, "bf16 or fp32"), ((x[0, 0],), {}, "batch, rows, vocab"), ((x, t.int()), {}, "int64"),
            ((x, t[:1]), {}, "tokens must"), ((x, None, torch.zeros(2, dtype=torch.int32, device=cuda)), {}, "with tokens"),
            ((x, t, torch.zeros(2, dtype=torch.long, device=cuda)), {}, "int32"), ((x, t), {"repetition": 0.0}, "repetition"),
            ((x, t), {"frequency": torch.zeros(3, device=cuda)}, "penalty"), ((x,), {"bias": torch.zeros(99, device=cuda)}, "bias"),
            ((x,), {"bias": torch.zeros(2, 100, device=cuda, dtype=BF)}, "float32"),
            ((x,), {"allowed": torch.zeros(2, 3, dtype=torch.int32, device=cuda)}, "allowed"),
            ((x,), {"allowed": torch.zeros(2, 4, dtype=torch.long, device=cuda)}, "allowed"), ((x,), {"fill": float("-inf")}, "fill"),
            ((x.to(BF),), {"fill": -3.4e38}, "fill"), ((x,), {"out": torch.zeros(2, 3, 100, device=cuda, dtype=BF)}, "out must"),
            ((x,), {"out": torch.zeros(1, 3, 100, device=cuda).expand(2, 3, 100)}, "out must"),
            ((x, t.cpu()), {}, "one device"),
            ((x[:, 0],), {"allowed": torch.zeros(2, 1, 4, dtype=torch.int32, device=cuda)}, "allowed")]:
        with pytest.raises(AssertionError, match=text):
            adjust_logits(*args, **kw)


@pytest.mark.gpu
def test_other_streams_agree(cuda):
    x, kw = case(4, 9, 5001, BF, 300, "each", 2, 3, seed=9)
    xd, d = x.to(cuda), dev(kw, cuda)
    want = adjust_logits(xd, **d)
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            outs += [adjust_logits(xd, **d) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.gpu
def test_overlapping_out_is_refused(cuda):
    """In place is fine, any other overlap has no defined result."""
    flat = torch.randn(2 * 3 * 100 + 100, device=cuda)
    x = flat[:600].view(2, 3, 100)
    for out in (flat[100:].view(2, 3, 100), flat[:600].view(3, 2, 100).transpose(0, 1)):
        with pytest.raises(AssertionError, match="overlap"):
            adjust_logits(x, bias=torch.ones(100, device=cuda), out=out)
    want = x + 1
    assert torch.equal(adjust_logits(x, bias=torch.ones(100, device=cuda), out=x), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("V", [40, 2051])
def test_finite_logits_stay_finite(cuda, dtype, V):
    """The type's lowest and highest values, as a caller bans or forces a token, under
    penalties and biases that take them past its range: the value itself, not an
    infinite one, so the draw that follows sees finite logits only. Infinite and nan
    logits and biases go through."""
    top, inf = torch.finfo(dtype).max, float("inf")
    x = torch.zeros(3, 2, V, dtype=dtype)
    x[:, :, 0::4], x[:, :, 1::4], x[:, :, 2::4] = -top, top, 1.5
    tokens = torch.arange(V)[None].repeat(3, 1)
    rep, freq = torch.tensor([1.3, 0.5, 1.0]), torch.tensor([0.5, 0.0, 1e38])
    bias = torch.zeros(3, V)
    bias[0, 0::4], bias[1, 1::4], bias[2, 0::8] = -3e38, 3e38, -3e38
    kw = dict(repetition=rep, frequency=freq, presence=0.1, bias=bias)
    ref = orc.adjust_logits(x, tokens, None, **kw)
    assert torch.isfinite(ref).all() and ref.abs().max() == top
    got = adjust_logits(x.to(cuda), tokens.to(cuda), **dev(kw, cuda)).cpu()
    assert torch.isfinite(got).all()
    # one rounding to the dtype and at most four fp32 ones of terms of the size of the result or of 3.4e38
    tol = 1.001 * (torch.finfo(dtype).eps / 2 * ref.abs() + 4 * 2.0 ** -24 * 3.5e38 * (ref.abs() > 1e30)) + 1e-6
    assert ((got.double() - ref).abs() <= tol).all()
    assert (got[0, :, 0::4] == -top).all() and (got[1, :, 1::4] == top).all()

    wild = x.clone()
    wild[0, 0, 2], wild[0, 0, 6], wild[0, 1, 2] = -inf, inf, torch.nan
    bias[1, 2] = -inf
    out = adjust_logits(wild.to(cuda), tokens.to(cuda), **dev(kw, cuda)).cpu()
    assert out[0, 0, 2] == -inf and out[0, 0, 6] == inf and torch.isnan(out[0, 1, 2]) and (out[1, :, 2] == -inf).all()
    keep = torch.ones_like(wild, dtype=torch.bool)
    keep[0, 0, 2] = keep[0, 0, 6] = keep[0, 1, 2] = False
    keep[1, :, 2] = False
    assert torch.equal(out[keep], got[keep])


@pytest.mark.gpu
def test_out_over_another_input_is_refused(cuda):
    """Every argument that the launch reads beside the logits: a bias inside the result,
    a result over the mask, the history, the lengths or a penalty."""
    B, R, V = 2, 3, 96
    x = torch.randn(B, R, V, device=cuda)
    buf = torch.zeros(B * R * V + 64, device=cuda)
    out = buf[:B * R * V].view(B, R, V)

    def inside(dtype, n):  # n numbers of dtype within out's memory
        return buf[128:].view(dtype)[:n]

    tokens = torch.zeros(B, 4, dtype=torch.long, device=cuda)
    for kw in (dict(bias=inside(torch.float32, V)), dict(allowed=inside(torch.int32, 3)),
               dict(tokens=inside(torch.long, B * 4).view(B, 4)), dict(tokens=tokens, lengths=inside(torch.int32, B)),
               dict(tokens=tokens, repetition=inside(torch.float32, B)), dict(tokens=tokens, frequency=inside(torch.float32, B)),
               dict(tokens=tokens, presence=buf[:B])):
        with pytest.raises(AssertionError, match="overlap"):
            adjust_logits(x, **kw, out=out)
    bias = buf[B * R * V - V + 64:]  # ends behind the result, begins in it
    with pytest.raises(AssertionError, match="overlap"):
        adjust_logits(x, bias=bias, out=out)
    assert (buf == 0).all()
    # apart in the same memory, and empty ones
    far = torch.zeros(B * R * V + V, device=cuda)
    far[B * R * V:] = 1.0
    assert torch.equal(adjust_logits(x, bias=far[B * R * V:], out=far[:B * R * V].view(B, R, V)), x + 1)
    assert torch.equal(adjust_logits(x, tokens[:, :0], bias=far[B * R * V:], out=out), x + 1)
    none = adjust_logits(x[:0], tokens[:0], bias=far[B * R * V:], out=torch.empty(0, R, V, device=cuda))
    assert none.shape == (0, R, V)


@pytest.mark.gpu
def test_in_place_whatever_a_single_row_s_stride_is(cuda):
    """One sequence's last logits: a view of them by another way is the same memory,
    although torch gives the dimension of one another stride."""
    for batch, rows in ((1, 1), (1, 3), (3, 1)):
        big = torch.randn(batch, rows + 2, 100, device=cuda)[:, 2:].contiguous()
        x = big.as_strided((batch, rows, 100), (rows * 100 if batch > 1 else 7, 100 if rows > 1 else 3, 1))
        want = big + 1
        assert adjust_logits(x, bias=torch.ones(100, device=cuda), out=big) is not None
        assert torch.equal(big, want)
        adjust_logits(big, bias=torch.ones(100, device=cuda), out=x)
        assert torch.equal(big, want + 1)
    x = torch.randn(1, 5, 100, device=cuda)
    last, same = x[:, -1], x[0, -1:]
    want = last + 1
    adjust_logits(last, bias=torch.ones(100, device=cuda), out=same)
    assert torch.equal(x[:, -1], want)
