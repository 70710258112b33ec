"""The int8 codes of 8-bit pages to the last one: round(x / scale), the quotient in fp32, ties to even."""
from __future__ import annotations

import pytest
import torch

from _pool_util import BF, D, I8
from kernels.paged import paged_attention_inputs8


def halves(tokens, heads, seed):
    """Values of which every fourth is exactly half of its block's largest, on either side of 0 (63.5 steps, whatever the
    scale: the fp32 quotient decides); the largest ones fall on the first token of each 16."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, heads, D), generator=g).to(BF)
    x[0::16, :, 3] = (torch.rand((-(-tokens // 16), heads), generator=g) * 4 + 6).to(BF)
    top = x[0::16, :, 3].repeat_interleave(16, dim=0)[:tokens]
    sign = torch.where(torch.rand((tokens, heads, D // 4), generator=g) < 0.5, -0.5, 0.5)
    x[:, :, 1::4] = (top[..., None].float() * sign).to(BF)
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("context", [0, 5])
def test_int8_codes_are_the_rounded_quotients(cuda, context):
    """Keys, under tables that turn nothing (sin 0, cos 1), and values are bf16 numbers, so scale and quotient are one fp32
    division each: there is nothing to be off by. After a context of 5 the first block keeps its scale or doubles it."""
    heads, n = 3, 400
    tables = torch.zeros((512, D // 2), device=cuda), torch.ones((512, D // 2), device=cuda)
    k, v = (torch.zeros((1, heads, 512, D), dtype=I8, device=cuda) for _ in range(2))
    ks, vs = (torch.zeros((1, heads, 32), device=cuda) for _ in range(2))
    table = torch.zeros((1, 1), dtype=torch.int32, device=cuda)
    x = torch.cat([halves(n, heads, s) for s in (1, 2, 3)], dim=1)  # (tokens, q | k | v heads, 64)
    x[:context] *= 0.25  # so that the first block's scale grows when the others come
    for lo, hi in ((0, context), (context, n)):
        if hi > lo:
            paged_attention_inputs8(x[lo:hi].reshape(hi - lo, -1).to(cuda), heads, *tables, k, v, ks, vs, table,
                                    torch.tensor([0, hi - lo], dtype=torch.int32, device=cuda),
                                    torch.tensor([hi], dtype=torch.int32, device=cuda))
    ties = 0
    for new, codes, scales in ((x[:, heads:2 * heads], k, ks), (x[:, 2 * heads:], v, vs)):
        new = new.float().transpose(0, 1)  # (heads, tokens, 64)
        scale = scales[0].cpu().repeat_interleave(16, dim=1)[:, :n, None]
        blocks = torch.nn.functional.pad(new, (0, 0, 0, -n % 16)).unflatten(1, (-1, 16))
        need = blocks.abs().amax(dim=(2, 3)) / 127
        assert torch.equal(scales[0, :, (context > 0):-(-n // 16)].cpu(), need[:, (context > 0):])
        quotient = new / scale
        ties += int(((quotient.abs() % 1) == 0.5).sum())
        want = torch.round(quotient).to(I8)
        assert int((codes[0, :, context:n].cpu() != want[:, context:]).sum()) == 0
    assert ties > 1000


@pytest.mark.gpu
def test_infinite_values_count_as_the_largest_finite_ones(cuda):
    """Not an error of the caller's that should spread: the block's other codes stay codes."""
    tables = torch.zeros((16, D // 2), device=cuda), torch.ones((16, D // 2), device=cuda)
    k, v = (torch.zeros((1, 1, 16, D), dtype=I8, device=cuda) for _ in range(2))
    ks, vs = (torch.zeros((1, 1, 1), device=cuda) for _ in range(2))
    x = torch.zeros((16, 3, D), dtype=BF)
    x[2, 1:, 7], x[3, 1:, 8], x[4, 1:, 9] = float("inf"), float("-inf"), 1e38
    paged_attention_inputs8(x.view(16, -1).to(cuda), 1, *tables, k, v, ks, vs, torch.zeros((1, 1), dtype=torch.int32, device=cuda),
                            torch.tensor([0, 16], dtype=torch.int32, device=cuda), torch.tensor([16], dtype=torch.int32, device=cuda))
    scale = torch.finfo(torch.float32).max / 127
    want = torch.zeros((16, D))
    want[2, 7], want[3, 8], want[4, 9] = 127, -127, round(1e38 / scale)
    # keys are multiplied by the tables' zeros too: an infinite one leaves nan in its pair, which no rule covers
    assert float(vs[0, 0, 0]) == pytest.approx(scale, rel=1e-6) and torch.equal(v[0, 0].cpu().float(), want)
