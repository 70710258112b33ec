"""The ragged serving step run as a program runs it (perf/e2e_sampling.serve):
prompts of different lengths, paged cache, adjusted logits and the draw, with
sequences that wait, join and leave."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.gpu
def test_serving_matches_eager_backbone(cuda):
    from kernels.kv_cache import rope_tables
    from perf.e2e_sampling import Cfg, backbone_eager, init_params, serve
    cfg = Cfg(vocab=1001, mask=1000, max_seq=512, d=256, heads=4, layers=4, d_ff=512, bs=16)
    p = init_params(cfg, 0, cuda)
    tables = rope_tables(64, cfg.max_seq, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(0)
    prompts = [torch.randint(0, cfg.mask, (16 * n,), generator=g, device=cuda) for n in (1, 17, 0, 5, 9)]
    n_blocks = [2, 1, 3, 1, 0]
    allowed = torch.full((-(-cfg.vocab // 32),), -1, dtype=torch.int32, device=cuda)
    allowed[10:] = 0  # tokens 0 .. 319
    worst = []

    def check(before, block, logits):
        with torch.no_grad():
            cache = [None] * cfg.layers
            if len(before):
                pos = torch.arange(len(before), device=cuda)
                causal = (pos[None, :] // cfg.bs) <= (pos[:, None] // cfg.bs)
                backbone_eager(cfg, p, tables, before[None], cache, True, mask=causal)
            want = backbone_eager(cfg, p, tables, block[None], cache, False)[0].float()
            # a few bf16 ulps of the logit scale, as for the rectangular cache (the
            # rotation's single rounding against the eager path's five among them)
            worst.append(float((want - logits.float()).abs().max() / want.abs().max()))

    def go(check=None):
        with torch.no_grad():  # 14 pages: not all prompts at once
            return serve(cfg, p, tables, prompts, n_blocks, 4, 14, page_size=32, repetition=1.5, allowed=allowed, seed=3,
                         check=check)

    out = go(check)
    print("serving: logits against the eager backbone, max-abs / scale:", [f"{w:.4f}" for w in worst], flush=True)
    assert len(worst) == sum(n_blocks) and max(worst) <= 4 * 2.0 ** -8
    for t, prompt, n in zip(out, prompts, n_blocks):
        assert len(t) == len(prompt) + 16 * n and torch.equal(t[:len(prompt)], prompt)
        assert (t[len(prompt):] < 320).all(), "a token that the grammar forbids was drawn"
    assert all(torch.equal(a, b) for a, b in zip(out, go())), "the same run again draws other tokens"
