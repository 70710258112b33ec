"""Fused SUBS parameterization + ancestral sampling step for BD3-LM
sampling, on MI355X.

`subs_sample_step(logits, block, mask_index, keep)` returns the block after
one denoising step of sample_bd3lm (sample/sampler.py:110-122): SUBS
log-probs of the raw logits (model/subs.py:11-43), q = exp(log_probs) *
(1 - s/t) with q[mask] = s/t, a Gumbel-max draw with float64 noise
(sample_categorical, :11-34), and masked positions replaced by the draw.
bd3_subs_sample_ws does it without writing any (rows, vocab)
intermediate (the reference materialises the log-probs, the carry tensor,
q, the uniforms and the noise, several of them in float64).

`adjust_logits` applies penalties for repeated tokens, biases and grammar masks
to the logits before that step (no reference counterpart).

Noise: pass `u` (float64, the shape of the logits; e.g. torch.rand_like's
draw) to reproduce the reference's arithmetic on the same uniforms, or let
the kernel draw them from a counter-based Philox4x32-10 stream
(`PhiloxStream`): same distribution, nothing materialised.
"""
from __future__ import annotations

import threading

import torch
from torch import Tensor

from kernels._native import host


class PhiloxStream:
    """Seed and running offset of the kernel's Philox4x32-10 draws: each
    step takes a fresh offset, so no counter is ever reused."""

    def __init__(self, seed: int | None = None):
        self.seed = int(torch.initial_seed() if seed is None else seed) & (2 ** 64 - 1)
        self.offset = 0
        self._lock = threading.Lock()

    def next_offset(self) -> int:
        with self._lock:
            off = self.offset
            self.offset += 1
            return off


_default_stream: PhiloxStream | None = None


def default_stream() -> PhiloxStream:
    global _default_stream
    if _default_stream is None:
        _default_stream = PhiloxStream()
    return _default_stream


def subs_sample_step(
    logits: Tensor,   # (..., vocab) raw backbone logits, bf16 or fp32
    block: Tensor,    # (...) int64 current tokens ([MASK] where still masked)
    mask_index: int,
    keep: float,      # s / t of this step (0 at the last step)
    u: Tensor | None = None,            # (..., vocab) float64 uniforms in [0, 1), or None
    generator: PhiloxStream | None = None,
) -> Tensor:
    """The block after one ancestral step (a new int64 tensor shaped like `block`)."""
    assert logits.is_cuda and logits.dtype in (torch.bfloat16, torch.float32), \
        "logits must be bf16 or fp32 CUDA tensors"
    assert logits.shape[:-1] == block.shape, "block must match the logits' leading dims"
    assert 0.0 <= keep <= 1.0, "keep = s / t must lie in [0, 1]"
    if u is not None:
        assert u.shape == logits.shape and u.dtype == torch.float64 and u.device == logits.device
        seed = offset = 0
    else:
        gen = generator or default_stream()
        seed, offset = gen.seed, gen.next_offset()
    return host().subs_sample(logits, block, mask_index, keep, u, seed, offset)


def adjust_logits(
    logits: Tensor,                 # (batch, rows, vocab) or (batch, vocab), bf16 or fp32
    tokens: Tensor | None = None,   # (batch, history) int64: what each sequence holds so far
    lengths: Tensor | None = None,  # (batch) int32: how much of it counts (default: all)
    repetition: float | Tensor = 1.0,
    frequency: float | Tensor = 0.0,
    presence: float | Tensor = 0.0,
    bias: Tensor | None = None,     # (vocab) or (batch, vocab) float32
    allowed: Tensor | None = None,  # int32 words of bits, (words), (batch, words) or (batch, rows, words)
    fill: float = -1e6,
    out: Tensor | None = None,
) -> Tensor:
    """Penalties for tokens a sequence already holds, biases and a grammar mask,
    for the logits that subs_sample_step draws from.

    With c the number of times a token occurs in the first lengths[b] of
    tokens[b]: where c > 0 its logit x becomes x / repetition (x * repetition if
    x <= 0) minus frequency * c + presence; then bias is added; then tokens whose
    bit (bit v % 32 of word v // 32) is 0 are set to `fill`, which SUBS's own
    [MASK] logit (-1e6, model/subs.py:8) is by default: finite, as the draw wants
    it, also in a row whose mask allows nothing. In fp32, rounded once; what leaves
    the dtype's range becomes its largest value of that sign, unless the logit or
    its bias is infinite. The penalties are numbers or (batch) float32 tensors of
    finite values (not looked at), repetition at least 2^-126; tokens outside the
    vocabulary count for nothing. `out=logits` works in place; out overlaps no
    other argument."""
    assert logits.is_cuda and logits.dtype in (torch.bfloat16, torch.float32), \
        "logits must be bf16 or fp32 CUDA tensors"
    assert logits.dim() in (2, 3), "logits must be (batch, rows, vocab) or (batch, vocab)"
    if logits.dim() == 3:
        return host().adjust_logits(logits, tokens, lengths, repetition, frequency, presence, bias, allowed, fill, out)
    assert allowed is None or allowed.dim() <= 2, "allowed must be (words) or (batch, words) for (batch, vocab) logits"
    assert out is None or out.shape == logits.shape, "out must have the logits' shape and dtype, with last stride 1"
    r = host().adjust_logits(logits.unsqueeze(1), tokens, lengths, repetition, frequency, presence, bias, allowed, fill,
                             None if out is None else out.unsqueeze(1))
    return r.squeeze(1)
