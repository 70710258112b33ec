"""Which bounds a cache has: selections that would rank pages by bounds that no call formed are refused. On the CPU, where a
selection that is let through ends at the kernels' own refusal of CPU tensors."""
from __future__ import annotations

import pytest
import torch

from kernels.paged import PagedKVCache

D, BF = 64, torch.bfloat16
REFUSED, PASSED = "update_bounds in every step", "CUDA"


def cache(pages=64, layers=2, page=16):
    return PagedKVCache(layers, pages, 1, page, device="cpu", bounds=True)


def step(c, seqs, tokens, formed=(0, 1), commit=True):
    """A step whose bounds are formed in some layers."""
    batch = c.batch(seqs, tokens)
    for layer in formed:
        batch.bounds_formed(layer)
    if commit:
        batch.commit()
    return batch


def select(batch, layer=0, bs=1, top=4, **kw):
    with pytest.raises(AssertionError) as e:
        batch.attention(torch.zeros(batch.tokens, 1, D, dtype=BF), layer, bs, top=top, **kw)
    text = str(e.value)
    assert (REFUSED in text) != (PASSED in text), text
    return PASSED in text


def test_committed_steps_with_and_without_bounds():
    c = cache()
    a = c.add()
    step(c, [a], [200])
    assert select(c.batch([a], [1]))
    step(c, [a], [30], formed=(0,))  # tokens 200-229: layer 1 is left behind at 200
    batch = c.batch([a], [1])
    # the token at 230 ranks pages up to 230 // 16 - 1 = 13: 208 tokens
    assert select(batch, 0) and not select(batch, 1)
    # pages 0 to 11 hold 192 of the 200 tokens
    assert select(batch, 1, recent=2) and not select(batch, 1, recent=0)
    assert select(batch, 1, top=15), "every page is taken: nothing is ranked"
    assert select(batch, 1, first=13, top=15), "the others are always taken"
    assert not select(batch, 1, top=14)


def test_a_gap_is_not_covered_by_later_steps():
    c = cache()
    a = c.add()
    step(c, [a], [100])
    step(c, [a], [64], formed=())
    step(c, [a], [64])
    assert not select(c.batch([a], [1]))
    step(c, [a], [1])
    assert not select(c.batch([a], [1]))


def test_a_short_step_without_bounds_is_covered_by_the_next_in_its_page():
    """page_bounds goes over all keys of the pages that a step touches, earlier ones among them."""
    c = cache()
    a = c.add()
    step(c, [a], [96])
    step(c, [a], [5], formed=())
    assert select(c.batch([a], [1])), "tokens 96-100 lie in the page that is always taken"
    step(c, [a], [4])
    step(c, [a], [100])
    assert select(c.batch([a], [1]))


def test_drafts_do_not_count():
    c = cache()
    a = c.add()
    step(c, [a], [160])
    step(c, [a], [64], commit=False)
    step(c, [a], [64], formed=())
    assert not select(c.batch([a], [1]))


def test_bounds_formed_after_the_commit():
    c = cache()
    a, b = c.add(), c.add()
    first = step(c, [a, b], [160, 0], formed=())
    assert not select(c.batch([a], [1]))
    first.bounds_formed(0)
    batch = c.batch([a, b], [1, 1])
    assert select(batch, 0) and not select(batch, 1)
    # an older step's call forms its last page without the tokens that came since
    later = step(c, [a], [100], formed=(0,))
    assert select(c.batch([a], [1]), 0)
    first.bounds_formed(0)
    assert not select(c.batch([a], [1]), 0)
    later.bounds_formed(0)
    assert select(c.batch([a], [1]), 0)


def test_steps_of_several_blocks():
    """The later blocks of a step rank pages of the step itself."""
    c = cache()
    a = c.add()
    prompt = c.batch([a], [200])
    assert not select(prompt, bs=16)
    prompt.bounds_formed(0)
    assert select(prompt, bs=16) and not select(prompt, 1, bs=16)
    assert select(prompt, 1, bs=1 << 30), "one block: its pages are its own"
    prompt.bounds_formed(1)
    prompt.commit()
    assert select(c.batch([a], [16]), bs=16)
    assert not select(c.batch([a], [48]), bs=16)


def test_a_recycled_page_brings_no_bounds():
    c = cache(pages=14)
    a = c.add()
    step(c, [a], [200])
    c.free(a)
    b = c.add()
    step(c, [b], [200], formed=())
    assert not select(c.batch([b], [1]))


def test_every_sequence_counts():
    c = cache()
    a, b = c.add(), c.add()
    step(c, [a], [200])
    step(c, [b], [200], formed=())
    assert select(c.batch([a], [1])) and not select(c.batch([b], [1])) and not select(c.batch([a, b], [1, 1]))
    assert select(c.batch([a, b], [1, 0])), "no tokens, no selection"
    short = c.add()
    assert select(c.batch([a, short], [1, 40]))


def test_layers_are_counted_from_either_end():
    c = cache()
    a = c.add()
    batch = step(c, [a], [200], formed=(-1,), commit=False)
    assert select(batch, 1, bs=16) and select(batch, -1, bs=16) and not select(batch, 0, bs=16) and not select(batch, -2, bs=16)
    batch.commit()
    assert select(c.batch([a], [1]), 1) and not select(c.batch([a], [1]), 0)
    with pytest.raises(IndexError):
        batch.bounds_formed(2)
