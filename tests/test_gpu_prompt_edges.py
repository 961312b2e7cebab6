"""Packed prompts whose blocks, values or scores are out of the ordinary.

Tolerances are those of ``test_gpu_prompt_attention.py`` where nothing else is said.
"""

from __future__ import annotations

import pytest
import torch

from fragpack_b200.ops.fragpack_ext import check, extension
from fragpack_b200.ops.prompt_attn import prompt_attention, prompt_status
from tests.test_gpu_prompt_attention import DIM, SCALE, _check, _inputs, _reference, _starts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,h,group", [
    ([1] * 70, 3, 2), ([0, 5, 0, 0, 130, 0], 2, 4), ([50] * 400 + [0, 1, 300] * 30 + [700], 7, 1), ([4097, 12], 1, 8),
    ([2, 0, 1] * 200 + [300, 7], 4, 8),
])
def test_blocks_in_falling_order(lens, h, group) -> None:
    """Blocks without an item come first and every CTA's items fall in number: the same bits as in rising order."""
    tokens = sum(lens)
    q, k, v = _inputs(tokens, h, group, seed=tokens)
    rising, falling = (torch.full((tokens, h * group, DIM), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    prompt_attention(q, k, v, _starts(lens), SCALE, rising)
    check(extension().fp_debug_falling_blocks(1))
    try:
        prompt_attention(q, k, v, _starts(lens), SCALE, falling)
    finally:
        check(extension().fp_debug_falling_blocks(0))
    _check(rising, _reference(q, k, v, lens), tokens)
    assert torch.equal(rising, falling)
    assert prompt_status() == 0
