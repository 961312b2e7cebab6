"""What the operators before the cache promise beside their results (no GPU)."""

from __future__ import annotations

import pytest

from fragpack_b200.ops.fragpack_ext import extension


@pytest.mark.parametrize("scale", [3e38, 7e-39, 2.0**-140])
def test_scales_whose_powers_of_two_leave_the_range_are_refused(scale) -> None:
    """Weights are powers of two of scale * log2(e) * score: that product must be an ordinary FP32 number."""
    lib, at = extension(), 1 << 20
    code = lib.fp_prompt_attention(at, 1024, 128, at, 256, 128, at, 256, 128, at, 1, 4, at, 1024, 128, 2, 4, scale, None)
    assert code == -1 and "scale" in lib.fp_last_error().decode()
