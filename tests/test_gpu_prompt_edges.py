"""Packed prompts whose blocks, values or scores are out of the ordinary.

Tolerances are those of ``test_gpu_prompt_attention.py`` where nothing else is said.
"""

from __future__ import annotations

import math

import pytest
import torch

from fragpack_b200.ops.fragpack_ext import check, extension
from fragpack_b200.ops.prompt_attn import PROMPT_WAIT_TIMEOUT, prompt_attention, prompt_status
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


def _stray_reference(q, k, v, lens):
    """As ``_reference``, infinities and NaN of the values added where a row sees them (every weight is positive)."""
    out, tolerance = _reference(q, k, torch.where(torch.isfinite(v), v, torch.zeros_like(v)), lens)
    group, t0 = q.shape[1] // k.shape[1], 0
    for n in lens:
        rows = slice(t0, t0 + n)
        up, down, nan = (torch.cummax(x[rows].int(), 0).values.bool().repeat_interleave(group, 1) if n else x[rows]
                         for x in (v == float("inf"), v == float("-inf"), torch.isnan(v)))
        if n:
            part = out[rows]
            part[up & ~down] = float("inf")
            part[down & ~up] = float("-inf")
            part[nan | (up & down)] = float("nan")
        t0 += n
    return out, tolerance


def _check_stray(got, want) -> None:
    out, tolerance = want
    got = got.double()
    for kind in (torch.isnan, lambda x: x == float("inf"), lambda x: x == float("-inf")):
        assert torch.equal(kind(got), kind(out))
    sound = torch.isfinite(out)
    assert bool(((got - out).abs() <= tolerance)[sound].all())


@pytest.mark.parametrize("h,group", [(2, 1), (3, 2), (2, 8)])
@pytest.mark.parametrize("lens,every", [
    ([400], 40), ([700, 3, 1025], 97), ([1, 80, 79, 160, 81] * 30, 50), ([300] * 160 + [0, 7] * 20, 333), ([257], 1),
    ([513, 600], 3000),
])
def test_stray_values_show_in_the_rows_that_see_them_alone(lens, every, h, group) -> None:
    """Infinities of both signs and NaN in single dims of about one token in `every`, many items of a CTA among them."""
    tokens = sum(lens)
    q, k, v = _inputs(tokens, h, group, seed=every)
    gen = torch.Generator().manual_seed(every)
    for head in range(h):
        for t in torch.randperm(tokens, generator=gen)[: max(3, tokens // every)].tolist():
            dim = int(torch.randint(0, DIM, (1,), generator=gen))
            v[t, head, dim] = (float("inf"), float("-inf"), float("nan"))[t % 3]
    out = torch.zeros(tokens, h * group, DIM, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    _check_stray(out, _stray_reference(q, k, v, lens))
    assert prompt_status() == 0


@pytest.mark.parametrize("what", ["first inf", "last nan", "all inf", "all nan", "large"])
def test_stray_values_take_the_time_of_sound_ones(what) -> None:
    n, h, group = 4096, 2, 8
    q, k, v = _inputs(n, h, group, seed=21)
    bad = v.clone()
    if what == "large":
        bad = bad.sign() * 3e38
    else:
        where, value = what.split()
        bad[{"first": 0, "last": n - 1, "all": slice(None)}[where]] = float(value)
    out, starts = torch.zeros_like(q), _starts([n])

    def milliseconds(values):
        best = float("inf")
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            prompt_attention(q, k, values, starts, SCALE, out)
            end.record()
            torch.cuda.synchronize()
            best = min(best, begin.elapsed_time(end))
        return best

    sound = milliseconds(v)
    assert milliseconds(bad) <= 2.0 * sound + 0.02
    _check_stray(out, _stray_reference(q, k, bad, [n]))


def test_values_of_the_largest_size() -> None:
    """Their weighted mean is in range, whatever their sums are, in prompts of any length."""
    lens = [1, 90, 2000, 5]
    q, k, v = _inputs(sum(lens), 2, 4, seed=22)
    v = v.sign() * 3e38
    out = torch.zeros_like(q)
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    _check(out, _reference(q, k, v, lens), sum(lens))


def test_values_of_a_small_size() -> None:
    """2^-85, in prompts of up to 3,000 tokens: as accurate as others."""
    lens = [1, 90, 3000, 5]
    q, k, v = _inputs(sum(lens), 2, 4, seed=26)
    v = (v.float() * 2.0**-85).to(torch.bfloat16)
    out = torch.zeros_like(q)
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    _check(out, _reference(q, k, v, lens), sum(lens))


def test_one_infinity_in_a_very_long_prompt() -> None:
    n = 140_000
    q, k, v = _inputs(n, 1, 8, seed=23)
    want = torch.zeros_like(q)
    prompt_attention(q, k, v, _starts([n]), SCALE, want)
    v[0, 0, 3], v[n - 50, 0, 4] = float("inf"), float("-inf")
    out = torch.zeros_like(q)
    prompt_attention(q, k, v, _starts([n]), SCALE, out)
    assert prompt_status() == 0
    want[..., 3], want[n - 50 :, :, 4] = float("inf"), float("-inf")
    assert torch.equal(out, want)


@pytest.mark.parametrize("group", [1, 8])
@pytest.mark.parametrize("low", [-4.0, -500.0])
def test_scores_of_minus_infinity(group, low) -> None:
    """Rows that see only such scores are NaN, as the definition has it; later ones ignore them, however low theirs are."""
    n, first = 300, 101
    q, k, v = _inputs(n, 1, group, seed=24)
    q[:], k[:] = 0.0, 0.0
    q[..., 0] = 8.0
    k[:first, 0, 0] = float("-inf")
    k[first:, 0, 0] = low + torch.arange(n - first, device="cuda") / 64.0
    out = torch.zeros_like(q)
    prompt_attention(q, k, v, _starts([n]), SCALE, out)
    want, tolerance = _reference(q, k, v, [n])
    assert bool(torch.isnan(want[:first]).all()) and bool(torch.isnan(out[:first]).all())
    _check(out[first:], (want[first:], tolerance[first:]), n - first)


def test_status_of_a_call_on_another_stream() -> None:
    """Reading the status waits for calls on every stream of the device: this one reports after some 40 ms."""
    q, k, v = _inputs(500, 2, 8, seed=8)
    starts, out = _starts([500]), torch.zeros_like(q)
    assert prompt_status() == 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    check(extension().fp_debug_wait_limit(80_000_000, 1))
    try:
        with torch.cuda.stream(side):
            prompt_attention(q, k, v, starts, SCALE, out)
        assert prompt_status() == PROMPT_WAIT_TIMEOUT
    finally:
        check(extension().fp_debug_wait_limit(0, -1))
    torch.cuda.synchronize()
    assert prompt_status() == 0


@pytest.mark.parametrize("h,group", [(1, 8), (2, 2)])
def test_the_caller_chooses_the_precision_of_the_weights(h, group) -> None:
    """The largest weight is an exact 1 at lag 0; at the default it may be one that BF16 has to round.

    Key 0 has the score 0 and key 200 that of a weight of 128.5, halfway between two BF16 values: relative to the first
    key tile's maximum its rounding is off by 2^-8, relative to its own by nothing, and key 0's weight of 1 / 128.5 is
    off by 2^-8 of that.  All other keys are 2^-60 of key 0 and vanish.
    """
    n = 900
    q, k, v = _inputs(n, h, group, seed=25)
    log2_score = 16.0 * SCALE * 1.4426950408889634  # of a key's dim 0 or 1, in powers of two
    q[:], k[:] = 0.0, 0.0
    q[..., :2] = 16.0
    k[..., 0] = -60.0 / log2_score
    score = math.log2(128.5) / log2_score
    k[0, :, 0], k[200, :, 0] = 0.0, score
    k[200, :, 1] = score - float(k[200, 0, 0])
    want, _ = _reference(q, k, v, [n])
    error = {}
    for lag in (0.0, 8.0):
        out = torch.zeros_like(q)
        prompt_attention(q, k, v, _starts([n]), SCALE, out, lag)
        _check(out, _reference(q, k, v, [n]), n)
        error[lag] = (out.double() - want)[200:]
    v0, v200 = (v[t].repeat_interleave(group, 0).double().abs() for t in (0, 200))
    # The result's rounding, key 0's weight's, and FP32 scores and exponentials (as in _reference).
    assert bool((error[0.0].abs() <= 2.0**-8 * want[200:].abs() + 2.0**-8 * v0 / 128.5 + 2.0**-10 * (v200 + v0 / 128.5)).all())
    assert float(error[8.0].square().mean()) > 2.0 * float(error[0.0].square().mean())


@pytest.mark.parametrize("lag", [-1.0, 8.5, float("nan"), float("inf")])
def test_impossible_lags_are_refused(lag) -> None:
    q, k, v = _inputs(20, 2, 4)
    with pytest.raises(RuntimeError, match="lag"):
        prompt_attention(q, k, v, _starts([20]), SCALE, torch.empty_like(q), lag)
