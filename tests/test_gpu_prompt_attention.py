"""Attention of packed whole prompts against a plain implementation in 64 bits.

Tolerance of one output o = sum p v / sum p: every probability is rounded to
BF16 once, half a step of 2^-8 relative, so the numerator is off by at most
2^-8 sum p |v|; scores are FP32 sums of 128 products of BF16 values (off by at
most 2^-24 * 128 relative to sum |q||k|, which the inputs keep below 2^-11 in
the exponent) and the exponentials are good to 2^-12, together below 2^-10
sum p |v|; the result is rounded to BF16, 2^-8 |o|.
"""

from __future__ import annotations

import pytest
import torch

from fragpack_b200.ops.fragpack_ext import check, extension
from fragpack_b200.ops.prompt_attn import PROMPT_WAIT_TIMEOUT, prompt_attention, prompt_status

pytestmark = pytest.mark.gpu
DIM = 128
SCALE = DIM**-0.5


def _reference(q, k, v, lens, scale=SCALE):
    """64-bit outputs and their tolerances, prompt by prompt; rows past the prompts are None-like NaN."""
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    size = out.clone()
    group = q.shape[1] // k.shape[1]
    t0 = 0
    for n in lens:
        rows = slice(t0, t0 + n)
        qd, kd, vd = (x[rows].double().transpose(0, 1) for x in (q, k, v))
        kd, vd = kd.repeat_interleave(group, 0), vd.repeat_interleave(group, 0)
        logits = qd @ kd.transpose(1, 2) * scale
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        p = torch.softmax(logits.masked_fill(hidden, float("-inf")), -1)
        out[rows] = (p @ vd).transpose(0, 1)
        size[rows] = (p @ vd.abs()).transpose(0, 1)
        t0 += n
    return out, 2.0**-8 * out.abs() + (2.0**-8 + 2.0**-10) * size


def _check(got, want, rows) -> None:
    out, tolerance = want
    got, out, tolerance = got[:rows].double(), out[:rows], tolerance[:rows]
    assert not torch.isnan(got).any()
    worst = ((got - out).abs() / (tolerance + 1e-30)).max() if rows else 0.0
    assert bool(((got - out).abs() <= tolerance).all()), float(worst)


def _inputs(tokens, h, group, seed=0, layout="packed"):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    heads = h * group + 2 * h
    if layout == "heads outermost":
        qkv = torch.randn(heads, tokens, DIM, generator=gen, device="cuda").to(torch.bfloat16).transpose(0, 1)
    elif layout == "padded rows":
        qkv = torch.randn(tokens, heads + 1, DIM + 8, generator=gen, device="cuda").to(torch.bfloat16)[:, :heads, :DIM]
    else:
        qkv = torch.randn(tokens, heads, DIM, generator=gen, device="cuda").to(torch.bfloat16)
    return qkv[:, : h * group], qkv[:, h * group : h * group + h], qkv[:, h * group + h :]


def _starts(lens):
    return torch.tensor([0, *lens], dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)


LENS = [
    [1], [2], [127], [128], [129], [255], [256], [257], [1, 1, 1], [0, 5, 0, 0, 130, 0], [33, 1, 200, 16, 15, 17],
    [700, 3, 1025], [1] * 70, [64] * 40 + [0] * 40 + [3], [2, 0, 1] * 200 + [300, 7],
]


@pytest.mark.parametrize("h,group", [(1, 8), (4, 8), (2, 4), (3, 2), (2, 1)])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "+".join(map(str, x[:6])) + ("..." if len(x) > 6 else ""))
def test_prompts(lens, h, group) -> None:
    tokens = sum(lens)
    q, k, v = _inputs(tokens, h, group, seed=tokens)
    out = torch.full((tokens, h * group, DIM), float("nan"), dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    _check(out, _reference(q, k, v, lens), tokens)
    assert prompt_status() == 0


@pytest.mark.parametrize("lens,h,group", [([4097], 1, 8), ([2500, 2049], 2, 1), ([1999, 5, 3000], 2, 4)])
def test_long_prompts(lens, h, group) -> None:
    tokens = sum(lens)
    q, k, v = _inputs(tokens, h, group, seed=7)
    out = torch.full((tokens, h * group, DIM), float("nan"), dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    _check(out, _reference(q, k, v, lens), tokens)


@pytest.mark.parametrize("h,group", [(7, 1), (9, 2), (5, 4)])
def test_more_keys_than_are_walked_at_a_time(h, group) -> None:
    """Heads in chunks of four and three, three, and four and one."""
    lens = [50] * 400 + [0, 1, 300] * 30 + [700]
    tokens = sum(lens)
    assert 4 <= (64 << 20) // (tokens * 512) < 5
    q, k, v = _inputs(tokens, h, group, seed=17)
    out = torch.full((tokens, h * group, DIM), float("nan"), dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    _check(out, _reference(q, k, v, lens), tokens)
    assert prompt_status() == 0


@pytest.mark.parametrize("layout", ["heads outermost", "padded rows"])
@pytest.mark.parametrize("h,group", [(2, 4), (1, 2)])
def test_strided_tensors(layout, h, group) -> None:
    lens = [140, 1, 60]
    q, k, v = _inputs(201, h, group, layout=layout)
    store = torch.zeros(h * group, 201, DIM, dtype=torch.bfloat16, device="cuda")
    out = store.transpose(0, 1)
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    _check(out, _reference(q, k, v, lens), 201)


def test_tokens_far_apart() -> None:
    """Token strides that take offsets past 32 bits, in the inputs and the result, heads redone key by key among them."""
    lens, h, group = [17, 3, 22], 2, 2
    q, k, v = _inputs(sum(lens), h, group, seed=8)
    v[30, 1, 7] = float("inf")
    heads = torch.cat([q, k, v, torch.zeros_like(q)], 1)
    stride = (1 << 32) // (sum(lens) - 1) // 8 * 8 + 8
    far = torch.empty((sum(lens) - 1) * stride + heads.shape[1] * DIM, dtype=torch.bfloat16, device="cuda")
    assert far.numel() > 1 << 32
    far = far.as_strided(heads.shape, (stride, DIM, 1))
    far.copy_(heads)
    out = torch.zeros_like(q)
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    at = h * group
    prompt_attention(far[:, :at], far[:, at : at + h], far[:, at + h : at + 2 * h], _starts(lens), SCALE, far[:, at + 2 * h :])
    assert torch.equal(far[:, at + 2 * h :], out) and bool(torch.isinf(out[30:, 2:, 7]).all())


@pytest.mark.parametrize("group", [1, 8])
def test_what_lies_outside_the_prompts_reaches_nothing_and_stays(group) -> None:
    """Rows before, between (clamped starts) and behind the prompts hold NaN; their outputs keep their fill."""
    lens = [100, 45]
    q, k, v = _inputs(200, 2, group)
    want = _reference(q[10:], k[10:], v[10:], lens)
    for t in (q, k, v):
        t[:10], t[155:] = float("nan"), float("inf")
    out = torch.full((200, 2 * group, DIM), 7.0, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts(lens) + 10, SCALE, out)
    _check(out[10:155], want, 145)
    assert bool((out[:10] == 7).all()) and bool((out[155:] == 7).all())


@pytest.mark.parametrize("group", [1, 2, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min])
def test_later_tokens_reach_no_earlier_one(group, bad) -> None:
    """NaN, infinities and the lowest value in the keys and values of a prompt's later tokens."""
    n, first_bad = 400, 301
    q, k, v = _inputs(n, 2, group, seed=3)
    want = _reference(q[:first_bad], k[:first_bad], v[:first_bad], [first_bad])
    k[first_bad:], v[first_bad:] = bad, bad
    v[first_bad + 40 :] = 0.5
    out = torch.zeros(n, 2 * group, DIM, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts([n]), SCALE, out)
    _check(out, want, first_bad)
    if bad != bad:
        assert bool(torch.isnan(out[first_bad:]).all())


def test_value_infinities_show_where_they_are_seen() -> None:
    q, k, v = _inputs(260, 1, 4, seed=9)
    v[200, 0, 5], v[130, 0, 6] = float("inf"), float("-inf")
    out = torch.zeros(260, 4, DIM, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts([260]), SCALE, out)
    assert bool((out[200:, :, 5] == float("inf")).all()) and bool(torch.isfinite(out[:200, :, 5]).all())
    assert bool((out[130:, :, 6] == float("-inf")).all()) and bool(torch.isfinite(out[:130, :, 6]).all())
    rest = torch.ones(DIM, dtype=torch.bool, device="cuda")
    rest[5:7] = False
    assert bool(torch.isfinite(out[..., rest]).all())


@pytest.mark.parametrize("group", [1, 8])
def test_values_whose_weighted_sum_passes_the_range(group) -> None:
    """Equal weights over 1e38: the result is 1e38, though the sum of the values is not in range."""
    n = 700
    q, k, v = _inputs(n, 2, group, seed=12)
    q[:] = 0.0
    v[:] = 1e38
    v[:, 1, 3] = -1e38
    out = torch.zeros(n, 2 * group, DIM, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts([n]), SCALE, out)
    # One rounding to BF16, and 2^-24 for each of at most 700 terms of a sum in FP32.
    want = v.repeat_interleave(group, 1).double()
    assert float(((out.double() - want) / want).abs().max()) <= 2.0**-8 + 700 * 2.0**-24


@pytest.mark.parametrize("where", ["q", "k", "v", "v inf"])
def test_prompts_of_nothing_but_nan_and_infinities(where) -> None:
    """A step that a broken layer left without a number: the result says so, in the time of a sound one."""
    lens = [4000, 1, 333]
    q, k, v = _inputs(sum(lens), 4, 4, seed=13)
    {"q": q, "k": k, "v": v, "v inf": v}[where].fill_(float("inf") if where == "v inf" else float("nan"))
    out = torch.zeros_like(q)
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    assert bool((out == float("inf")).all() if where == "v inf" else torch.isnan(out).all())


def test_single_tokens_return_their_values() -> None:
    q, k, v = _inputs(9, 3, 8)
    out = torch.empty(9, 24, DIM, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts([1] * 9), SCALE, out)
    assert torch.equal(out, v.repeat_interleave(8, 1))


def test_rising_scores_and_large_ones() -> None:
    """Scores that rise with the key's position move the running maximum in every tile; |score| up to 300."""
    n = 900
    q, k, v = _inputs(n, 1, 2, seed=4)
    q[:], k[:] = 0.0, 0.0
    q[..., 0], k[:, 0, 0] = 8.0, torch.arange(n, device="cuda") / 2.0
    out = torch.zeros(n, 2, DIM, dtype=torch.bfloat16, device="cuda")
    for sign in (1.0, -1.0):
        k[:, 0, 0] *= sign
        prompt_attention(q, k, v, _starts([n]), SCALE, out)
        _check(out, _reference(q, k, v, [n]), n)


def test_a_prompt_alone_and_among_others_gives_the_same_bits() -> None:
    lens = [513, 40, 777]
    q, k, v = _inputs(sum(lens), 2, 4, seed=6)
    out = torch.zeros(sum(lens), 8, DIM, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts(lens), SCALE, out)
    again = torch.zeros_like(out)
    t0 = 0
    for n in lens:
        rows = slice(t0, t0 + n)
        prompt_attention(q[rows], k[rows], v[rows], _starts([n]), SCALE, again[rows])
        t0 += n
    assert torch.equal(out, again)


def test_scale_and_empty_calls() -> None:
    q, k, v = _inputs(150, 1, 8)
    out = torch.zeros(150, 8, DIM, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts([150]), 0.01, out)
    _check(out, _reference(q, k, v, [150], 0.01), 150)
    before = out.clone()
    prompt_attention(q, k, v, _starts([]), SCALE, out)
    prompt_attention(q, k, v, _starts([0, 0]), SCALE, out)
    prompt_attention(q[:0], k[:0], v[:0], _starts([0]), SCALE, out[:0])
    assert torch.equal(out, before)


def test_captured_and_replayed_beside_another_stream() -> None:
    lens = [300, 77]
    q, k, v = _inputs(377, 2, 8, seed=1)
    starts = _starts(lens)
    out = torch.zeros(377, 16, DIM, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, starts, SCALE, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prompt_attention(q, k, v, starts, SCALE, out)
    q2, k2, v2 = _inputs(377, 2, 8, seed=2)
    for a, b in ((q, q2), (k, k2), (v, v2)):
        a.copy_(b)
    starts.copy_(_starts([200, 177]))
    side = torch.cuda.Stream()
    other = torch.zeros_like(out)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        prompt_attention(q2, k2, v2, _starts([200, 177]), SCALE, other)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, other)
    _check(out, _reference(q, k, v, [200, 177]), 377)


def test_a_wait_that_runs_out_is_reported() -> None:
    """The loader leaves a key tile out: the call returns, says so, and the next call is sound."""
    q, k, v = _inputs(500, 2, 8, seed=8)
    want = torch.zeros(500, 16, DIM, dtype=torch.bfloat16, device="cuda")
    prompt_attention(q, k, v, _starts([500]), SCALE, want)
    out = torch.zeros_like(want)
    assert prompt_status() == 0
    check(extension().fp_debug_wait_limit(20_000_000, 1))
    try:
        prompt_attention(q, k, v, _starts([500]), SCALE, out)
        torch.cuda.synchronize()
    finally:
        check(extension().fp_debug_wait_limit(0, -1))
    assert prompt_status() == PROMPT_WAIT_TIMEOUT
    assert prompt_status() == 0
    prompt_attention(q, k, v, _starts([500]), SCALE, out)
    assert torch.equal(out, want) and prompt_status() == 0


def test_refusals() -> None:
    q, k, v = _inputs(20, 2, 4)
    out, starts = torch.empty(20, 8, DIM, dtype=torch.bfloat16, device="cuda"), _starts([20])
    good = dict(q=q, k=k, v=v, starts=starts, scale=SCALE, out=out)
    prompt_attention(**good)
    shifted = torch.empty(20 * 2 * DIM + 1, dtype=torch.bfloat16, device="cuda")[1:].view(20, 2, DIM)
    for wrong in (
        dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(q=q.half()),
        dict(k=k[:19]), dict(v=v[:, :1]), dict(out=out[:, :4]), dict(starts=starts.long()), dict(starts=starts.cpu()),
        dict(starts=starts[:0]), dict(k=shifted), dict(v=shifted), dict(out=out.float()),
        dict(k=k[:1].expand(20, 2, DIM)),
    ):
        with pytest.raises(RuntimeError):
            prompt_attention(**{**good, **wrong})
    with pytest.raises(ValueError):
        prompt_attention(q[:, :6], k, v, starts, SCALE, out[:, :6])
    with pytest.raises(ValueError):
        prompt_attention(q[:, :3], k, v, starts, SCALE, out[:, :3])
    torch.cuda.synchronize()
