"""Norms and rotation of query and key heads against a plain implementation in 64 bits.

Tolerance of one result y = factor * (a cos t - b sin t), a and b the normed
members of its pair: the one rounding to BF16 is off by at most half a step,
2^-8 |y|; sine and cosine are off by at most 2^-20 (special-function unit
2^-20.9, plus 2^-24 from the angle and 2^-24 from the scaling), the norm's
factor by at most 2^-20 relative (128 squares summed in FP32: at most 2^-24 a
step over 11 steps; reciprocal root 2^-22), products and sum 2^-23: together
below 2^-18 factor (|a| + |b|).  Dims that are only normed have b = 0.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from fragpack_b200.compression.attn_tables import device_tables
from fragpack_b200.ops.hbm_kv import HbmKvStore, page_bytes
from fragpack_b200.ops.rotary import make_rotary, norm_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
DIM, EPS = 128, 1e-6


def _reference(x, weight, positions, freq, factor, rot_dim, interleaved, eps=EPS):
    """64-bit result and its tolerance; x [T, heads, 128]."""
    x = x.double()
    if weight is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.double()
    angle = positions.double()[:, None] * torch.as_tensor(freq, device=x.device)
    cos, sin = angle.cos()[:, None] * factor, angle.sin()[:, None] * factor
    half = rot_dim // 2
    i = torch.arange(half, device=x.device)
    m, n = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, size = x.clone(), x.abs()
    y[..., m], y[..., n] = x[..., m] * cos - x[..., n] * sin, x[..., n] * cos + x[..., m] * sin
    size[..., m] = size[..., n] = factor * (x[..., m].abs() + x[..., n].abs())
    return y, 2.0**-8 * y.abs() + 2.0**-18 * size + 1e-37


def _check(got, want) -> None:
    y, tolerance = want
    assert not torch.isnan(got).any()
    assert bool(((got.double() - y).abs() <= tolerance).all()), float(((got.double() - y).abs() / tolerance).max())


def _heads(tokens, hq, h, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(tokens, hq + 2 * h, DIM, generator=gen, device="cuda") * scale
    qkv = qkv.to(torch.bfloat16)
    return qkv, qkv[:, :hq], qkv[:, hq : hq + h], qkv[:, hq + h :]


CASES = [
    # tokens, hq, h, rot_dim, interleaved, weights, position dtype, highest position
    (1, 32, 4, 128, False, torch.bfloat16, torch.int64, 8192),
    (1, 1, 1, 128, True, None, torch.int32, 2),
    (3, 5, 3, 64, False, torch.float32, torch.int32, 131072),
    (17, 8, 1, 96, True, torch.bfloat16, torch.int64, 131072),
    (33, 7, 7, 8, False, None, torch.int64, 1 << 20),
    (129, 64, 8, 128, False, None, torch.int64, 1 << 33),
    (300, 9, 2, 120, False, torch.float32, torch.int64, 1000),
    (40, 6, 3, 120, True, None, torch.int32, (1 << 31) - 1),
    (1000, 32, 32, 128, False, torch.bfloat16, torch.int64, 32768),
    (5, 4, 2, 0, False, torch.bfloat16, torch.int64, 100),
    # From 65,536 rows on a half warp takes sixteen heads of a token.
    (2107, 30, 3, 64, True, torch.float32, torch.int64, 32768),
    (901, 73, 1, 128, False, None, torch.int32, 4096),
]


@pytest.mark.parametrize("tokens,hq,h,rot_dim,interleaved,weights,pos_type,highest", CASES)
def test_norm_rotary(tokens, hq, h, rot_dim, interleaved, weights, pos_type, highest) -> None:
    _, q, k, _ = _heads(tokens, hq, h)
    gen = torch.Generator(device="cuda").manual_seed(3)
    positions = torch.randint(0, highest, (tokens,), generator=gen, device="cuda").to(pos_type)
    positions[0] = highest - 1
    wq = wk = None
    if weights is not None:
        wq, wk = torch.randn(2, DIM, generator=gen, device="cuda").to(weights).unbind(0)
    rotary = make_rotary(q.device, rot_dim, 10000.0, interleaved)
    freq, factor = rotary_frequencies(rot_dim, 10000.0)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    norm_rotary(q, k, positions, rotary, q_out, k_out, wq, wk, EPS)
    _check(q_out, _reference(q, wq, positions, freq, factor, rot_dim, interleaved))
    _check(k_out, _reference(k, wk, positions, freq, factor, rot_dim, interleaved))


@pytest.mark.parametrize("scaling", [
    {"type": "linear", "factor": 4.0},
    {"type": "bands", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original": 8192},
    {"type": "ramp", "factor": 4.0, "original": 8192},
    {"type": "ramp", "factor": 16.0, "original": 4096, "attention_factor": 0.7, "beta_fast": 20.0},
])
def test_scaled_frequencies_and_factor(scaling) -> None:
    _, q, k, _ = _heads(50, 4, 2)
    positions = torch.arange(40000, 40050, device="cuda")
    rotary = make_rotary(q.device, 128, 500000.0, False, scaling)
    freq, factor = rotary_frequencies(128, 500000.0, scaling)
    assert rotary.factor == factor
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    norm_rotary(q, k, positions, rotary, q_out, k_out)
    _check(q_out, _reference(q, None, positions, freq, factor, 128, False))
    _check(k_out, _reference(k, None, positions, freq, factor, 128, False))


def test_given_frequencies_and_negative_positions() -> None:
    _, q, _, _ = _heads(9, 3, 1)
    freq = [0.0, 1.0, -0.25, 7.0]  # standing, ordinary, backwards, more than a turn per token
    rotary = make_rotary(q.device, 8, interleaved=True, frequencies=freq, factor=1.5)
    positions = torch.arange(-4, 5, device="cuda", dtype=torch.int32)
    q_out = torch.empty_like(q)
    norm_rotary(q, None, positions, rotary, q_out, None)
    _check(q_out, _reference(q, None, positions, np.array(freq), 1.5, 8, True))


def test_in_place_and_strided_results_equal_fresh_ones() -> None:
    qkv, q, k, v = _heads(77, 8, 2)
    before = qkv.clone()
    positions = torch.arange(77, device="cuda")
    rotary = make_rotary(q.device)
    w = torch.rand(DIM, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    norm_rotary(q, k, positions, rotary, q_out, k_out, w, w)
    assert torch.equal(qkv, before)
    # Heads outermost.
    other_q, other_k = (torch.empty(t.shape[1], 77, DIM, dtype=t.dtype, device="cuda").transpose(0, 1) for t in (q, k))
    norm_rotary(q, k, positions, rotary, other_q, other_k, w, w)
    assert torch.equal(other_q, q_out) and torch.equal(other_k, k_out)
    norm_rotary(q, k, positions, rotary, q, k, w, w)
    assert torch.equal(q, q_out) and torch.equal(k, k_out)
    assert torch.equal(v, before[:, 10:])


def test_unrotated_dims_keep_their_bits_and_rows_stay_apart() -> None:
    _, q, k, _ = _heads(40, 4, 2)
    odd = torch.tensor([0x7FC1, 0xFF80, 0x0001, 0x8000, 0x7F80, 0xFFFF], device="cuda").to(torch.int16)
    q.view(torch.int16)[7, 2, 64:70] = odd
    rotary = make_rotary(q.device, 64)
    positions = torch.arange(40, device="cuda")
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    norm_rotary(q, k, positions, rotary, q_out, k_out)
    assert torch.equal(q_out[..., 64:].contiguous().view(torch.int16), q[..., 64:].contiguous().view(torch.int16))
    # A row that holds NaN and infinities spoils itself alone.
    w = torch.ones(DIM, device="cuda")
    norm_rotary(q, k, positions, rotary, q_out, k_out, w, w)
    bad = torch.isnan(q_out).any(-1)
    assert bad[7, 2] and int(bad.sum()) == 1 and not torch.isnan(k_out).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_at_any_address(dtype) -> None:
    """A weight that is a slice of a larger tensor: only its own alignment is asked for."""
    _, q, k, _ = _heads(20, 3, 2)
    rotary, positions = make_rotary(q.device), torch.arange(20, device="cuda")
    freq, factor = rotary_frequencies()
    weights = torch.rand(2 * DIM + 1, device="cuda").to(dtype)[1:]
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    norm_rotary(q, k, positions, rotary, q_out, k_out, weights[:DIM], weights[DIM:])
    _check(q_out, _reference(q, weights[:DIM], positions, freq, factor, 128, False))
    _check(k_out, _reference(k, weights[DIM:], positions, freq, factor, 128, False))


def test_rows_of_zeros_and_of_large_and_small_values() -> None:
    q = torch.zeros(3, 2, DIM, dtype=torch.bfloat16, device="cuda")
    q[1], q[2] = 1e18, 1e-18
    positions = torch.tensor([5, 6, 7], device="cuda")
    w = torch.ones(DIM, device="cuda")
    rotary = make_rotary(q.device)
    freq, factor = rotary_frequencies()
    out = torch.empty_like(q)
    norm_rotary(q, None, positions, rotary, out, None, w)
    _check(out, _reference(q, w, positions, freq, factor, 128, False))
    assert not out[0].any()


def test_no_tokens_no_heads() -> None:
    _, q, k, _ = _heads(4, 2, 2)
    rotary = make_rotary(q.device)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    norm_rotary(q[:0], k[:0], none, rotary, q[:0], k[:0])
    before = k.clone()
    norm_rotary(q[:, :0], k, torch.arange(4, device="cuda"), make_rotary(q.device, 0), q[:, :0], k)
    assert torch.equal(k, before)


def test_captured_on_another_stream_and_replayed_with_new_inputs() -> None:
    _, q, k, _ = _heads(20, 8, 4)
    positions = torch.arange(20, device="cuda")
    rotary = make_rotary(q.device)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    norm_rotary(q, k, positions, rotary, q_out, k_out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        norm_rotary(q, k, positions, rotary, q_out, k_out)
    q.copy_(torch.randn(q.shape, device="cuda"))
    positions += 1000
    graph.replay()
    want_q, want_k = torch.empty_like(q), torch.empty_like(k)
    norm_rotary(q, k, positions, rotary, want_q, want_k)
    assert torch.equal(q_out, want_q) and torch.equal(k_out, want_k)


# ---------------------------------------------------------------------------- append

L, T, NB = 2, 128, 24
FILL = np.int16(np.uint16(0xA5A5).view(np.int16))


def _store(h, staging_slots=NB, max_tokens=2048):
    device = torch.device("cuda", torch.cuda.current_device())
    table = np.broadcast_to(np.arange(22, dtype=np.uint8), (L, 2, h, 22)).copy()
    arenas = [torch.empty(NB, page_bytes(h), dtype=torch.uint8, device=device) for _ in range(L)]
    store = HbmKvStore(arenas, h, device_tables(table, device), max_tokens, staging_slots, 4)
    store.arenas = arenas
    store.staging.view(torch.int16).fill_(int(FILL))
    store.scratch.view(torch.int16).fill_(int(FILL))
    return store


def _records(store, layer, blocks):
    """Staged bits of the blocks' records, wherever each store placed them."""
    addr = store.rec_addr[layer].cpu().numpy()
    pools = [(t.data_ptr(), t.numel(), t.view(-1)) for t in (store.staging, store.scratch)]
    rows = []
    for b in blocks:
        for a in addr[b].ravel().tolist():
            (base, flat), = [(base, flat) for base, size, flat in pools if base <= a < base + size]
            rows.append(flat[a - base : a - base + 32768].view(torch.int16))
    return torch.stack(rows)


# name -> steps; a step is a list of rows (block list, first position, token count); "pad": unstored tokens.
LAYOUTS = {
    "one token": [[([3], 0, 1)], [([3], 1, 1)]],
    "whole blocks": [[([1, 2, 3], 0, 3 * T)]],
    "shifted rows": [[([4], 0, 5), ([5, 6], 0, T + 37), ([9], 0, 16)]],
    "continued block": [[([7, 8], 0, 21)], [([7, 8], 21, 200)]],
    "decode batch": [[([b], 0, 10 + 3 * b) for b in range(16)], [([b], 10 + 3 * b, 1) for b in range(16)]],
    "many rows": [[([b], 0, 1 + 11 * b % T) for b in range(20)]],
    # More than 384 tokens: groups of sixteen that start anywhere among the input's sixteens, beside single tokens.
    "long rows": [
        [([1], 0, 5), ([2, 3, 4, 5], 0, 3 * T + 37), ([6], 0, 16), ([7], 0, 1), ([8, 9], 0, T + 2)],
        [([1], 5, 100), ([5, 13], 3 * T + 37 - 3 * T, 98), ([10, 11, 12], 0, 301), ([9], 2, 1)],
    ],
}


@pytest.mark.parametrize("h,group", [(1, 8), (5, 2), (4, 8), (32, 1)])
@pytest.mark.parametrize("name", list(LAYOUTS))
def test_append_equals_norm_rotary_then_write(name, h, group) -> None:
    """Bit for bit: staged records, rotated queries and kept keys; unwritten scalars keep their fill."""
    interleaved, keep = group == 2, h != 5
    a, b = _store(h), _store(h)
    rotary = make_rotary(a.counters.device, 128 if h != 1 else 64, 10000.0, interleaved)
    w = torch.rand(2, DIM, device="cuda").to(torch.bfloat16) if h == 4 else (None, None)
    seen = set()  # every block stays live: a slot given back would bring its old block's scalars along
    for step, rows in enumerate(LAYOUTS[name]):
        pos = [p for _, start, n in rows for p in range(start, start + n)]
        slots = [blocks[p // T] * T + p % T for blocks, start, n in rows for p in range(start, start + n)]
        if name in ("shifted rows", "decode batch", "long rows"):  # unstored tokens before, inside and behind
            pos, slots = [9] + pos[:3] + [0] + pos[3:] + [1, 2], [-1] + slots[:3] + [-7] + slots[3:] + [-1, -1]
        if name == "whole blocks":  # input order broken inside a group of sixteen
            pos[32:34], slots[32:34] = pos[33:31:-1], slots[33:31:-1]
        n = len(slots)
        positions = torch.tensor(pos, device="cuda")
        slot_t = torch.tensor(slots, device="cuda")
        touched = sorted({s // T for s in slots if s >= 0})
        seen.update(touched)
        for s in (a, b):
            s.prepare(slot_t, n, np.array(sorted(seen), np.int32))
        for layer in range(L):
            _, q, k, v = _heads(n, h * group, h, seed=10 * step + layer)
            q_out, k_out = torch.zeros_like(q), torch.zeros_like(k)
            want_q, want_k = torch.zeros_like(q), torch.zeros_like(k)
            a.append(layer, q, k, v, positions, slot_t, rotary, q_out, k_out if keep else None, w[0], w[1])
            norm_rotary(q, k, positions, rotary, want_q, want_k, w[0], w[1])
            b.write(layer, want_k, v, slot_t)
            assert torch.equal(q_out, want_q)
            if keep:
                assert torch.equal(k_out, want_k)
            assert torch.equal(_records(a, layer, touched), _records(b, layer, touched)), layer
        for s in (a, b):
            s.commit()


def test_append_in_place_and_captured() -> None:
    """The decode step's form: queries and keys in place, one captured launch, replayed on new tokens."""
    h, n = 4, 6
    store, plain = _store(h), _store(h)
    rotary = make_rotary(store.counters.device)
    slot_t = torch.arange(n, device="cuda") * T
    for s in (store, plain):
        s.prepare(slot_t, n, np.arange(n, dtype=np.int32))
    qkv, q, k, v = _heads(n, 8 * h, h)
    positions = torch.full((n,), 4096, device="cuda", dtype=torch.int32)
    store.append(0, q, k, v, positions, slot_t, rotary, q, k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        store.append(0, q, k, v, positions, slot_t, rotary, q, k)
    fresh, _, _, _ = _heads(n, 8 * h, h, seed=5)
    qkv.copy_(fresh)
    slot_t += 1
    positions += 1
    graph.replay()
    fq, fk, fv = fresh[:, : 8 * h], fresh[:, 8 * h : 9 * h], fresh[:, 9 * h :]
    norm_rotary(fq, fk, positions, rotary, fq, fk)
    assert torch.equal(qkv, fresh)
    # The first call's token sits at offset 0; the replayed one must equal a write of the rotated keys.
    plain.append(0, *_heads(n, 8 * h, h)[1:], positions - 1, slot_t - 1, rotary, torch.empty_like(q))
    plain.write(0, fk, fv, slot_t)
    assert torch.equal(_records(store, 0, range(n)), _records(plain, 0, range(n)))


def test_append_refuses_what_it_cannot_take() -> None:
    h = 4
    store = _store(h)
    rotary = make_rotary(store.counters.device)
    _, q, k, v = _heads(3, 8, h)
    pos, slots = torch.arange(3, device="cuda"), torch.arange(3, device="cuda")
    out = torch.empty_like(q)
    good = dict(layer=0, query=q, key=k, value=v, positions=pos, slot_mapping=slots, rotary=rotary, query_out=out)
    store.prepare(slots, 3, np.zeros(0, np.int32))
    store.append(**good)
    shifted = torch.empty(3 * 8 * DIM + 1, dtype=torch.bfloat16, device="cuda")[1:].view(3, 8, DIM)
    for wrong in (
        dict(layer=L), dict(layer=-1), dict(key=k[:, :2]), dict(value=v[:2]), dict(value=v.float()),
        dict(query=q.half()), dict(query=q[:2]), dict(query_out=out[:, :4]), dict(query=shifted),
        dict(positions=pos[:2]), dict(positions=pos.float()), dict(slot_mapping=slots.int()),
        dict(slot_mapping=slots[:2]), dict(key_out=k.float()), dict(positions=pos.cpu()),
        dict(query_weight=torch.ones(64, device="cuda")), dict(key_weight=torch.ones(DIM, device="cuda").half()),
        dict(query_weight=torch.ones(DIM, device="cuda"), key_weight=torch.ones(DIM, device="cuda").bfloat16()),
        dict(query=q.transpose(1, 2).contiguous().transpose(1, 2)),
    ):
        with pytest.raises(RuntimeError):
            store.append(**{**good, **wrong})
    torch.cuda.synchronize()


def test_rotary_frequency_period() -> None:
    """A frequency of exactly a quarter turn per token: four tokens bring every pair back, at any distance."""
    q = torch.randn(3, 1, DIM, device="cuda").to(torch.bfloat16)
    q[1:] = q[0]
    rotary = make_rotary(q.device, 128, frequencies=[math.pi / 2] * 64)
    out = torch.empty_like(q)
    norm_rotary(q, None, torch.tensor([0, 4, 1 << 20], device="cuda"), rotary, out, None)
    assert torch.equal(out[0], q[0]) and torch.equal(out[1], q[0])
    assert bool(((out[2].double() - q[0].double()).abs() <= 2.0**-8 * q[0].double().abs() + 1e-4).all())


def _far_apart(heads, stride):
    """The same values with tokens `stride` scalars apart, so that offsets pass 32 bits."""
    tokens = heads.shape[0]
    far = torch.empty((tokens - 1) * stride + heads.shape[1] * DIM, dtype=torch.bfloat16, device="cuda")
    assert far.numel() > 1 << 32
    far = far.as_strided(heads.shape, (stride, DIM, 1))
    far.copy_(heads)
    return far


@pytest.mark.parametrize("tokens", [40, 420])
def test_tokens_far_apart(tokens) -> None:
    """Rows of 2^32 scalars and more, in place, alone and on the way into the store (few and many tokens)."""
    h, group = 2, 2
    qkv, q, k, v = _heads(tokens, h * group, h, seed=3)
    far = _far_apart(qkv, -(-(1 << 32) // (tokens - 1) // 8) * 8 + 8)
    positions, slots = torch.arange(tokens, device="cuda"), torch.arange(tokens, device="cuda")
    near, wide = _store(h), _store(h)
    rotary = make_rotary(near.counters.device)
    for store in (near, wide):
        store.prepare(slots, tokens, np.arange(-(-tokens // T), dtype=np.int32))
    wide.append(0, far[:, : h * group], far[:, h * group : h * (group + 1)], far[:, h * (group + 1) :], positions, slots,
                rotary, far[:, : h * group], far[:, h * group : h * (group + 1)])
    near.append(0, q, k, v, positions, slots, rotary, q, k)
    assert torch.equal(far, qkv)
    blocks = range(-(-tokens // T))
    assert torch.equal(_records(near, 0, blocks), _records(wide, 0, blocks))
    norm_rotary(far[:, : h * group], None, positions, rotary, far[:, : h * group], None)
    norm_rotary(q, None, positions, rotary, q, None)
    assert torch.equal(far, qkv)
