"""Host-side contracts of norm_rotary, HbmKvStore.append and prompt_attention (no GPU)."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from fragpack_b200.compression.attn_tables import device_tables
from fragpack_b200.integrations.vllm import backend
from fragpack_b200.ops.fragpack_ext import FpHeads, FpRotary, FpStore, extension, pack_heads
from fragpack_b200.ops.hbm_kv import HbmKvStore, page_bytes
from fragpack_b200.ops.prompt_attn import prompt_attention
from fragpack_b200.ops.rotary import make_rotary, norm_rotary, rotary_frequencies


def test_plain_and_linear_frequencies() -> None:
    freq, factor = rotary_frequencies(128, 10000.0)
    assert factor == 1.0 and freq.dtype == np.float64 and freq.shape == (64,)
    for i in (0, 1, 17, 63):
        assert freq[i] == pytest.approx(10000.0 ** (-2 * i / 128), rel=1e-14)
    slow, factor = rotary_frequencies(128, 10000.0, {"type": "linear", "factor": 8})
    assert factor == 1.0 and np.array_equal(slow, freq / 8)


def test_band_scaling_keeps_fast_pairs_and_slows_slow_ones() -> None:
    rule = {"type": "bands", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original": 8192}
    plain, _ = rotary_frequencies(128, 500000.0)
    freq, factor = rotary_frequencies(128, 500000.0, rule)
    assert factor == 1.0
    for f, g in zip(plain, freq):
        wavelength = 2 * math.pi / f
        if wavelength < 8192 / 4.0:
            assert g == f
        elif wavelength > 8192:
            assert g == pytest.approx(f / 8, rel=1e-14)
        else:
            smooth = (8192 / wavelength - 1.0) / 3.0
            assert g == pytest.approx((1 - smooth) * f / 8 + smooth * f, rel=1e-12)


def test_ramp_scaling() -> None:
    rule = {"type": "ramp", "factor": 4.0, "original": 4096}
    plain, _ = rotary_frequencies(64, 10000.0)
    freq, factor = rotary_frequencies(64, 10000.0, rule)
    assert factor == pytest.approx(0.1 * math.log(4.0) + 1.0)
    first = math.floor(64 * math.log(4096 / (2 * math.pi * 32)) / (2 * math.log(10000.0)))
    last = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000.0)))
    assert np.array_equal(freq[: first + 1], plain[: first + 1])
    assert freq[last:] == pytest.approx(plain[last:] / 4)
    middle = (first + last) // 2
    part = (middle - first) / (last - first)
    assert freq[middle] == pytest.approx(plain[middle] * (1 - part) + plain[middle] / 4 * part)
    assert rotary_frequencies(64, 10000.0, {**rule, "attention_factor": 1.25})[1] == 1.25


@pytest.mark.parametrize("bad", [
    dict(rot_dim=127), dict(base=1.0), dict(base=0.0), dict(scaling={"type": "cubic", "factor": 2}),
    dict(scaling={"type": "linear"}), dict(scaling={"type": "linear", "factor": 0.5}),
    dict(scaling={"type": "bands", "factor": 2, "low_freq_factor": 4, "high_freq_factor": 4, "original": 1}),
])
def test_impossible_frequencies_are_refused(bad) -> None:
    with pytest.raises(ValueError):
        rotary_frequencies(**bad)


def test_turns_are_the_binary_fractions_of_the_frequencies() -> None:
    cpu = torch.device("cpu")
    rotary = make_rotary(cpu, 8, frequencies=[math.pi, math.pi / 2, -math.pi / 2, 5 * math.pi])
    assert rotary.turns.dtype == torch.int64
    bits = rotary.turns.numpy().view(np.uint64).tolist()
    assert bits == [1 << 63, 1 << 62, 3 << 62, 1 << 63]  # a half, a quarter, minus a quarter, two and a half turns
    plain = make_rotary(cpu, 128, 10000.0).turns.numpy().view(np.uint64).astype(np.float64) / 2.0**64
    assert plain == pytest.approx(rotary_frequencies(128, 10000.0)[0] / (2 * math.pi), rel=1e-14)
    single = make_rotary(cpu, 8, frequencies=torch.tensor([1.0, 0.1, 0.01, 0.001]))  # a model's float32 table
    assert single.turns.numpy().view(np.uint64)[1] == int(float(np.float32(0.1)) / (2 * math.pi) * 2.0**64)
    for bad in (dict(rot_dim=12), dict(rot_dim=136), dict(rot_dim=8, frequencies=[1.0]),
                dict(rot_dim=8, frequencies=[1.0, 2.0, float("nan"), 1.0])):
        with pytest.raises(ValueError):
            make_rotary(cpu, **bad)


def _cpu_store():
    cpu, heads = torch.device("cpu"), 2
    table = np.broadcast_to(np.arange(22, dtype=np.uint8), (1, 2, heads, 22)).copy()
    return HbmKvStore([torch.zeros(4, page_bytes(heads), dtype=torch.uint8)], heads, device_tables(table, cpu), 16, 2, 1)


def test_operators_have_no_cpu_fallback() -> None:
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    k, positions, rotary = q[:, :2], torch.arange(3), make_rotary(torch.device("cpu"))
    with pytest.raises(RuntimeError, match="CUDA"):
        norm_rotary(q, k, positions, rotary, q, k)
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt_attention(q, k, k, torch.tensor([0, 3], dtype=torch.int32), 0.1, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        _cpu_store().append(0, q, k, k, positions, positions, rotary, q)


def test_library_refuses_before_any_launch() -> None:
    """Bad geometry and alignment come back as messages; the pointers are never used."""
    lib, at = extension(), 1 << 20

    def message(code):
        assert code == -1
        return lib.fp_last_error().decode()

    def prompt(q=at, q_token=1024, k_token=256, prompts=1, tokens=4, kv=2, group=4, scale=0.1, out=at):
        return lib.fp_prompt_attention(q, q_token, 128, at, k_token, 128, at, 256, 128, at, prompts, tokens, out, 1024,
                                       128, kv, group, scale, None)

    assert "group" in message(prompt(group=3)) and "group" in message(prompt(group=16))
    assert "scale" in message(prompt(scale=0.0)) and "scale" in message(prompt(scale=float("nan")))
    assert "aligned" in message(prompt(q=at + 2)) and "aligned" in message(prompt(q_token=1028))
    assert "aligned" in message(prompt(k_token=0)) and "aligned" in message(prompt(k_token=-256))
    assert "null" in message(prompt(out=None))
    assert "geometry" in message(prompt(prompts=-1)) and "geometry" in message(prompt(tokens=1 << 40))
    assert prompt(prompts=0) == 0 and prompt(tokens=0) == 0

    def heads(base=at, out=at, token=512, count=2):
        return ctypes.byref(FpHeads(base, out, token, 128, token, 128, count))

    def rotate(q=None, k=None, rot=128, tokens=3, positions=at, turns=at):
        rotary = FpRotary(turns=turns, rot_dim=rot, interleaved=0, factor=1.0)
        return lib.fp_norm_rotary(q or heads(), k or heads(), None, None, 0, positions, 1, tokens,
                                  ctypes.byref(rotary), 1e-6, None)

    assert "multiple of 8" in message(rotate(rot=12)) and "multiple of 8" in message(rotate(rot=136))
    assert "aligned" in message(rotate(q=heads(base=at + 8))) and "aligned" in message(rotate(k=heads(token=129)))
    assert "aligned" in message(rotate(q=heads(out=at + 2)))
    assert "null" in message(rotate(turns=None)) and "null" in message(rotate(positions=None))
    assert "null" in message(rotate(q=heads(out=None))) and "null" in message(rotate(k=heads(base=None)))
    assert "count" in message(rotate(tokens=-1)) and rotate(tokens=0) == 0

    store = FpStore(**{name: at for name, kind in FpStore._fields_ if kind is ctypes.c_void_p}, overflow_records=1, L=1,
                    H=2, NB=4, S_p=1, S_t=1, ovf_words=1, cap=16)
    rotary = FpRotary(turns=at, rot_dim=128, interleaved=0, factor=1.0)

    def append(k=None, value=at, layer=0, slots=at):
        return lib.fp_hbm_append(ctypes.byref(store), heads(), k or heads(), value, 256, 128, None, None, 0, at, 1, slots,
                                 3, ctypes.byref(rotary), 1e-6, layer, None)

    assert "layer" in message(append(layer=1)) and "layer" in message(append(layer=-1))
    assert "key heads" in message(append(k=heads(count=3)))
    assert "aligned" in message(append(value=at + 4)) and "null" in message(append(slots=None))


def test_groups_know_whole_prompts() -> None:
    table = torch.arange(60, dtype=torch.int32).view(6, 10)
    qsl = np.array([0, 1, 201, 351, 451, 452], np.int64)  # row 0 decodes
    seq = np.array([500, 200, 150, 612, 1], np.int64)     # rows 1, 2 and 4 are whole prompts
    cpu = torch.device("cpu")
    together = backend.plan_prefill_groups(table, 1, 5, qsl, seq, 100, cpu)
    assert [(g.tok0, g.tok1, g.whole) for g in together] == [(1, 452, False)]
    apart = backend.plan_prefill_groups(table, 1, 5, qsl, seq, 100, cpu, split_whole=True)
    assert [(g.tok0, g.tok1, g.whole) for g in apart] == [(1, 351, True), (351, 451, False), (451, 452, True)]
    assert apart[0].cu_seqlens_q.tolist() == [0, 200, 350] and apart[2].cu_seqlens_q.tolist() == [0, 1]


@pytest.mark.parametrize("fused_append", [True, False])
@pytest.mark.parametrize("over_prompt", [True, False])
def test_run_layer_calls_the_operators_it_is_asked_for(monkeypatch, fused_append, over_prompt) -> None:
    calls = []

    class Store:
        def write(self, layer, key, value, slots):
            calls.append(("write", key.shape[0]))

        def append(self, layer, q, k, v, positions, slots, rotary, q_out, k_out, *rest):
            assert q_out is not None and (k_out is not None) == over_prompt
            calls.append(("append", k.shape[0]))

        def encode(self, layer, max_close):
            calls.append("encode")

        def commit(self):
            calls.append("commit")

    monkeypatch.setattr(backend, "norm_rotary", lambda q, *a: calls.append(("norm_rotary", q.shape[0])))
    monkeypatch.setattr(backend, "prompt_attention", lambda q, k, v, starts, *a: calls.append(("prompt", starts.tolist())))
    monkeypatch.setattr(backend, "fused_prefill_attention", lambda q, *a: calls.append(("records", q.shape[0])))
    table = torch.arange(20, dtype=torch.int32).view(2, 10)
    groups = backend.plan_prefill_groups(table, 0, 2, np.array([0, 7, 12]), np.array([7, 300]), 100,
                                         torch.device("cpu"), split_whole=True)
    none = torch.zeros(0)
    md = backend.FragPackMetadata(
        store=Store(), layer_tables=[None], layer_index={}, last_layer=0, slot_mapping=torch.arange(12), num_tokens=12,
        num_decodes=0, decode_block_table=none, decode_seq_lens=none, units=1, decode_workspace=(none,) * 3,
        max_close=0, prefills=groups, wk=none, wv=none, prompt_attention=over_prompt,
    )
    q = torch.zeros(12, 8, 128, dtype=torch.bfloat16)
    transform = backend.HeadTransform(make_rotary(torch.device("cpu")), torch.arange(12))
    backend.run_layer(md, 0, q, q[:, :2], q[:, :2], q.clone(), 0.1, transform=transform, fused_append=fused_append)
    first = [("append", 12)] if fused_append else [("norm_rotary", 12), ("write", 12)]
    second = [("prompt", [0, 7])] if over_prompt else [("records", 7)]
    assert calls == first + second + [("records", 5), "encode", "commit"]


def test_packed_heads_are_the_structure() -> None:
    fields = (1 << 40, 0, 3, -4, 5, 6, 7)
    structure = FpHeads(*fields)
    assert ctypes.string_at(ctypes.byref(structure), ctypes.sizeof(FpHeads)) == pack_heads(*fields)
