"""What the operators before the cache promise beside their results (no GPU)."""

from __future__ import annotations

import copy
import ctypes
from dataclasses import replace
from decimal import Decimal, localcontext
import pickle
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from fragpack_b200.integrations.vllm import backend
from fragpack_b200.ops.fragpack_ext import extension
from fragpack_b200.ops.rotary import make_rotary


@pytest.mark.parametrize("scale", [3e38, 7e-39, 2.0**-140])
def test_scales_whose_powers_of_two_leave_the_range_are_refused(scale) -> None:
    """Weights are powers of two of scale * log2(e) * score: that product must be an ordinary FP32 number."""
    lib, at = extension(), 1 << 20
    code = lib.fp_prompt_attention(at, 1024, 128, at, 256, 128, at, 256, 128, at, 1, 4, at, 1024, 128, 2, 4, scale, None)
    assert code == -1 and "scale" in lib.fp_last_error().decode()


def _described(rotary):
    native = rotary._native
    return native.turns, native.rot_dim, native.interleaved, native.factor


def test_a_rotary_describes_what_it_says() -> None:
    """Also one that was derived from another by replacing fields, copied or pickled."""
    rotary = make_rotary(torch.device("cpu"), 64, interleaved=True)
    other = make_rotary(torch.device("cpu"), 128)
    derived = [
        replace(rotary, factor=2.0), replace(rotary, interleaved=False), replace(rotary, rot_dim=32),
        replace(rotary, turns=other.turns, rot_dim=128), copy.copy(rotary), copy.deepcopy(rotary),
        pickle.loads(pickle.dumps(rotary)),
    ]
    for x in derived:
        assert _described(x) == (x.turns.data_ptr(), x.rot_dim, x.interleaved, x.factor)
        assert ctypes.addressof(x._ref._obj) == ctypes.addressof(x._native)
    assert derived[0].factor == 2.0 and not derived[1].interleaved and derived[2].rot_dim == 32
    for x in derived[4:]:
        assert torch.equal(x.turns, rotary.turns) and (x.rot_dim, x.interleaved, x.factor) == (64, True, 1.0)


def test_a_rotary_without_its_turns_is_refused() -> None:
    rotary = make_rotary(torch.device("cpu"), 64)
    for wrong in (dict(rot_dim=72), dict(rot_dim=12), dict(rot_dim=136), dict(rot_dim=-8), dict(turns=rotary.turns[:31]),
                  dict(turns=rotary.turns.int()), dict(turns=torch.zeros(64, dtype=torch.int64)[::2])):
        with pytest.raises(ValueError):
            replace(rotary, **wrong)


@pytest.mark.parametrize("rot_dim,base", [(128, 10000.0), (64, 500000.0), (96, 1000000.0), (8, 2.0)])
def test_turns_are_within_the_stated_bound_of_the_exact_ones(rot_dim, base) -> None:
    """2^-54 turns per token (see csrc/rotary.cu), against 60-digit decimal arithmetic."""
    with localcontext() as context:
        context.prec = 60
        pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494")
        for i, bits in enumerate(make_rotary(torch.device("cpu"), rot_dim, base).turns.tolist()):
            frequency = (-Decimal(2 * i) / Decimal(rot_dim) * Decimal(base).ln()).exp()
            exact = frequency / (2 * pi)
            assert abs(Decimal(bits % 2**64) / Decimal(2**64) - exact) <= Decimal(2) ** -54


BANDS = {"type": "bands", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original": 8192}
RAMP = {"type": "ramp", "factor": 4.0, "original": 4096}


@pytest.mark.parametrize("scaling", [
    {k: x for k, x in BANDS.items() if k != "original"}, {k: x for k, x in BANDS.items() if k != "low_freq_factor"},
    {k: x for k, x in BANDS.items() if k != "high_freq_factor"}, {k: x for k, x in RAMP.items() if k != "original"},
    {**RAMP, "original": 0}, {**BANDS, "original": -1}, {**RAMP, "beta_slow": 0.0}, {**RAMP, "beta_fast": 0.5},
    {"type": "linear", "factor": float("inf")}, {**RAMP, "beta_fast": float("nan")},
    {**RAMP, "attention_factor": float("nan")},
])
def test_scalings_without_a_meaning_are_refused(scaling) -> None:
    with pytest.raises(ValueError):
        make_rotary(torch.device("cpu"), 64, 10000.0, scaling=scaling)


def test_bases_and_factors_that_are_no_numbers_are_refused() -> None:
    for wrong in (dict(base=float("nan")), dict(base=float("inf")), dict(factor=float("nan")), dict(factor=float("-inf"))):
        with pytest.raises(ValueError):
            make_rotary(torch.device("cpu"), 64, **wrong)


def test_run_layer_attends_over_prompts_with_the_most_precise_weights(monkeypatch) -> None:
    """As the attention over records, which it replaces: a lag of 0."""
    calls = []
    monkeypatch.setattr(backend, "prompt_attention", lambda *args: calls.append(args))
    table, none = torch.arange(20, dtype=torch.int32).view(2, 10), torch.zeros(0)
    groups = backend.plan_prefill_groups(table, 0, 2, np.array([0, 7, 12]), np.array([7, 5]), 100, torch.device("cpu"),
                                         split_whole=True)
    store = SimpleNamespace(write=lambda *a: None, encode=lambda *a: None, commit=lambda: None)
    md = backend.FragPackMetadata(
        store=store, layer_tables=[None], layer_index={}, last_layer=0, slot_mapping=torch.arange(12), num_tokens=12,
        num_decodes=0, decode_block_table=none, decode_seq_lens=none, units=1, decode_workspace=(none,) * 3,
        max_close=0, prefills=groups, wk=none, wv=none, prompt_attention=True,
    )
    q = torch.zeros(12, 8, 128, dtype=torch.bfloat16)
    backend.run_layer(md, 0, q, q[:, :2], q[:, :2], q.clone(), 0.1)
    assert [(args[3].tolist(), args[4], args[6]) for args in calls] == [([0, 7, 12], 0.1, 0.0)]
