"""Forms of norm_rotary and HbmKvStore.append at the borders between their kernels."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fragpack_b200.ops.rotary import make_rotary, norm_rotary
from tests.test_gpu_rotary import T, _heads, _records, _store

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,hq,h", [(384, 180, 4), (385, 180, 4), (384, 64, 8), (16, 5000, 2)])
def test_append_of_many_heads(tokens, hq, h) -> None:
    """The largest appends that go row by row, and the first that go by groups: as norm_rotary and write, bit for bit."""
    a, b = _store(h), _store(h)
    rotary, w = make_rotary(a.counters.device), torch.rand(2, 128, device="cuda")
    slots, positions = torch.arange(tokens, device="cuda"), torch.arange(7, 7 + tokens, device="cuda")
    _, q, k, v = _heads(tokens, hq, h, seed=tokens)
    for s in (a, b):
        s.prepare(slots, tokens, np.arange(-(-tokens // T), dtype=np.int32))
    q_out, k_out, want_q, want_k = (torch.zeros_like(x) for x in (q, k, q, k))
    a.append(0, q, k, v, positions, slots, rotary, q_out, k_out, w[0], w[1])
    norm_rotary(q, k, positions, rotary, want_q, want_k, w[0], w[1])
    b.write(0, want_k, v, slots)
    assert torch.equal(q_out, want_q) and torch.equal(k_out, want_k)
    blocks = range(-(-tokens // T))
    assert torch.equal(_records(a, 0, blocks), _records(b, 0, blocks))
