"""The three operators together, as a layer uses them.

Requests go through whole-prompt prefill, later chunks and decode steps via
``run_layer`` with projected heads that are neither normed nor rotated yet.
Every output row must match fp32 causal attention over that request's normed
and rotated history (those values come from ``norm_rotary``, which
``test_gpu_rotary.py`` holds to 64 bits) within the bar of the other attention
flows, 1e-2 max-abs and 2e-3 mean-abs on BF16 outputs; and fused, two-step and
record-reading paths must leave the same bytes in the store.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fragpack_b200.compression.attn_tables import calibrate, device_tables
from fragpack_b200.integrations.vllm.backend import (
    FragPackMetadata,
    HeadTransform,
    count_closes,
    plan_prefill_groups,
    run_layer,
)
from fragpack_b200.ops.fused_attn_decode import RecordTables, decode_units, workspace_elems
from fragpack_b200.ops.hbm_kv import HbmKvStore, page_bytes
from fragpack_b200.ops.prompt_attn import prompt_status
from fragpack_b200.ops.rotary import make_rotary, norm_rotary

pytestmark = pytest.mark.gpu

L, H, G, D, T, NB = 2, 2, 4, 128, 128, 24
HQ, SCALE, MAX_TOKENS, PAGES = H * G, D**-0.5, 1024, 8


class Request:
    def __init__(self, blocks):
        self.blocks, self.computed = blocks, 0
        self.history = [(torch.zeros(0, H, D), torch.zeros(0, H, D)) for _ in range(L)]


def _reference(q, k, v):
    """fp32 causal attention of the last rows; q [n, HQ, D], k / v [ctx, H, D]."""
    n, ctx = q.shape[0], k.shape[0]
    kk, vv = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    logits = torch.einsum("nhd,thd->hnt", q, kk) * SCALE
    hidden = torch.arange(ctx)[None, :] > torch.arange(ctx - n, ctx)[:, None]
    return torch.einsum("hnt,thd->nhd", logits.masked_fill(hidden, float("-inf")).softmax(-1), vv)


def _run(fused_append: bool, over_prompt: bool, split: bool = False, norms: bool = True):
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator().manual_seed(43)
    sample = (torch.randn(8, L, 2, T, H, D, generator=gen) * 0.5).to(torch.bfloat16)
    table = calibrate(sample.view(torch.int16).numpy().view(np.uint16))
    caches = [torch.zeros(NB, page_bytes(H), dtype=torch.uint8, device=device) for _ in range(L)]
    store = HbmKvStore(caches, H, device_tables(table, device), MAX_TOKENS, staging_slots=3, overflow_records=64)
    layer_tables = [RecordTables(*store.layer_tables(i)) for i in range(L)]
    sms = torch.cuda.get_device_properties(device).multi_processor_count
    sizes = workspace_elems(H, decode_units(3, H, sms))
    workspace = (torch.empty(sizes[0], device=device), torch.empty(sizes[1], device=device),
                 torch.empty(sizes[2], dtype=torch.int32, device=device))
    wk = torch.empty(PAGES, T, H, D, dtype=torch.bfloat16, device=device)
    rotary = make_rotary(device, base=500000.0)
    weights = (torch.rand(L, 2, D, generator=gen) * 0.2 + 0.4).to(device) if norms else [(None, None)] * L
    a, b, c = Request([3, 7, 1, 9, 11]), Request([5, 2, 8, 4]), Request([20, 13, 6])
    steps = [
        [(a, 300), (b, 77)],           # whole prompts, one group
        [(a, 1), (b, 1), (c, 1)],      # two decodes and a prompt of one token
        [(a, 1), (b, 60), (c, 200)],   # a decode and chunks over cached blocks
        [(a, 1), (b, 1), (c, 1)],
    ]
    outputs = []
    for rows in steps:
        decodes = [(r, n) for r, n in rows if n == 1 and r.computed > 0]
        ordered = decodes + [(r, n) for r, n in rows if not (n == 1 and r.computed > 0)]
        nd, num = len(decodes), len(ordered)
        qlen = np.array([n for _, n in ordered], np.int64)
        seq = np.array([r.computed + n for r, n in ordered], np.int64)
        qsl = np.concatenate(([0], np.cumsum(qlen)))
        total = int(qsl[-1])
        pos = np.concatenate([np.arange(r.computed, r.computed + n) for r, n in ordered])
        slots = np.concatenate([[r.blocks[p // T] * T + p % T for p in range(r.computed, r.computed + n)]
                                for r, n in ordered])
        slot_t, pos_t = torch.from_numpy(slots).to(device), torch.from_numpy(pos).to(device)
        blocks = torch.zeros(num, 5, dtype=torch.int32)
        for i, (r, _) in enumerate(ordered):
            blocks[i, : len(r.blocks)] = torch.tensor(r.blocks)
        blocks = blocks.to(device)
        live = np.array([r.blocks[r.computed // T] for r, _ in ordered if r.computed % T], np.int32)
        store.prepare(slot_t, total, live)
        md = FragPackMetadata(
            store=store, layer_tables=layer_tables, layer_index={}, last_layer=L - 1, slot_mapping=slot_t,
            num_tokens=total, num_decodes=nd, decode_block_table=blocks[:nd],
            decode_seq_lens=torch.from_numpy(seq[:nd].astype(np.int32)).to(device),
            units=decode_units(max(nd, 1), H, sms), decode_workspace=workspace,
            max_close=min(max(count_closes(seq, qlen), nd), MAX_TOKENS),
            prefills=plan_prefill_groups(blocks, nd, num, qsl, seq, PAGES, device, split) if num > nd else [],
            wk=wk, wv=torch.empty_like(wk), prompt_attention=over_prompt,
        )
        for layer in range(L):
            qkv = torch.randn(total, HQ + 2 * H, D, generator=gen).mul(0.5).to(torch.bfloat16).to(device)
            q, k, v = qkv[:, :HQ], qkv[:, HQ : HQ + H], qkv[:, HQ + H :]
            wq, wk_ = weights[layer]
            ready_q, ready_k = torch.empty_like(q), torch.empty_like(k)
            norm_rotary(q, k, pos_t, rotary, ready_q, ready_k, wq, wk_)
            out = torch.full((total, HQ, D), float("nan"), dtype=torch.bfloat16, device=device)
            run_layer(md, layer, q, k, v, out, SCALE, transform=HeadTransform(rotary, pos_t, wq, wk_),
                      fused_append=fused_append)
            outputs.append(out)
            assert torch.equal(q, ready_q)
            for i, (r, n) in enumerate(ordered):
                t0, t1 = int(qsl[i]), int(qsl[i + 1])
                hk, hv = (torch.cat([old, new[t0:t1].float().cpu()])
                          for old, new in zip(r.history[layer], (ready_k, v)))
                r.history[layer] = (hk, hv)
                err = (out[t0:t1].float().cpu() - _reference(ready_q[t0:t1].float().cpu(), hk, hv)).abs()
                assert float(err.max()) <= 1e-2 and float(err.mean()) <= 2e-3, (layer, i, n)
        for r, n in ordered:
            r.computed += n
    stats = store.stats()
    assert stats.err_staging == 0 and stats.err_overflow == 0 and prompt_status() == 0
    # The closed blocks of a (301..), b (137) and c (201 tokens): two, one and one.
    assert stats.encoded == 4 * L * 2 * H
    pages = torch.empty(4, T, H, D, dtype=torch.bfloat16, device=device)
    held = []
    for layer in range(L):
        values = torch.empty_like(pages)
        store.gather(layer, torch.tensor([3, 7, 5, 20], dtype=torch.int32, device=device), pages, values)
        held += [pages.clone(), values]
    return outputs, held


@pytest.mark.parametrize("over_prompt,split", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("norms", [True, False])
def test_layers_from_projected_heads(over_prompt, split, norms) -> None:
    fused, held = _run(True, over_prompt, split, norms)
    steps, also_held = _run(False, over_prompt, split, norms)
    assert all(torch.equal(x, y) for x, y in zip(fused, steps))
    assert all(torch.equal(x, y) for x, y in zip(held, also_held))


def test_prompts_over_their_own_keys_equal_prompts_over_records_to_rounding() -> None:
    direct, held = _run(True, True)
    records, also_held = _run(True, False)
    assert all(torch.equal(x, y) for x, y in zip(held, also_held))
    for x, y in zip(direct, records):
        assert float((x.float() - y.float()).abs().max()) <= 1e-2


def test_operators_chained_in_one_captured_graph() -> None:
    """append -> prompt_attention, two graphs over the same store, replayed in turn on new inputs."""
    device = torch.device("cuda", torch.cuda.current_device())
    table = np.broadcast_to(np.arange(22, dtype=np.uint8), (1, 2, H, 22)).copy()
    arena = [torch.zeros(NB, page_bytes(H), dtype=torch.uint8, device=device)]
    store = HbmKvStore(arena, H, device_tables(table, device), MAX_TOKENS, staging_slots=NB, overflow_records=4)
    rotary, n = make_rotary(device), 500
    slots = torch.arange(n, device=device)
    positions = torch.arange(n, device=device, dtype=torch.int32)
    starts = torch.tensor([0, 333, n], dtype=torch.int32, device=device)
    store.prepare(slots, n, np.arange(4, dtype=np.int32))
    from fragpack_b200.ops.prompt_attn import prompt_attention

    def layer(buf, out):
        q, k, v = buf[:, :HQ], buf[:, HQ : HQ + H], buf[:, HQ + H :]
        store.append(0, q, k, v, positions, slots, rotary, q, k)
        prompt_attention(q, k, v, starts, SCALE, out)

    gen = torch.Generator(device="cuda").manual_seed(1)
    fresh = [torch.randn(n, HQ + 2 * H, D, generator=gen, device=device).to(torch.bfloat16) for _ in range(2)]
    want = []
    for x in fresh:
        buf, out = x.clone(), torch.zeros(n, HQ, D, dtype=torch.bfloat16, device=device)
        layer(buf, out)
        want.append((out, store.scratch.clone(), store.staging.clone()))
    bufs = [x.clone() for x in fresh]
    outs = [torch.zeros_like(want[0][0]) for _ in fresh]
    graphs = [torch.cuda.CUDAGraph() for _ in fresh]
    for g, buf, out in zip(graphs, bufs, outs):
        with torch.cuda.graph(g):
            layer(buf, out)
    for turn in (0, 1, 1, 0):
        bufs[turn].copy_(fresh[turn])
        outs[turn].zero_()
        graphs[turn].replay()
        assert torch.equal(outs[turn], want[turn][0])
        assert torch.equal(store.scratch, want[turn][1]) and torch.equal(store.staging, want[turn][2])
