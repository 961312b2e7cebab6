"""Cases and plain forms of the operators between a layer's QKV projection and its attention output.

Three operators: ``norm_rotary`` (RMS norm of every query and key head and the position rotation in one pass),
``HbmKvStore.append`` (the same, and the new keys and values go to their places in the paged store's staging records on
the way) and ``prompt_attention`` (causal attention of packed whole prompts over the keys and values at hand).

``run`` computes them in elementary torch operations in 32 bits (angles in 64), or, where ``own`` is true, by the calls
that a user of ``fragpack_b200`` makes.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DIM = 128  # head dimension of the framework's records
BLOCK = 128  # tokens of a block
EPS = 1e-6
# Parameters of the two band-wise frequency scalings.
BANDS = {"factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original": 8192}
RAMP = {"factor": 4.0, "original": 8192, "beta_fast": 32.0, "beta_slow": 1.0}


# ---------------------------------------------------------------------------- cases


def _rotary(name, tokens, q_heads, kv_heads, *, rot_dim, interleaved, scaling, norms, decode, context, base=500000.0):
    return {"name": name, "op": "norm_rotary", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "rot_dim": rot_dim, "interleaved": interleaved, "scaling": scaling, "norms": norms, "decode": decode,
            "context": context, "base": base}


def _append(name, rows, shortest, longest, first, q_heads, kv_heads, *, rot_dim=128, interleaved=False, scaling="none",
            norms=True, keep_keys=False, base=1000000.0, lens_seed=1):
    return {"name": name, "op": "append", "rows": rows, "shortest": shortest, "longest": longest, "first": first,
            "lens_seed": lens_seed, "q_heads": q_heads, "kv_heads": kv_heads, "rot_dim": rot_dim,
            "interleaved": interleaved, "scaling": scaling, "norms": norms, "keep_keys": keep_keys, "base": base}


def _prompts(name, rows, shortest, longest, q_heads, kv_heads, lens_seed=1):
    return {"name": name, "op": "prompt", "rows": rows, "shortest": shortest, "longest": longest,
            "lens_seed": lens_seed, "q_heads": q_heads, "kv_heads": kv_heads}


def listed():
    """Geometries of the repository's benchmark configurations (query heads / KV heads, batch, context)."""
    return [
        # One decode step of four sequences, a model with norms of its query and key heads: launch latency only.
        _rotary("rotary decode 4", 4, 32, 4, rot_dim=128, interleaved=False, scaling="none", norms=True, decode=True,
                context=8192, base=1000000.0),
        # An odd decode batch with the older layout: neighbouring pairs, half of the head, positions interpolated.
        _rotary("rotary batch 131 part", 131, 32, 8, rot_dim=64, interleaved=True, scaling="linear", norms=False,
                decode=True, context=32768, base=10000.0),
        # A prefill step of the 64-query-head geometry at far positions, frequencies scaled by wavelength.
        _rotary("rotary prefill 16384", 16384, 64, 8, rot_dim=128, interleaved=False, scaling="bands", norms=False,
                decode=False, context=32768),
        # The smallest store append: one sequence decodes one token.
        _append("append decode 1", 1, 1, 1, 8191, 32, 4),
        # The largest decode batch of the configurations.
        _append("append decode 128", 128, 1, 1, 32767, 64, 8, norms=False, scaling="bands", base=500000.0),
        # Ragged prefill chunks that continue open blocks from odd offsets.
        _append("append chunks ragged", 7, 1, 700, 333, 32, 8, norms=False, scaling="ramp"),
        # Two whole prompts of the prefill configuration (as many KV heads as query heads); the rotated keys are kept
        # for the prompt's own attention.
        _append("append prompts mha", 2, 8192, 8192, 0, 32, 32, keep_keys=True),
        # One short prompt: latency.
        _prompts("prompt 77", 1, 77, 77, 32, 4),
        # A batch of short questions of every length up to 300, one-token ones among them.
        _prompts("prompts short 64", 64, 1, 300, 32, 4),
        # The ragged configuration's lengths.
        _prompts("prompts ragged 16", 16, 1000, 4096, 32, 8),
        # Two prompts of the prefill configuration, one query head per KV head.
        _prompts("prompts mha 2x8192", 2, 8192, 8192, 32, 32),
        # The longest context, one rank's eighth of the 64-query-head geometry.
        _prompts("prompt 32768 shard", 1, 32768, 32768, 8, 1),
    ]


HEADS = [(32, 4), (32, 8), (64, 8), (16, 4), (8, 1), (32, 32), (16, 8)]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    q_heads, kv_heads = rng.choice(HEADS)
    op = rng.choice(("norm_rotary", "append", "prompt", "prompt"))
    layout = {"rot_dim": rng.choice((32, 64, 96, 128, 128)), "interleaved": rng.random() < 0.4,
              "scaling": rng.choice(("none", "linear", "bands", "ramp")), "norms": rng.random() < 0.5}
    if op == "norm_rotary":
        tokens = _log_uniform(rng, 1, 16384 * 72 // (q_heads + kv_heads) // 2)
        c = _rotary("", tokens, q_heads, kv_heads, decode=rng.random() < 0.4, context=max(tokens, rng.randrange(1, 131072)),
                    base=rng.choice((10000.0, 500000.0, 1000000.0)), **layout)
    elif op == "append":
        total = _log_uniform(rng, 1, 16384 * 64 // (q_heads + 2 * kv_heads) // 2)
        rows = min(total, _log_uniform(rng, 1, 128))
        longest = max(1, total // rows)
        first = rng.choice((0, rng.randrange(0, 32768)))
        c = _append("", rows, max(1, longest // rng.choice((1, 2, 50))), longest, first, q_heads, kv_heads,
                    keep_keys=rng.random() < 0.5, lens_seed=rng.randrange(1 << 20),
                    base=rng.choice((10000.0, 1000000.0)), **layout)
    else:
        rows = _log_uniform(rng, 1, 64)
        # The pairs of all heads stay below the largest listed case's.
        most = int(math.sqrt(32768 * 32768 * 8 / 2 / rows / q_heads))
        longest = _log_uniform(rng, 1, min(most, 32768))
        c = _prompts("", rows, max(1, longest // rng.choice((1, 4, 1000))), longest, q_heads, kv_heads,
                     rng.randrange(1 << 20))
    del c["name"]
    return c


def _lens(case):
    rng = random.Random(case["lens_seed"])
    return [rng.randint(case["shortest"], case["longest"]) for _ in range(case["rows"])]


def work(case):
    hq, h = case["q_heads"], case["kv_heads"]
    if case["op"] == "norm_rotary":
        n = case["tokens"]
        return {"bytes": n * (4 * DIM * (hq + h) + 8), "flops": n * (hq + h) * DIM * (7 if case["norms"] else 3)}
    n = sum(_lens(case))
    if case["op"] == "append":
        kept = 2 * DIM * h if case["keep_keys"] else 0
        return {"bytes": n * (4 * DIM * (hq + 2 * h) + kept + 16),
                "flops": n * (hq + h) * DIM * (7 if case["norms"] else 3)}
    pairs = sum(m * (m + 1) // 2 for m in _lens(case))
    return {"bytes": n * 2 * DIM * (2 * hq + 2 * h), "flops": 4 * DIM * hq * pairs}


# ---------------------------------------------------------------------------- inputs


def _projection(case, tokens, seed):
    """The packed QKV projection of a step: BF16 [T, Hq + 2 H, 128]; channel scales and K outliers as in real caches."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    hq, h = case["q_heads"], case["kv_heads"]
    qkv = torch.randn(tokens, hq + 2 * h, DIM, generator=gen, device="cuda")
    scales = torch.exp(0.5 * torch.randn(2 * h, DIM, generator=gen, device="cuda"))
    scales[:h, torch.randperm(DIM, generator=gen, device="cuda")[:4]] *= 8.0
    qkv[:, hq:] *= scales
    return qkv.to(torch.bfloat16), gen


def _inverse_frequencies(case):
    """Radians per token of every rotated pair, in 64 bits, and the factor on the rotated values."""
    rot, base = case["rot_dim"], case["base"]
    freq = base ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if case["scaling"] == "linear":
        return freq / 4.0, 1.0
    if case["scaling"] == "bands":
        turns = BANDS["original"] * freq / (2 * np.pi)  # rotations over the original context
        low, high = BANDS["low_freq_factor"], BANDS["high_freq_factor"]
        keep = np.clip((turns - low) / (high - low), 0.0, 1.0)
        return freq * keep + freq / BANDS["factor"] * (1.0 - keep), 1.0
    if case["scaling"] == "ramp":
        def pair_of(rotations):
            return rot * math.log(RAMP["original"] / (rotations * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(pair_of(RAMP["beta_fast"])), 0)
        high = min(math.ceil(pair_of(RAMP["beta_slow"])), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - low) / max(high - low, 1e-3), 0.0, 1.0)
        return freq * (1 - ramp) + freq / RAMP["factor"] * ramp, 0.1 * math.log(RAMP["factor"]) + 1.0
    return freq, 1.0


def _own_rotary(case):
    from fragpack_b200.ops.rotary import make_rotary

    scaling = {"none": None, "linear": {"type": "linear", "factor": 4.0}, "bands": {"type": "bands", **BANDS},
               "ramp": {"type": "ramp", **RAMP}}[case["scaling"]]
    return make_rotary(torch.device("cuda"), rot_dim=case["rot_dim"], base=case["base"],
                       interleaved=case["interleaved"], scaling=scaling)


def _append_plan(case):
    """Positions, slots and the staged blocks of an append: rows own disjoint runs of blocks, in row order."""
    lens = _lens(case)
    rng = random.Random(case["lens_seed"] + 1)
    first = [case["first"] - (rng.randrange(0, min(case["first"], 127) + 1) if case["rows"] > 1 else 0) for _ in lens]
    positions, slots, blocks, used = [], [], [], 0
    for n, p0 in zip(lens, first):
        p = np.arange(p0, p0 + n, dtype=np.int64)
        touched = int(p[-1] // BLOCK - p[0] // BLOCK) + 1
        slots.append(p - p0 // BLOCK * BLOCK + used * BLOCK)
        positions.append(p)
        blocks += range(used, used + touched)
        used += touched
    return np.concatenate(positions), np.concatenate(slots), len(blocks)


def _store_with_open_blocks(kv_heads, blocks):
    """A one-layer store in which block b sits in staging slot blocks - 1 - b (claimed in order, 32 at a time)."""
    from fragpack_b200.compression.attn_tables import device_tables
    from fragpack_b200.ops.hbm_kv import HbmKvStore, page_bytes

    device = torch.device("cuda", torch.cuda.current_device())
    table = np.broadcast_to(np.arange(22, dtype=np.uint8), (1, 2, kv_heads, 22)).copy()
    arena = torch.empty(blocks, page_bytes(kv_heads), dtype=torch.uint8, device=device)
    store = HbmKvStore([arena], kv_heads, device_tables(table, device), max_tokens=128, staging_slots=blocks,
                       overflow_records=1)
    for b0 in range(0, blocks, 32):
        b1 = min(b0 + 32, blocks)
        slots = torch.arange(b0, b1, device=device) * BLOCK
        store.prepare(slots, b1 - b0, np.arange(b0, dtype=np.int32))
    return store, arena


def prepare(case, seed):
    hq, h = case["q_heads"], case["kv_heads"]
    if case["op"] == "prompt":
        lens = _lens(case)
        qkv, _ = _projection(case, sum(lens), seed)
        starts = torch.tensor(np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32, device="cuda")
        return {"case": case, "q": qkv[:, :hq], "k": qkv[:, hq:hq + h], "v": qkv[:, hq + h:], "starts": starts,
                "lens": lens, "out": torch.zeros(sum(lens), hq, DIM, dtype=torch.bfloat16, device="cuda")}
    if case["op"] == "append":
        positions, slots, blocks = _append_plan(case)
        tokens = len(positions)
    else:
        tokens = case["tokens"]
    qkv, gen = _projection(case, tokens, seed)
    if case["op"] == "append":
        positions = torch.from_numpy(positions).cuda()
    elif case["decode"]:
        positions = torch.randint(0, case["context"], (tokens,), generator=gen, device="cuda")
    else:
        positions = torch.arange(case["context"] - tokens, case["context"], device="cuda")
    state = {"case": case, "q": qkv[:, :hq], "k": qkv[:, hq:hq + h], "v": qkv[:, hq + h:], "positions": positions,
             "q_weight": None, "k_weight": None,
             "query_out": torch.zeros(tokens, hq, DIM, dtype=torch.bfloat16, device="cuda"),
             "key_out": torch.zeros(tokens, h, DIM, dtype=torch.bfloat16, device="cuda")}
    if case["norms"]:
        weights = 1.0 + 0.3 * torch.randn(2, DIM, generator=gen, device="cuda")
        state["q_weight"], state["k_weight"] = weights.to(torch.bfloat16).unbind(0)
    freq, factor = _inverse_frequencies(case)
    state["freq"], state["factor"] = torch.from_numpy(freq).cuda(), factor
    if case["op"] == "append":
        state["slots"] = torch.from_numpy(slots).cuda()
        state["blocks"] = blocks
        if own:
            state["store"], state["arena"] = _store_with_open_blocks(h, blocks)
            state["staging"] = state["store"].staging.view(torch.bfloat16).view(blocks, 2, h, BLOCK * DIM)
        else:
            state["staging"] = torch.zeros(blocks, 2, h, BLOCK * DIM, dtype=torch.bfloat16, device="cuda")
            state["places"] = torch.from_numpy(np.stack((_key_places(), _value_places()))).cuda()
    if own:
        state["rotary"] = _own_rotary(case)
    return state


def _key_places():
    """Where token `t`, dim `d` of a block stands in its raw K record (scalars): [128, 128]."""
    t, d = np.arange(BLOCK)[:, None], np.arange(DIM)[None, :]
    owner = 32 * (t // 16) + 4 * (t % 8) + d // 2 % 4
    return 8 * (256 * (d // 16) + owner) + 4 * (t // 8 % 2) + 2 * (d // 8 % 2) + d % 2


def _value_places():
    """The same for a V record, where tokens and dims change roles."""
    t, d = np.arange(BLOCK)[:, None], np.arange(DIM)[None, :]
    owner = 32 * (d // 16) + 4 * (d % 8) + t // 2 % 4
    return 8 * (256 * (t // 16) + owner) + 4 * (d // 8 % 2) + 2 * (t // 8 % 2) + t % 2


# ---------------------------------------------------------------------------- plain forms


def _norm_and_rotate(x, weight, cos, sin, interleaved):
    """x [T, heads, 128] -> 32-bit values, unrounded; cos / sin [T, 1, rot / 2]."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos.shape[-1]
    turned, rest = x[..., : 2 * half], x[..., 2 * half :]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _plain_rotary(s):
    angle = s["positions"].double()[:, None] * s["freq"]
    cos = (angle.cos() * s["factor"]).float()[:, None]
    sin = (angle.sin() * s["factor"]).float()[:, None]
    layout = s["case"]["interleaved"]
    return (_norm_and_rotate(s["q"], s["q_weight"], cos, sin, layout).to(torch.bfloat16),
            _norm_and_rotate(s["k"], s["k_weight"], cos, sin, layout).to(torch.bfloat16))


def _plain_append(s):
    query, key = _plain_rotary(s)
    staging, kv_heads = s["staging"], s["case"]["kv_heads"]
    block, offset = s["slots"] // BLOCK, s["slots"] % BLOCK
    record = (s["blocks"] - 1 - block)[:, None] * 2 * kv_heads + torch.arange(kv_heads, device="cuda")
    base = record[..., None] * (BLOCK * DIM)
    flat = staging.view(-1)
    flat[base + s["places"][0][offset][:, None]] = key
    flat[base + kv_heads * BLOCK * DIM + s["places"][1][offset][:, None]] = s["v"]
    out = {"query": query, "staging": staging}
    return {**out, "key": key} if s["case"]["keep_keys"] else out


def _padded(x, starts, longest):
    """Packed [T, heads, 128] -> [R, heads, longest, 128] in 32 bits (rows past a prompt hold its neighbours)."""
    at = (starts[:-1, None].long() + torch.arange(longest, device="cuda")).clamp(max=x.shape[0] - 1)
    return x[at].transpose(1, 2).float()


def _plain_prompts(s):
    starts, longest, group = s["starts"], max(s["lens"]), s["case"]["q_heads"] // s["case"]["kv_heads"]
    at = torch.arange(longest, device="cuda")
    hidden = at[None, :] > at[:, None]
    length = starts[1:] - starts[:-1]
    real = (at < length[:, None]).nonzero(as_tuple=True)
    out = torch.empty_like(s["out"])
    # As many query heads at a time as keep the scores below 8 GB.
    step = max(1, (1 << 31) // (len(s["lens"]) * longest * longest))
    for h0 in range(0, s["case"]["q_heads"], step):
        heads = torch.arange(h0, min(h0 + step, s["case"]["q_heads"]), device="cuda")
        q = _padded(s["q"][:, heads], starts, longest)
        k = _padded(s["k"][:, heads // group], starts, longest)
        v = _padded(s["v"][:, heads // group], starts, longest)
        p = torch.matmul(q, k.transpose(2, 3)).mul_(DIM**-0.5).masked_fill_(hidden, -math.inf)
        p.sub_(p.amax(-1, keepdim=True)).exp_()
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[:, h0 : h0 + step] = o.transpose(1, 2)[real].to(torch.bfloat16)
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_run(state, op)
    if op == "norm_rotary":
        return _plain_rotary(state)
    return _plain_append(state) if op == "append" else _plain_prompts(state)


def _own_run(s, op):
    if op == "prompt":
        from fragpack_b200.ops.prompt_attn import prompt_attention

        prompt_attention(s["q"], s["k"], s["v"], s["starts"], DIM**-0.5, s["out"])
        return s["out"]
    if op == "norm_rotary":
        from fragpack_b200.ops.rotary import norm_rotary

        norm_rotary(s["q"], s["k"], s["positions"], s["rotary"], s["query_out"], s["key_out"], s["q_weight"],
                    s["k_weight"], EPS)
        return s["query_out"], s["key_out"]
    keep = s["case"]["keep_keys"]
    s["store"].append(0, s["q"], s["k"], s["v"], s["positions"], s["slots"], s["rotary"], s["query_out"],
                      s["key_out"] if keep else None, s["q_weight"], s["k_weight"], EPS)
    out = {"query": s["query_out"], "staging": s["staging"]}
    return {**out, "key": s["key_out"]} if keep else out


# ---------------------------------------------------------------------------- definitions in 64 bits


def _exact_heads(case, x, weight, positions):
    """[T, heads, 128] in 64 bits: each pair as a complex number times factor * exp(i position frequency)."""
    freq, factor = _inverse_frequencies(case)
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / DIM + EPS).sqrt() * weight.double()
    rot, half = case["rot_dim"], case["rot_dim"] // 2
    first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)
    turn = torch.polar(torch.full((1, 1), factor, dtype=torch.float64, device="cuda"),
                       positions.double()[:, None] * torch.from_numpy(freq).cuda())
    pair = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    y = x.clone()
    y[..., first], y[..., second] = pair.real, pair.imag
    return y


def _exact_staging(case, key, value, slots, blocks):
    """Records of the open blocks, in slot order, from token-major blocks by reordering their axes."""
    h = case["kv_heads"]
    pages = torch.zeros(2, blocks * BLOCK, h, DIM, dtype=torch.float64, device="cuda")
    pages[0, slots], pages[1, slots] = key, value.double()
    pages = pages.view(2, blocks, BLOCK, h, DIM).flip(1)  # block b is staged in slot blocks - 1 - b
    # token = (row group, j, g), dim = (word, f, c, e) of a K record; exchanged in a V record.
    k = pages[0].reshape(blocks, 8, 2, 8, h, 8, 2, 4, 2).permute(0, 4, 5, 1, 3, 7, 2, 6, 8)
    v = pages[1].reshape(blocks, 8, 2, 4, 2, h, 8, 2, 8).permute(0, 5, 1, 6, 8, 3, 7, 2, 4)
    return torch.stack((k.reshape(blocks, h, -1), v.reshape(blocks, h, -1)), 1)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] != "prompt":
        query = _exact_heads(case, s["q"], s["q_weight"], s["positions"])
        key = _exact_heads(case, s["k"], s["k_weight"], s["positions"])
        if case["op"] == "norm_rotary":
            return query, key
        out = {"query": query, "staging": _exact_staging(case, key, s["v"], s["slots"], s["blocks"])}
        return {**out, "key": key} if case["keep_keys"] else out
    # Row blocks of one prompt and one KV head at a time, only the keys that they see.
    out, group = torch.empty(s["out"].shape, dtype=torch.float64, device="cuda"), case["q_heads"] // case["kv_heads"]
    t0 = 0
    for n in s["lens"]:
        for h in range(case["kv_heads"]):
            k, v = s["k"][t0 : t0 + n, h].double(), s["v"][t0 : t0 + n, h].double()
            heads = slice(h * group, (h + 1) * group)
            for r0 in range(0, n, 2048):
                r1 = min(r0 + 2048, n)
                q = s["q"][t0 + r0 : t0 + r1, heads].double()
                logits = torch.einsum("rgd,td->rgt", q, k[:r1]) / math.sqrt(DIM)
                later = torch.arange(r1, device="cuda") > torch.arange(r0, r1, device="cuda")[:, None, None]
                weights = torch.softmax(logits.masked_fill(later, -math.inf), -1)
                out[t0 + r0 : t0 + r1, heads] = torch.einsum("rgt,td->rgd", weights, v[:r1])
        t0 += n
    return out
