"""Causal attention of packed whole prompts over BF16 keys and values (sm_100a, tcgen05).

A prompt's first prefill step attends only to keys and values that the same
step has just produced.  :func:`prompt_attention` reads them where they are,
in the layer's projection, instead of the store: no record is decoded and no
workspace is filled (the reference sends such a step through ``store.gather``
and FlashAttention like any other, ``fragpack/integrations/vllm/backend.py:560-575``;
:func:`fragpack_b200.ops.prefill_attn.prefill_attention` serves the steps that
also see cached blocks).
"""

from __future__ import annotations

import ctypes

import torch

from fragpack_b200.ops.fragpack_ext import check, extension, on_device, require_cuda, stream_ptr
from fragpack_b200.ops.fused_attn_decode import GQA

PROMPT_WAIT_TIMEOUT = 1
LONGEST_LAG = 8.0


def prompt_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    starts: torch.Tensor,
    scale: float,
    out: torch.Tensor,
    lag: float = LONGEST_LAG,
) -> None:
    """Attend every prompt's tokens over itself, causally.

    Prompt ``r`` owns the rows ``starts[r] .. starts[r + 1]`` of all four
    tensors; each of its rows sees the prompt's rows up to and including
    itself.  Rows outside every prompt are left as they were, and what they
    hold reaches no result.  Infinities and NaN reach the rows that see them and
    no others, and those of ``v`` take no more time than other values.  Values up
    to BF16's largest are summed in range; those below about 2**-85 lose bits, as
    weighted sums start at 2**-126.

    Args:
        q: BF16 ``[T, H * G, 128]`` queries.
        k, v: BF16 ``[T, H, 128]`` keys and values.  Tokens and heads of all
            tensors may be strided by 16-byte multiples.
        starts: int32 ``[R + 1]`` first row of each prompt, non-decreasing;
            entries are clamped to ``0 .. T``.
        scale: Softmax scale, positive (times log2(e) a normal FP32 number).
        out: BF16 ``[T, H * G, 128]`` output; must not overlap the inputs.
        lag: Precision of the BF16 weights, 0 to ``LONGEST_LAG``: how far (in
            powers of two) a row's largest score may rise above the reference
            point of its weights before that follows.  At 0 the largest weight
            is an exact 1, as in ``prefill_attention``; the RMS error is then
            1.08 to 1.12 times that of FP32 attention rounded once, against
            1.16 to 1.34 at the default, and a call takes 1 to 20 % longer.

    Raises:
        ValueError: If the query group does not divide ``GQA``.
        RuntimeError: For rejected arguments or a failed launch.

    Async/thread-safety:
        One kernel on the current CUDA stream; CUDA-graph safe; allocates nothing.
    """
    device = q.get_device()
    if device < 0:
        require_cuda(q, "q")
    q_shape, kv_shape = q.shape, k.shape
    if len(q_shape) != 3 or len(kv_shape) != 3 or kv_shape[1] == 0:
        raise RuntimeError("q, k and v must be [T, heads, 128]")
    tokens, kv_heads = kv_shape[0], kv_shape[1]
    group = q_shape[1] // kv_heads
    if group == 0 or group * kv_heads != q_shape[1] or GQA % group:
        raise ValueError(f"query heads {q_shape[1]} need a group dividing {GQA}")
    if kv_shape[2] != 128 or v.shape != kv_shape or q_shape[0] != tokens or q_shape[2] != 128:
        raise RuntimeError("q must be [T, H * G, 128] and k, v [T, H, 128]")
    if out.shape != q_shape:
        raise RuntimeError("out must have the shape of q")
    rows = []
    for t in (q, k, v, out):
        stride = t.stride()
        if t.dtype is not torch.bfloat16 or t.get_device() != device or stride[2] != 1:
            raise RuntimeError(f"q, k, v and out must be bfloat16 on cuda:{device} with a contiguous head dim")
        rows.append((t.data_ptr(), stride[0], stride[1]))
    if starts.dtype is not torch.int32 or starts.dim() != 1 or not starts.is_contiguous() or starts.numel() == 0:
        raise RuntimeError("starts must be contiguous int32 [R + 1]")
    if starts.get_device() != device:
        raise RuntimeError(f"starts must be on cuda:{device}")
    with on_device(device):
        check(
            extension().fp_prompt_attention_lag(
                *rows[0], *rows[1], *rows[2], starts.data_ptr(), starts.shape[0] - 1, tokens, *rows[3], kv_heads,
                group, scale, lag, stream_ptr(),
            )
        )


def prompt_status() -> int:
    """Status word of the prompt kernel on the current device (synchronises) and clear it.

    Returns:
        0, or ``PROMPT_WAIT_TIMEOUT`` if a bounded device-side wait ran out
        since the last read (the outputs of those calls are invalid).
    """
    word = ctypes.c_int32(0)
    check(extension().fp_prompt_status(ctypes.byref(word)))
    return int(word.value)


__all__ = ["LONGEST_LAG", "PROMPT_WAIT_TIMEOUT", "prompt_attention", "prompt_status"]
