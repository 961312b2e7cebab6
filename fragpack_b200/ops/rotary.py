"""Norms of query and key heads with the position rotation, one pass (sm_100a).

What a decoder layer does to its projected heads before they meet the cache:
an optional RMS norm of every query and key head and the rotation by the
token's position.  :func:`norm_rotary` does it for callers that hand rotated
heads to the attention backend (whose ``forward`` writes the keys itself, as
the reference's, ``fragpack/integrations/vllm/backend.py:504-579``);
``HbmKvStore.append`` does the same on the way into the store.  The reference
has no counterpart: its engine rotates before the backend is called.

A :class:`Rotary` holds the frequencies in turns per token as 64-bit binary
fractions: ``position * frequency`` modulo one turn is one integer product,
which adds no error at any position, and no table of angles is kept.  The
fractions are as good as float64 frequencies: within 2**-54 turns per token up
to one radian per token.
"""

from __future__ import annotations

from ctypes import byref
from dataclasses import dataclass, field
import math
from typing import Any

import numpy as np
import torch

from fragpack_b200.ops.fragpack_ext import (
    FpRotary,
    check,
    extension,
    on_device,
    pack_heads,
    require_cuda,
    stream_ptr,
)

HEAD_DIM = 128
_BF16, _FP32, _INT64, _INT32 = torch.bfloat16, torch.float32, torch.int64, torch.int32


def rotary_frequencies(
    rot_dim: int = HEAD_DIM, base: float = 10000.0, scaling: dict[str, Any] | None = None
) -> tuple[np.ndarray, float]:
    """Frequencies of the rotated pairs and the factor on the rotated dims.

    Pair ``i`` turns by ``base ** (-2 i / rot_dim)`` radians per token.  For
    contexts longer than the model was trained on, ``scaling`` names a rule:

    * ``{"type": "linear", "factor"}``: every frequency divided by ``factor``
      (positions interpolated);
    * ``{"type": "bands", "factor", "low_freq_factor", "high_freq_factor",
      "original"}``: pairs that turn at least ``high_freq_factor`` times over
      the ``original`` context keep their frequency, those that turn at most
      ``low_freq_factor`` times are divided by ``factor``, linear in the
      number of turns in between;
    * ``{"type": "ramp", "factor", "original", "beta_fast", "beta_slow"}``:
      the same idea, linear in the pair's index between the pairs that turn
      ``beta_fast`` (default 32) and ``beta_slow`` (default 1) times, and the
      rotated dims are multiplied by ``"attention_factor"`` (default
      ``0.1 ln(factor) + 1``).

    Args:
        rot_dim: Rotated dims, even.
        base: Base of the geometric progression.
        scaling: A rule as above, or None.

    Returns:
        float64 ``[rot_dim / 2]`` radians per token, and the factor.

    Raises:
        ValueError: For an unknown rule or impossible parameters.
    """
    if rot_dim < 0 or rot_dim % 2 or not 1.0 < base < math.inf:
        raise ValueError(f"rotated dims {rot_dim} must be even and the base {base} above 1")
    freq = base ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / max(rot_dim, 1))
    if scaling is None:
        return freq, 1.0
    rule, factor = scaling.get("type"), float(scaling.get("factor", 0.0))
    if rule not in ("linear", "bands", "ramp"):
        raise ValueError(f"unknown rotary scaling {rule!r}")
    if not 1.0 <= factor < math.inf:
        raise ValueError(f"rotary scaling needs a factor of at least 1, not {factor}")
    if rule == "linear":
        return freq / factor, 1.0
    needed = ("original", "low_freq_factor", "high_freq_factor") if rule == "bands" else ("original",)
    missing = [name for name in needed if name not in scaling]
    if missing:
        raise ValueError(f"rotary scaling {rule!r} needs {', '.join(missing)}")
    original = float(scaling["original"])
    if not 0.0 < original < math.inf:
        raise ValueError(f"rotary scaling needs an original context above 0, not {original}")
    if rule == "bands":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not high > low:
            raise ValueError("rotary bands need high_freq_factor above low_freq_factor")
        turns = original * freq / (2.0 * math.pi)
        keep = np.clip((turns - low) / (high - low), 0.0, 1.0)
        return freq * keep + freq / factor * (1.0 - keep), 1.0

    def pair_turning(times: float) -> float:
        return rot_dim * math.log(original / (2.0 * math.pi * times)) / (2.0 * math.log(base))

    beta_fast, beta_slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    if not 0.0 < beta_slow <= beta_fast < math.inf:
        raise ValueError(f"a rotary ramp needs beta_fast {beta_fast} of at least beta_slow {beta_slow}, which is above 0")
    first = max(math.floor(pair_turning(beta_fast)), 0)
    last = min(math.ceil(pair_turning(beta_slow)), rot_dim - 1)
    ramp = np.clip((np.arange(rot_dim // 2) - first) / max(last - first, 1e-3), 0.0, 1.0)
    attention = float(scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0))
    return freq * (1.0 - ramp) + freq / factor * ramp, attention


@dataclass(frozen=True)
class Rotary:
    """A position rotation on one device (see :func:`make_rotary`).

    Attributes:
        turns: int64 ``[rot_dim / 2]`` CUDA tensor: turns per token as 64-bit
            binary fractions (the bits of unsigned integers).
        rot_dim: Rotated dims of a head, a multiple of 8 up to 128.
        interleaved: Pairs are dims ``(2 i, 2 i + 1)`` instead of
            ``(i, i + rot_dim / 2)``.
        factor: Multiplies the rotated dims.

    Raises:
        ValueError: For rotated dims out of range or without their turns.
    """

    turns: torch.Tensor
    rot_dim: int
    interleaved: bool
    factor: float
    _native: FpRotary = field(init=False, repr=False, compare=False)
    _ref: Any = field(init=False, repr=False, compare=False)  # by reference, made once

    def __post_init__(self) -> None:
        _check_rot_dim(self.rot_dim)
        turns = self.turns
        if turns.dtype is not _INT64 or turns.dim() != 1 or not turns.is_contiguous() or len(turns) < self.rot_dim // 2:
            raise ValueError(f"turns must be contiguous int64 [{self.rot_dim // 2}], not {turns.dtype} {tuple(turns.shape)}")
        native = FpRotary(turns=turns.data_ptr(), rot_dim=self.rot_dim, interleaved=int(bool(self.interleaved)),
                          factor=self.factor)
        object.__setattr__(self, "_native", native)
        object.__setattr__(self, "_ref", byref(native))

    def __reduce__(self) -> tuple[Any, ...]:
        # Copies and pickles describe their own tensor.
        return Rotary, (self.turns, self.rot_dim, self.interleaved, self.factor)


def _check_rot_dim(rot_dim: int) -> None:
    if rot_dim < 0 or rot_dim > HEAD_DIM or rot_dim % 8:
        raise ValueError(f"rotated dims {rot_dim} must be a multiple of 8 up to {HEAD_DIM}")


def make_rotary(
    device: torch.device,
    rot_dim: int = HEAD_DIM,
    base: float = 10000.0,
    interleaved: bool = False,
    scaling: dict[str, Any] | None = None,
    frequencies: Any = None,
    factor: float | None = None,
) -> Rotary:
    """Build a :class:`Rotary` on ``device``.

    Args:
        device: Where the heads live.
        rot_dim: Rotated dims, a multiple of 8 up to 128 (0: no rotation);
            further dims of a head stay as they are.
        base, scaling: See :func:`rotary_frequencies`.
        interleaved: Layout of the pairs.
        frequencies: Radians per token ``[rot_dim / 2]``, in place of those of
            ``base`` and ``scaling``.
        factor: Factor on the rotated dims, in place of the rule's.

    Raises:
        ValueError: For impossible parameters.
    """
    _check_rot_dim(rot_dim)
    if frequencies is None:
        freq, rule_factor = rotary_frequencies(rot_dim, base, scaling)
    else:
        if isinstance(frequencies, torch.Tensor):
            frequencies = frequencies.detach().cpu().to(torch.float64).numpy()
        freq = np.asarray(frequencies, dtype=np.float64)
        rule_factor = 1.0
        if freq.shape != (rot_dim // 2,) or not np.isfinite(freq).all():
            raise ValueError(f"frequencies must be {rot_dim // 2} finite numbers")
    factor = float(rule_factor if factor is None else factor)
    if not math.isfinite(factor):
        raise ValueError(f"the factor on the rotated dims must be finite, not {factor}")
    # The fraction of a turn per token; whole turns per token change nothing.
    fractions = [int(f / (2.0 * math.pi) * 2.0**64) % (1 << 64) for f in freq.tolist()]
    bits = np.array(fractions + [0] * (not fractions), dtype=np.uint64).view(np.int64)
    turns = torch.from_numpy(bits).to(device)
    return Rotary(turns, rot_dim, bool(interleaved), factor)


# These checks are most of a small call's host time, so the sound case takes one
# comparison each and the messages are found afterwards.
def head_set(name: str, heads: torch.Tensor, out: torch.Tensor | None, tokens: int, device: int) -> bytes:
    """Check one set of heads and its result on CUDA device ``device``; returns the ``fp_heads`` that describes them."""
    shape, stride = heads.shape, heads.stride()
    if (
        len(shape) != 3
        or shape[0] != tokens
        or shape[2] != HEAD_DIM
        or stride[2] != 1
        or heads.dtype is not _BF16
        or heads.get_device() != device
    ):
        raise RuntimeError(
            f"{name} must be bfloat16 [{tokens}, heads, {HEAD_DIM}] on cuda:{device} with a contiguous head dim, "
            f"not {heads.dtype} {tuple(shape)} on {heads.device} with strides {stride}"
        )
    if out is None:
        return pack_heads(heads.data_ptr(), 0, stride[0], stride[1], 0, 0, shape[1])
    to = out.stride()
    if out.shape != shape or to[2] != 1 or out.dtype is not _BF16 or out.get_device() != device:
        raise RuntimeError(
            f"{name}_out must be bfloat16 {tuple(shape)} on cuda:{device} with a contiguous head dim, "
            f"not {out.dtype} {tuple(out.shape)} on {out.device} with strides {to}"
        )
    return pack_heads(heads.data_ptr(), out.data_ptr(), stride[0], stride[1], to[0], to[1], shape[1])


def rotary_operands(
    positions: torch.Tensor,
    tokens: int,
    rotary: Rotary,
    query_weight: torch.Tensor | None,
    key_weight: torch.Tensor | None,
    device: int,
) -> tuple[int | None, int | None, int, int, int]:
    """Check what :func:`norm_rotary` and ``HbmKvStore.append`` share.

    Returns:
        Pointers of the two weights, whether they are FP32, the pointer of the
        positions and whether those are int64.
    """
    kind = positions.dtype
    if (
        (kind is not _INT64 and kind is not _INT32)
        or positions.shape != (tokens,)
        or not positions.is_contiguous()
        or positions.get_device() != device
        or rotary.turns.get_device() != device
    ):
        raise RuntimeError(
            f"positions must be contiguous int64 or int32 [{tokens}] on cuda:{device}, like the rotary's frequencies"
        )
    q = k = None
    dtype = _BF16
    if query_weight is not None:
        dtype = query_weight.dtype
        q = _weight(query_weight, dtype, device)
    if key_weight is not None:
        if q is None:
            dtype = key_weight.dtype
        k = _weight(key_weight, dtype, device)
    return q, k, dtype is _FP32, positions.data_ptr(), kind is _INT64


def _weight(weight: torch.Tensor, dtype: torch.dtype, device: int) -> int:
    if (
        (dtype is not _BF16 and dtype is not _FP32)
        or weight.dtype is not dtype
        or weight.shape != (HEAD_DIM,)
        or weight.stride(0) != 1
        or weight.get_device() != device
    ):
        raise RuntimeError(
            f"norm weights must both be bfloat16 or both float32, contiguous [{HEAD_DIM}] on cuda:{device}"
        )
    return weight.data_ptr()


_NO_HEADS = pack_heads(0, 0, 0, 0, 0, 0, 0)


def norm_rotary(
    query: torch.Tensor,
    key: torch.Tensor | None,
    positions: torch.Tensor,
    rotary: Rotary,
    query_out: torch.Tensor,
    key_out: torch.Tensor | None,
    query_weight: torch.Tensor | None = None,
    key_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> None:
    """RMS norm of every query and key head, then the position rotation.

    A head ``x`` becomes ``x * rsqrt(mean(x^2) + eps) * weight`` (left out
    without a weight), in FP32, and its pairs are rotated by ``position *
    frequency``; the result is rounded to BF16 once.

    Args:
        query: BF16 ``[T, Hq, 128]`` (tokens and heads may be strided by
            16-byte multiples, as the slices of a packed projection are).
        key: BF16 ``[T, H, 128]``, or None for queries alone.
        positions: int64 or int32 ``[T]``.
        rotary: The rotation.
        query_out, key_out: BF16 results of the same shapes; may be ``query``
            / ``key`` themselves, must not overlap the inputs otherwise.
        query_weight, key_weight: ``[128]`` BF16 or FP32, or None for no norm.
        eps: Added to the mean square.

    Raises:
        RuntimeError: For rejected arguments or a failed launch.

    Async/thread-safety:
        One kernel on the current CUDA stream; CUDA-graph safe; allocates nothing.
    """
    device = query.get_device()
    if device < 0:
        require_cuda(query, "query")
    if (key is None) != (key_out is None):
        raise RuntimeError("key and key_out come together")
    tokens = query.shape[0]
    q = head_set("query", query, query_out, tokens, device)
    k = _NO_HEADS if key is None else head_set("key", key, key_out, tokens, device)
    operands = rotary_operands(positions, tokens, rotary, query_weight, key_weight, device)
    with on_device(device):
        check(
            extension().fp_norm_rotary(
                q, k, *operands, tokens, rotary._ref, eps, stream_ptr(),
            )
        )


__all__ = ["Rotary", "make_rotary", "norm_rotary", "rotary_frequencies"]
