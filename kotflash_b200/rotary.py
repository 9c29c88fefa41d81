# SPDX-License-Identifier: Apache-2.0
"""Rotary positions for the queries and keys of ``attention``, the caches and their steps.

``apply_rotary`` turns column pairs of q and k by angles position * frequency,
q and k in one launch, with the rotation back as its gradient;
``rotary_frequencies`` gives the frequencies, also those stretched for contexts
longer than a model was trained on.  fp16 and bf16 on an sm_100 device through
``libkotflash_b200.so``; nothing falls back to another implementation.  The
reference has no positions (its callers rotate before ``attention``).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _ext

_DTYPES = {torch.float16: _ext.KF_F16, torch.bfloat16: _ext.KF_BF16}
_POSITION_BITS = {torch.int32: 32, torch.int64: 64}
_FLOAT64 = torch.float64
_CONTIGUOUS = torch.contiguous_format
_NONE = (0,) * 9
_pack, _is_sm100 = _ext.pack_rotary, _ext.is_sm100


def rotary_frequencies(
    rotated: int,
    *,
    base: float = 10000.0,
    scaling: str = "none",
    factor: float = 1.0,
    trained_length: Optional[int] = None,
    slow: float = 1.0,
    fast: float = 32.0,
    device: Union[torch.device, str, None] = None,
) -> Tuple[torch.Tensor, float]:
    """Frequencies of ``rotated / 2`` pairs and the magnitude that goes with them.

    Pair i turns base^(-2i / rotated) radians per position (float64).  scaling
    says how they change for contexts ``factor`` times as long as trained:

    * "none": not at all;
    * "linear": all divided by factor (positions interpolated);
    * "ntk": base grows by factor^(rotated / (rotated - 2)), so that the slowest
      pair is divided by factor and the fastest stays;
    * "yarn": pairs that turn ``slow`` times or less within trained_length are
      divided by factor, those that turn ``fast`` times or more stay, those
      between are blended in proportion to their turns, as published; q and k
      grow by the magnitude 0.1 ln(factor) + 1.  (A model that was trained with
      a blend by the pairs' index has other frequencies between the two: pass
      those.)

    Returns ``(frequencies, magnitude)`` for ``apply_rotary``; magnitude is 1
    but for "yarn".
    """
    if isinstance(rotated, bool) or not isinstance(rotated, int) or rotated <= 0 or rotated % 2:
        raise ValueError("rotated must be a positive even integer")
    if not (math.isfinite(base) and base > 0):
        raise ValueError("base must be positive and finite")
    if not (math.isfinite(factor) and factor >= 1):
        raise ValueError("factor must be finite and at least 1")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError("scaling must be 'none', 'linear', 'ntk' or 'yarn'")
    if scaling == "ntk" and rotated > 2:
        base = base * factor ** (rotated / (rotated - 2))
    f = torch.tensor([base ** (-i / rotated) for i in range(0, rotated, 2)], dtype=torch.float64)
    magnitude = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if trained_length is None or not trained_length > 0:
            raise ValueError("yarn needs trained_length")
        if not 0 <= slow < fast:
            raise ValueError("slow must be at least 0 and below fast")
        keep = ((trained_length * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0
    return f.to(device) if device is not None else f, magnitude


def _check(q, k, positions, frequencies) -> None:
    what = "apply_rotary"
    for t in (q,) if k is None else (q, k):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: q and k must be torch.Tensor instances")
        if t.ndim != 4:
            raise ValueError(f"{what}: expected 4-D tensors in [B, H, S, D] layout")
        if t.dtype != q.dtype:
            raise ValueError(f"{what}: dtypes must match")
    if q.dtype not in _DTYPES:
        raise TypeError(f"{what} supports float16 and bfloat16, got {q.dtype}")
    b, _, s, d = q.shape
    if k is not None and (k.shape[0] != b or k.shape[2] != s or k.shape[3] != d):
        raise ValueError(f"{what}: q and k must agree in batch, tokens and head_dim")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in _POSITION_BITS:
        raise TypeError(f"{what}: positions must be an int32 or int64 tensor")
    if positions.shape not in ((b, s), (s,)):
        raise ValueError(f"{what}: positions must be [B, S] or [S]")
    if not isinstance(frequencies, torch.Tensor) or frequencies.dtype != torch.float64:
        raise TypeError(f"{what}: frequencies must be a float64 tensor")
    if frequencies.ndim != 1 or not frequencies.is_contiguous() or not 0 < 2 * frequencies.shape[0] <= d:
        raise ValueError(f"{what}: frequencies must be contiguous, one for each pair of at most head_dim columns")
    if frequencies.requires_grad:
        raise RuntimeError(f"{what}: frequencies have no gradient")
    dev = q.device
    if dev.type != "cuda":
        raise RuntimeError(f"{what} requires CUDA tensors on an sm_100 (B200) device")
    for t in (positions, frequencies) if k is None else (k, positions, frequencies):
        if t.device != dev:
            raise ValueError(f"{what}: all tensors must be on the same device")
    if not _ext.is_sm100(dev.index):
        raise RuntimeError(f"{what} requires an sm_100 (B200) CUDA device")


def _rotate(q, k, positions, frequencies, interleaved, magnitude, inverse):
    """(q', k') as new contiguous tensors; either of q and k may be None."""
    if q is not None and q.stride(3) != 1:
        q = q.contiguous()
    if k is not None and k.stride(3) != 1:
        k = k.contiguous()
    q_out = None if q is None else torch.empty_like(q, memory_format=_CONTIGUOUS)
    k_out = None if k is None else torch.empty_like(k, memory_format=_CONTIGUOUS)
    outs = q_out, k_out
    if q is None or q.numel() == 0:  # the first of the two has something to rotate
        q, q_out, k, k_out = k, k_out, None, None
        if q is None or q.numel() == 0:
            return outs
    qs = q.shape
    index = q.get_device()
    second = _NONE
    second_out = _NONE
    if k is not None and k.numel():
        ks = k.shape
        _, h, s, d = ks
        second = (k.data_ptr(), *ks, *k.stride())
        second_out = (k_out.data_ptr(), *ks, h * s * d, s * d, d, 1)
    _, h, s, d = qs
    by_batch, by_token = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
    rc = _ext.load().kf_rotary(_pack(
        q.data_ptr(), *qs, *q.stride(), *second, q_out.data_ptr(), *qs, h * s * d, s * d, d, 1, *second_out,
        positions.data_ptr(), _POSITION_BITS[positions.dtype], by_batch, by_token, frequencies.data_ptr(),
        2 * frequencies.numel(), interleaved, inverse, magnitude, _DTYPES[q.dtype], _ext.raw_stream(index)))
    if rc:
        _ext.check(rc, "kf_rotary")
    return outs


class _Rotary(torch.autograd.Function):
    """The rotation, linear in q and k: tangents are rotated as q and k are,
    gradients back.  Neither of the two is a constant where one has a tangent."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved, magnitude, inverse, tangents):
        ctx.save_for_backward(positions, frequencies)
        if tangents:
            ctx.save_for_forward(positions, frequencies)
        ctx.set_materialize_grads(False)
        ctx.how = interleaved, magnitude, inverse
        outs = _rotate(q, k, positions, frequencies, interleaved, magnitude, inverse)
        constant = [] if tangents else [out for out, need in zip(outs, ctx.needs_input_grad) if out is not None and not need]
        if constant:
            ctx.mark_non_differentiable(*constant)
        return outs

    @staticmethod
    def backward(ctx, dq, dk):
        inverse = ctx.how[2]
        need_q, need_k = ctx.needs_input_grad[:2]
        dq, dk = _turned(ctx, dq if need_q else None, dk if need_k else None, not inverse)
        return dq, dk, None, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        return _turned(ctx, tq, tk, ctx.how[2])


def _turned(ctx, x, y, inverse):
    """A gradient's or tangent's rotation, differentiable as the call itself is."""
    if x is None and y is None:
        return None, None
    positions, frequencies = ctx.saved_tensors
    interleaved, magnitude, _ = ctx.how
    return _differentiable(x, y, positions, frequencies, interleaved, magnitude, inverse)


def _differentiable(q, k, positions, frequencies, interleaved, magnitude, inverse):
    """_rotate(), through autograd where q or k has a gradient or a tangent."""
    tangents = False
    if forward_ad._current_level >= 0:  # what unpack_dual() goes by; asking it costs 0.7 us where there is no level
        q_tangent, k_tangent = (t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (q, k))
        if q_tangent != k_tangent and q is not None and k is not None:  # one call would give the other a tangent
            return (_differentiable(q, None, positions, frequencies, interleaved, magnitude, inverse)[0],
                    _differentiable(None, k, positions, frequencies, interleaved, magnitude, inverse)[1])
        tangents = q_tangent or k_tangent
    if tangents or (((q is not None and q.requires_grad) or (k is not None and k.requires_grad)) and torch.is_grad_enabled()):
        return _Rotary.apply(q, k, positions, frequencies, interleaved, magnitude, inverse, tangents)
    return _rotate(q, k, positions, frequencies, interleaved, magnitude, inverse)


def apply_rotary(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    interleaved: bool = False,
    magnitude: float = 1.0,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Rotate q [B, Hq, S, D] and k [B, Hkv, S, D] (or None) by their positions.

    positions is int32 or int64, [B, S] or, for all batch entries, [S];
    frequencies float64 [R / 2] on the same device, finite, radians per position.  The
    first R columns turn in pairs, column i with i + R / 2 or, interleaved,
    2i with 2i + 1; the columns behind them pass.  Rotated columns are
    multiplied by magnitude.  Angles are worked out in 64 bits (exact to 32-bit
    rounding up to 2^28 radians, as position * frequency in float64 is), the
    rest in 32, rounded once.  Any strides; new contiguous tensors are returned, ``(q',
    k')``, or q' alone where k is None.  Differentiable in q and k, backwards and,
    with ``torch.autograd.forward_ad``, forwards.
    """
    try:  # what a valid call of q and k pays for; _check() finds out what to say
        index = q.get_device()
        b, _, s, d = q.shape
        kb, _, ks, kd = k.shape
        ps = positions.shape
        good = (
            index >= 0 and k.get_device() == index and positions.get_device() == index
            and frequencies.get_device() == index and _is_sm100(index) and q.dtype in _DTYPES and k.dtype is q.dtype
            and kb == b and ks == s and kd == d and positions.dtype in _POSITION_BITS and (ps == (b, s) or ps == (s,))
            and frequencies.dtype is _FLOAT64 and frequencies.dim() == 1 and 0 < 2 * frequencies.numel() <= d
            and frequencies.is_contiguous() and not frequencies.requires_grad)
    except (AttributeError, TypeError, ValueError, RuntimeError):
        good = False
    if not good:
        _check(q, k, positions, frequencies)
    magnitude = float(magnitude)
    if not math.isfinite(magnitude):
        raise ValueError("magnitude must be finite")
    interleaved = bool(interleaved)
    outs = _differentiable(q, k, positions, frequencies, interleaved, magnitude, False)
    return outs[0] if k is None else outs
