"""Rotary positions of queries and keys (no counterpart in the reference, which rotates inside
its MLA module only, modules/flash_mla.py:26-58).

``fastest_flash_rotary`` turns pair i of the row at position t by ``t * inv_freq[i]``, the
angle formed in 64 bits, in one launch of ``ffa_rotary`` for queries and keys; the gradient is
the same launch with the opposite angle. ``rotary_frequencies`` makes the frequencies, scaled
for contexts longer than the trained ones.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from ..kernels import _lib


def rotary_frequencies(
    rotary_dim: int,
    base: float = 10000.0,
    *,
    scaling: Optional[str] = None,
    factor: float = 1.0,
    original_max_position: Optional[int] = None,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    device: torch.device | str = "cpu",
) -> torch.Tensor:
    """float64 ``[rotary_dim // 2]`` frequencies ``base ** (-2 i / rotary_dim)``.

    ``scaling`` stretches them by ``factor`` for longer contexts:

    - ``None``      as they are (``factor`` has to be 1)
    - ``"linear"``  every frequency divided by ``factor`` (positions interpolated)
    - ``"ntk"``     a larger base: the highest frequency kept, the lowest divided by ``factor``
    - ``"yarn"``    pairs that turn more than ``beta_fast`` times over
      ``original_max_position`` tokens kept, those that turn less than ``beta_slow`` times
      divided by ``factor``, a linear ramp over the pairs between (its magnitude is
      ``yarn_magnitude(factor)``)
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even and positive (got {rotary_dim})")
    if not (math.isfinite(base) and base > 0.0 and math.isfinite(factor) and factor > 0.0):
        raise ValueError("base and factor must be positive")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r} (linear, ntk, yarn)")
    if scaling is None and factor != 1.0:
        raise ValueError("factor needs a scaling")
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = base ** (-2.0 * pair / rotary_dim)
    if scaling == "linear" or (scaling == "ntk" and rotary_dim == 2):
        freq = freq / factor
    elif scaling == "yarn":
        if original_max_position is None or original_max_position < 1:
            raise ValueError("yarn scaling needs original_max_position")
        if not beta_fast > beta_slow > 0.0:
            raise ValueError("yarn scaling needs beta_fast > beta_slow > 0")

        def pair_of(turns: float) -> float:
            """The (fractional) pair that turns this many times over the original context."""
            return (rotary_dim * math.log(original_max_position / (turns * 2.0 * math.pi))
                    / (2.0 * math.log(base)))

        if base == 1.0:
            raise ValueError("yarn scaling needs a base other than 1")
        lo = max(math.floor(pair_of(beta_fast)), 0)
        hi = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        ramp = ((pair - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        freq = freq * (1.0 - ramp) + freq / factor * ramp
    return freq.to(device)


def yarn_magnitude(factor: float) -> float:
    """The factor on rotated queries and keys that goes with ``"yarn"`` scaling."""
    return 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0


def check_frequencies(inv_freq: torch.Tensor, head_dim: int, device: torch.device) -> torch.Tensor:
    """inv_freq as the kernels read it, or an error."""
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1 or inv_freq.numel() < 1:
        raise ValueError("inv_freq must be a 1D tensor of frequencies, one for each pair")
    if inv_freq.dtype != torch.float64:
        raise TypeError(f"inv_freq must be float64 (got {inv_freq.dtype}): rotary_frequencies makes it")
    if 2 * inv_freq.numel() > head_dim:
        raise ValueError(f"{inv_freq.numel()} pairs do not fit head_dim {head_dim}")
    if inv_freq.device != device:
        raise RuntimeError(f"inv_freq is on {inv_freq.device}, the tensors on {device}")
    return inv_freq.contiguous()


def check_magnitude(magnitude: float) -> float:
    magnitude = float(magnitude)
    if not math.isfinite(magnitude):
        raise ValueError("magnitude must be finite")
    return magnitude


def in_and_out(t: torch.Tensor):
    """The tensor as the kernel reads it, its output, and their strides ahead of the last dim's."""
    stride = t.stride()
    if stride[-1] != 1 and t.size(-1) > 1:
        t = t.contiguous()
        stride = t.stride()
    out = torch.empty_like(t)
    out_stride = out.stride()
    if out_stride[-1] != 1 and t.size(-1) > 1:
        out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        out_stride = out.stride()
    return t, out, stride[:-1], out_stride[:-1]


def _rotate(q: Optional[torch.Tensor], k: Optional[torch.Tensor], inv_freq: torch.Tensor,
            positions: Optional[torch.Tensor], q_offset: int, interleaved: bool, magnitude: float,
            inverse: bool) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """One launch over 4D tensors (either may be None); outputs in the inputs' memory order."""
    x = q if q is not None else k
    a = _lib.RotaryArgs()
    a.batch, _, a.seqlen, a.head_dim = x.shape
    q_out = k_out = None
    if q is not None:  # (q and k: kept until the launch where they are copies)
        q, q_out, a.q_stride[:], a.q_out_stride[:] = in_and_out(q)
        a.q, a.q_out, a.heads_q = q.data_ptr(), q_out.data_ptr(), q.size(1)
    if k is not None:
        k, k_out, a.k_stride[:], a.k_out_stride[:] = in_and_out(k)
        a.k, a.k_out, a.heads_k = k.data_ptr(), k_out.data_ptr(), k.size(1)
    a.inv_freq = inv_freq.data_ptr()
    a.q_offset = q_offset
    if positions is not None:
        a.positions = positions.data_ptr()
        a.position_bytes = positions.element_size()
        a.position_stride[:] = [positions.stride(0) if positions.size(0) > 1 else 0,
                                positions.stride(1)]
    a.rotary_dim = 2 * inv_freq.numel()
    a.interleaved = interleaved
    a.inverse = inverse
    a.magnitude = magnitude
    a.dtype = _lib.dtype_code(x.dtype, allow_fp32=True)
    _lib.launch(_lib.load().ffa_rotary, a, x.device)
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """The gradient of a rotation is the rotation back, itself differentiable."""

    @staticmethod
    def forward(ctx, q, k, inv_freq, positions, q_offset, interleaved, magnitude, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(inv_freq, positions)
        ctx.how = (q_offset, interleaved, magnitude)
        ctx.inverse = inverse
        return _rotate(q, k, inv_freq, positions, q_offset, interleaved, magnitude, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        inv_freq, positions = ctx.saved_tensors
        if not ctx.needs_input_grad[0]:
            dq = None
        if not ctx.needs_input_grad[1]:
            dk = None
        if dq is not None or dk is not None:
            # (an autograd call of its own only where the gradient is differentiated again)
            rotate = _Rotary.apply if torch.is_grad_enabled() else _rotate
            dq, dk = rotate(dq, dk, inv_freq, positions, *ctx.how, not ctx.inverse)
        return dq, dk, None, None, None, None, None, None


def fastest_flash_rotary(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    inv_freq: torch.Tensor,
    *,
    positions: Optional[torch.Tensor] = None,
    q_offset: int = 0,
    interleaved: bool = False,
    magnitude: float = 1.0,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotary positions of ``q`` ``[B, H, S, D]`` and ``k`` ``[B, Hk, S, D]`` (or both
    ``[B, S, D]``; ``k`` may be None), as new tensors in their memory order.

    The first ``2 * len(inv_freq)`` dims turn: pair i of the row at position t, dims
    ``(i, i + len(inv_freq))``, or ``(2 i, 2 i + 1)`` with ``interleaved``, by the angle
    ``t * inv_freq[i]``, times ``magnitude``; the other dims are copied. ``positions`` (int32
    or int64, ``[S]``, ``[1, S]`` or ``[B, S]``) are the rows' positions, by default
    ``q_offset + 0 .. S - 1``. ``inv_freq`` is float64 (``rotary_frequencies``). bfloat16,
    float16 and float32; differentiable in q and k.
    """
    squeezed = q.dim() == 3
    if squeezed:
        q = q.unsqueeze(1)
        k = k.unsqueeze(1) if k is not None else None
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k must be 3D [B, S, D] or 4D [B, H, S, D]")
    B, _, S, D = q.shape
    if k is not None:
        if (k.size(0), k.size(2), k.size(3)) != (B, S, D):
            raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
        if k.dtype != q.dtype:
            raise TypeError(f"q/k dtypes differ: {q.dtype}, {k.dtype}")
    for name, t in (("q", q), ("k", k)):
        if t is not None and t.device.type != "cuda":
            raise RuntimeError(f"fastest_flash_attention_amd runs on ROCm GPU tensors only; {name} is "
                               f"on {t.device} (there is no CPU path)")
    if k is not None and k.device != q.device:
        raise RuntimeError("q and k must be on the same device")
    _lib.dtype_code(q.dtype, allow_fp32=True)
    inv_freq = check_frequencies(inv_freq, D, q.device)
    magnitude = check_magnitude(magnitude)
    if positions is not None:
        if q_offset:
            raise ValueError("q_offset and positions exclude each other")
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64 (got {positions.dtype})")
        if positions.device != q.device:
            raise RuntimeError(f"positions are on {positions.device}, q on {q.device}")
        if positions.dim() == 1:
            positions = positions.unsqueeze(0)
        if positions.dim() != 2 or positions.size(1) != S or positions.size(0) not in (1, B):
            raise ValueError(f"positions of shape {tuple(positions.shape)}, expected [S], [1, S] or "
                             f"[B, S] with B {B}, S {S}")
    how = (inv_freq, positions, int(q_offset), bool(interleaved), magnitude, False)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        q, k = _Rotary.apply(q, k, *how)
    else:
        q, k = _rotate(q, k, *how)
    if squeezed:
        q = q.squeeze(1)
        k = k.squeeze(1) if k is not None else None
    return q, k
