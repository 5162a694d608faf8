"""FastestFlashRotary — rotary positions as a module (no counterpart in the reference, whose
RotaryEmbedding serves its MLA module only, modules/flash_mla.py:26-58)."""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from ..ops.rotary import fastest_flash_rotary, rotary_frequencies, yarn_magnitude


class FastestFlashRotary(nn.Module):
    """Rotary positions of a model's heads: the frequencies, kept in 64 bits whatever dtype the
    model is cast to, and how pairs are laid out. It holds no parameters and no state that a
    checkpoint would carry.

    Args:
        rotary_dim: leading dims of each head that turn (even).
        base, scaling, factor, original_max_position: as in ``rotary_frequencies``.
        interleaved: pairs are neighbouring dims instead of the halves of ``rotary_dim``.
        magnitude: factor on rotated queries and keys; None: that of the scaling (1, or
            ``yarn_magnitude(factor)``).
    """

    def __init__(
        self,
        rotary_dim: int,
        base: float = 10000.0,
        *,
        interleaved: bool = False,
        scaling: Optional[str] = None,
        factor: float = 1.0,
        original_max_position: Optional[int] = None,
        magnitude: Optional[float] = None,
        device: Optional[torch.device | str] = None,
    ):
        super().__init__()
        self.rotary_dim = rotary_dim
        self.interleaved = interleaved
        if magnitude is None:
            magnitude = yarn_magnitude(factor) if scaling == "yarn" else 1.0
        self.magnitude = magnitude
        self._made_with = dict(rotary_dim=rotary_dim, base=base, scaling=scaling, factor=factor,
                               original_max_position=original_max_position)
        self.inv_freq = rotary_frequencies(
            **self._made_with, device=torch.empty(0).device if device is None else device)

    def _apply(self, fn, *args, **kwargs):
        # follow the module to its device, not to its dtype
        super()._apply(fn, *args, **kwargs)
        device = fn(self.inv_freq).device
        if self.inv_freq.is_meta and device.type != "meta":
            self.inv_freq = rotary_frequencies(**self._made_with, device=device)
        else:
            self.inv_freq = self.inv_freq.to(device)
        return self

    def append_options(self, device: torch.device) -> dict:
        """The rotation's arguments of ``fastest_flash_paged_append``."""
        if self.inv_freq.device != device:
            raise RuntimeError(f"the rotary module is on {self.inv_freq.device}, the cache on {device}")
        return dict(inv_freq=self.inv_freq, interleaved=self.interleaved, magnitude=self.magnitude)

    def forward(
        self,
        q: torch.Tensor,
        k: Optional[torch.Tensor] = None,
        *,
        positions: Optional[torch.Tensor] = None,
        q_offset: int = 0,
    ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """``fastest_flash_rotary`` of q and k ``[B, H, S, D]``."""
        return fastest_flash_rotary(q, k, self.inv_freq, positions=positions, q_offset=q_offset,
                                    interleaved=self.interleaved, magnitude=self.magnitude)

    def extra_repr(self) -> str:
        return (f"rotary_dim={self.rotary_dim}, interleaved={self.interleaved}, "
                f"magnitude={self.magnitude}")
