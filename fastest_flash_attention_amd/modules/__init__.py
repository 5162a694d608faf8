"""nn.Module wrappers: attention with the reference interfaces, and rotary positions."""

from .flash_gqa import FastestFlashGQA
from .flash_mha import FastestFlashMHA
from .flash_mla import FastestFlashMLA
from .flash_rotary import FastestFlashRotary

__all__ = ["FastestFlashMHA", "FastestFlashGQA", "FastestFlashMLA", "FastestFlashRotary"]
