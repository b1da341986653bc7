"""Optimizers in native kernels (``csrc/adamw.cu``).  An addition to the reference, whose training scripts take torch's."""
from .adamw import AdamW, adamw_step, decode_moments, moment_slots

__all__ = ["AdamW", "adamw_step", "decode_moments", "moment_slots"]
