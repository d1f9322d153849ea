"""Rotary frequency tables for ops.rope and ops.kv_append: float64 [dims / 2], scaled for contexts beyond the trained length.

The model's own layers use the plain table (volundr.py:663-664) inside vk_attn_prep; these are for everything else that
rotates (a drafter, an imported checkpoint with another convention, keys appended for a shared prefix)."""
import math

import torch

SCALINGS = ("none", "linear", "ntk", "parts")


def frequencies(dims, theta, *, scaling="none", factor=1.0, trained_len=4096, low=1.0, high=32.0, magnitude=None, device=None):
    """(freq, magnitude) for `dims` rotated elements of a head: freq_i = theta^(-2i / dims), then

    linear  every frequency divided by `factor` (positions interpolated);
    ntk     theta stretched to theta * factor^(dims / (dims - 2)): the fastest pair unchanged, the slowest divided by factor;
    parts   by the turns r_i = trained_len * freq_i / (2 pi) a pair makes over the trained length: divided by `factor` below
            `low` turns, unchanged above `high`, a linear ramp between.

    magnitude multiplies the rotated elements; the default is 1, and 0.1 ln(factor) + 1 for `parts`."""
    if dims < 0 or dims % 2 or not theta > 0 or not factor >= 1:
        raise ValueError("dims: even; theta: positive; factor: at least 1")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling: one of {SCALINGS}")
    if scaling == "parts" and not (high > low and trained_len > 0):
        raise ValueError("parts: high > low and a positive trained_len")
    if scaling == "ntk" and dims > 2:
        theta = theta * factor ** (dims / (dims - 2))
    f = theta ** (-torch.arange(0, dims, 2, dtype=torch.float64) / max(dims, 1))
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        keep = ((trained_len * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    if magnitude is None:
        magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "parts" else 1.0
    return f.to(device), float(magnitude)
