"""Rotate-half RoPE tables (HuggingFace ``cat(freqs, freqs)`` layout).

Same values as the reference's tables (gpu/decodev2/rope.py:20-53): float32
numpy arithmetic, then one cast to the cache dtype.
"""

from __future__ import annotations

import numpy as np
import torch

__all__ = ["rope_tables_numpy", "rope_tables_torch", "rope_tables_scaled", "apply_rope_torch"]


def rope_tables_numpy(max_seq: int, head_dim: int, theta: float) -> tuple[np.ndarray, np.ndarray]:
    if head_dim % 2:
        raise ValueError("even head_dim required")
    idx = np.arange(0, head_dim, 2, dtype=np.float32)
    inv = (1.0 / (np.float32(theta) ** (idx / np.float32(head_dim)))).astype(np.float32)
    ang = np.outer(np.arange(max_seq, dtype=np.float32), inv).astype(np.float32)
    ang = np.concatenate([ang, ang], axis=-1)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def rope_tables_torch(max_seq: int, head_dim: int, theta: float, *, device, dtype):
    cos, sin = rope_tables_numpy(max_seq, head_dim, theta)
    return (
        torch.from_numpy(cos).to(device=device, dtype=dtype),
        torch.from_numpy(sin).to(device=device, dtype=dtype),
    )


def rope_tables_scaled(max_seq: int, rot_dim: int, theta: float, *, scaling: str = "none", factor: float = 1.0,
                       original: int | None = None, fast: float = 32.0, slow: float = 1.0, ramp: str = "turns",
                       device, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """Tables ``[max_seq, rot_dim/2]`` of the first ``rot_dim`` elements of a head, one column per
    pair, for ``nf4_rope_kv_paged``; additive to the reference's (gpu/decodev2/rope.py:20-53).

    With ``inv_i = theta^(-2i/rot_dim)`` the angle of pair ``i`` at position ``p`` is ``p * inv_i``.
    ``scaling`` stretches the positions of a model trained on ``original`` of them by ``factor``:
    ``linear`` divides every angle; ``ntk`` raises theta to ``theta * factor^(rot_dim/(rot_dim-2))``,
    which leaves the fastest pair alone and slows the slowest by the factor; ``yarn`` leaves alone the
    pairs that turn more than ``fast`` times over ``original`` positions, divides those that turn
    fewer than ``slow`` times, blends in between, and multiplies cos and sin by
    ``1 + 0.1 ln(factor)``. Computed in float64: a float32 angle is off by 0.004 at position 65536.

    ``ramp`` says how ``yarn`` blends. ``turns``, as the method's paper defines it (Peng et al. 2023,
    "YaRN", section 3.2): linearly in the number of turns. ``pairs``, as checkpoints with yarn settings
    are commonly run: linearly in the pair's index, between the last whole index at or before the
    one of ``fast`` turns and the first at or after that of ``slow``, both drawn to the pairs there are.
    Turns fall geometrically with the index, so the two differ in between (pair 32 of 64 by a factor of
    1.7 for theta 1e6, 32768 positions, factor 4): take the one the checkpoint was made with."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("even rot_dim required")
    if max_seq < 1 or theta <= 0 or factor < 1:
        raise ValueError("max_seq and theta must be positive, factor at least 1")
    inv = theta ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
    gain = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "ntk":
        if rot_dim < 4:
            raise ValueError("ntk scaling needs at least two pairs")
        inv = (theta * factor ** (rot_dim / (rot_dim - 2))) ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
    elif scaling == "yarn":
        if original is None or original < 1 or not fast > slow > 0:
            raise ValueError("yarn scaling needs the original length and fast > slow > 0")
        if ramp == "turns":
            turns = original * inv / (2 * np.pi)
            keep = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
        elif ramp == "pairs":
            if theta <= 1:
                raise ValueError("a ramp over pairs needs theta above 1")
            # pair i turns original theta^(-2i/rot_dim) / (2 pi) times
            pair = lambda turns: rot_dim * np.log(original / (2 * np.pi * turns)) / (2 * np.log(theta))  # noqa: E731
            first, last = max(np.floor(pair(fast)), 0.0), min(np.ceil(pair(slow)), rot_dim - 1.0)
            # (both ends at one pair, or the last before the first: a step)
            keep = 1.0 - np.clip((np.arange(rot_dim // 2) - first) / max(last - first, 1e-3), 0.0, 1.0)
        else:
            raise ValueError(f"ramp {ramp!r} not in turns|pairs")
        inv = inv * keep + inv / factor * (1.0 - keep)
        gain = 1.0 + 0.1 * np.log(factor)
    elif scaling != "none":
        raise ValueError(f"scaling {scaling!r} not in none|linear|ntk|yarn")
    ang = np.outer(np.arange(max_seq, dtype=np.float64), inv)
    put = lambda a: torch.from_numpy(gain * a).to(device=device, dtype=dtype)
    return put(np.cos(ang)), put(np.sin(ang))


def apply_rope_torch(t: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """``t`` [n, heads, hd]; ``cos``/``sin`` [n, hd]. Tensor math in ``t``'s dtype."""
    if cos.ndim == 2:
        cos = cos[:, None, :]
        sin = sin[:, None, :]
    half = t.shape[-1] // 2
    swapped = torch.cat((-t[..., half:], t[..., :half]), dim=-1)
    return t * cos + swapped * sin
