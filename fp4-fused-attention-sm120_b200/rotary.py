"""Rotary positions: the table of cosines and sines, and the rotation.

``rotary`` turns the first ``2 * table.shape[1]`` elements of every row of a
[batch, heads, seq, head_dim] tensor (fp4attn_rotary); ``rotary_embedding`` is
the same under autograd, whose gradient turns back by the same angles.
"""
from __future__ import annotations

import ctypes
import math

from . import _serving as sv

__all__ = ["rotary_frequencies", "rotary_table", "rotary", "rotary_embedding"]


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_positions=None,
                       beta_fast=32.0, beta_slow=1.0):
    """(frequencies, table factor) of the rotary_dim / 2 pairs, in float64:
    base^(-2j / rotary_dim), for contexts ``factor`` times as long as trained

    - scaling=None: as they are;
    - "linear": divided by factor (position interpolation);
    - "ntk": base raised by factor^(d / (d - 2)), which leaves the fastest pair
      as it is and divides the slowest by factor;
    - "yarn": pairs that turn more than beta_fast times in
      original_positions are kept, those that turn less than beta_slow times
      are divided by factor, a linear ramp between; and the table is
      multiplied by 0.1 ln(factor) + 1."""
    if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > 256:
        raise ValueError("rotary_dim must be even, in [2, 256]")
    if not base > 1.0 or not factor >= 1.0 or not math.isfinite(base * factor):
        raise ValueError("base must be > 1 and factor >= 1")
    half = rotary_dim // 2
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs rotary_dim > 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freqs = [base ** (-2.0 * j / rotary_dim) for j in range(half)]
    if scaling in (None, "ntk"):
        return freqs, 1.0
    if scaling == "linear":
        return [f / factor for f in freqs], 1.0
    if scaling == "yarn":
        if original_positions is None or original_positions < 1:
            raise ValueError("yarn scaling needs original_positions")
        if not beta_fast > beta_slow > 0:
            raise ValueError("beta_fast > beta_slow > 0")

        def pair_that_turns(times):
            return rotary_dim * math.log(original_positions / (times * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_that_turns(beta_fast)), 0)
        high = min(math.ceil(pair_that_turns(beta_slow)), rotary_dim - 1)  # (may lie behind the last pair)
        high = max(high, low + 0.001)
        out = []
        for j, f in enumerate(freqs):
            ramp = min(1.0, max(0.0, (j - low) / (high - low)))
            out.append(f * (1.0 - ramp) + f / factor * ramp)
        return out, 0.1 * math.log(factor) + 1.0
    raise ValueError(f"unknown scaling {scaling!r}")


def rotary_table(max_positions, rotary_dim, base=10000.0, scaling=None, factor=1.0, original_positions=None,
                 beta_fast=32.0, beta_slow=1.0, device="cuda", stream=None):
    """float32 [max_positions, rotary_dim / 2, 2] of cos and sin of position *
    frequency (fp4attn_rotary_table); see rotary_frequencies for the scalings."""
    torch = sv.torch()
    freqs, table_factor = rotary_frequencies(rotary_dim, base, scaling, factor, original_positions, beta_fast,
                                             beta_slow)
    if max_positions < 1:
        raise ValueError("max_positions must be >= 1")
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("device must be a CUDA device")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    arr = (ctypes.c_double * len(freqs))(*freqs)
    with torch.cuda.device(device) if stream is None else sv.on(device, stream):
        table = torch.empty((max_positions, rotary_dim // 2, 2), dtype=torch.float32, device=device)
        sv.check(sv.lib().fp4attn_rotary_table(arr, len(freqs), max_positions, table_factor, table.data_ptr(),
                                               torch.cuda.current_stream().cuda_stream), "fp4attn_rotary_table")
    return table


def rotary(x, table, positions=None, interleaved=False, inverse=False, out=None, stream=None):
    """x [batch, heads, seq, head_dim] (float16 or float32, any strides with
    the last dimension contiguous) turned by its positions into ``out``
    (contiguous by default; ``out=x`` turns in place, and any other ``out`` may
    share no element with x).

    positions: int32 [seq] or [batch, seq], by default 0 .. seq - 1.
    interleaved: pairs (2j, 2j + 1) instead of (j, j + rotary_dim / 2).
    inverse: turn back, which is the gradient's rotation."""
    native = sv.native()
    if stream is None:
        return native.rotary(x, table, positions, interleaved, inverse, out)
    with sv.on(x.device, stream):
        return native.rotary(x, table, positions, interleaved, inverse, out)


def rotary_embedding(x, table, positions=None, interleaved=False):
    """``rotary`` that autograd can differentiate (with respect to x, any number
    of times): the gradient turns back by the same angles.

    As with every operation: when a backward pass is captured into a CUDA
    graph, no eager graph of the same leaves may be alive, for autograd would
    wait for the stream of that one, which ends the capture."""
    return sv.native().rotary_embedding(x, table, positions, interleaved)
