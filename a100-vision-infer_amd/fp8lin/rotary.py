"""Rotary positions: plans of frequencies, scaled for long contexts or not, and
the rotation of heads by them (include/fp8lin.h describes the operators).

`fused_rope` and `qk_norm_rope` are the reference's form: half layout, FP32
angles, BF16 between the products.  Here pairs are halves or neighbours, the
angle is exact at any position, and the result is rounded once.
"""
import ctypes
from collections import namedtuple

import torch

from ._lib import ERR_ARGUMENT, ERR_SHAPE, RotaryRecord, check, lib
from .ops import _fail, call

RotaryPlan = namedtuple("RotaryPlan", "steps magnitude neighbours")
RotaryPlan.__doc__ = """What rotates heads: steps int64 [rotary / 2] on the device (4 * round(frequency / 2 pi * 2^62) + axis of each pair, as
rotary_plan makes them), magnitude of the cosines and sines, and whether pairs are neighbours (2j, 2j + 1) or halves (j, j + rotary / 2)."""

_SCALINGS = {"default": 0, "linear": 1, "ntk": 2, "yarn": 3, "wavelength": 4}


def rotary_plan(rotary, theta=10000.0, scaling=None, neighbours=False, sections=None, frequencies=None, magnitude=None, device="cuda"):
    """A RotaryPlan of the first `rotary` dimensions of a head, with frequencies
    theta^(-2j / rotary) scaled by `scaling` (a model config's dict: rope_type
    "default", "linear", "ntk", "yarn" or "wavelength", factor,
    original_max_position_embeddings, and the turns between which "yarn"
    (beta_slow, beta_fast) and "wavelength" (low_freq_factor, high_freq_factor)
    blend; attention_factor sets the magnitude: fp8lin_rotary_frequencies has
    the formulas), or with the given `frequencies` (rotary / 2 numbers, radians
    per position).  sections: the config's mrope_section of three axes (pair j
    takes axis 1 where j % 3 == 1 and j < 3 sections[1], axis 2 where j % 3 == 2
    and j < 3 sections[2], else axis 0)."""
    rotary = int(rotary)
    if rotary <= 0 or rotary % 2:
        _fail(ERR_SHAPE, "A rotary plan needs an even, positive number of dimensions")
    half = rotary // 2
    freq, mag = (ctypes.c_double * half)(), ctypes.c_double(1.0)
    if frequencies is not None:
        values = [float(f) for f in frequencies]
        if len(values) != half or scaling is not None:
            _fail(ERR_ARGUMENT, "A rotary plan takes rotary / 2 frequencies, or a scaling")
        freq[:] = values
    else:
        scaling = scaling or {}
        kind = scaling.get("rope_type", scaling.get("type", "default"))
        if kind not in _SCALINGS:
            _fail(ERR_ARGUMENT, f"Unknown rotary scaling {kind!r}: one of {', '.join(_SCALINGS)}")
        low, high = [scaling.get(n) or 0.0 for n in (("low_freq_factor", "high_freq_factor") if kind == "wavelength" else ("beta_slow", "beta_fast"))]
        check(lib().fp8lin_rotary_frequencies(rotary, float(theta), _SCALINGS[kind], float(scaling.get("factor", 1.0)),
                                              float(scaling.get("original_max_position_embeddings", 0.0)), float(low), float(high), freq,
                                              ctypes.byref(mag)))
        if scaling.get("attention_factor") is not None:
            mag.value = float(scaling["attention_factor"])
    if magnitude is not None:
        mag.value = float(magnitude)
    axes = None
    if sections is not None:
        if len(sections) != 3:
            _fail(ERR_ARGUMENT, "Sections are of three axes")
        axes = (ctypes.c_int32 * half)(*[j % 3 if j % 3 and j < 3 * int(sections[j % 3]) else 0 for j in range(half)])
    steps = torch.empty(half, dtype=torch.int64)
    check(lib().fp8lin_rotary_steps(freq, axes, half, ctypes.c_void_p(steps.data_ptr())))
    return RotaryPlan(steps.to(device), mag.value, bool(neighbours))


def plan_record(plan, device):
    """The library's record of a plan whose steps are on the device."""
    steps = plan[0] if isinstance(plan, RotaryPlan) else None
    if not (isinstance(steps, torch.Tensor) and steps.dtype is torch.int64 and steps.dim() == 1 and steps.is_contiguous() and
            steps.device == device):
        _fail(ERR_ARGUMENT, "Rotation expects a RotaryPlan on the tensors' device")
    return RotaryRecord(steps.data_ptr(), 2 * steps.size(0), bool(plan[2]), float(plan[1]))


def positions_of(positions, tokens, device):
    """(axes, elements between them, pointer) of positions int64 [tokens] or [axes, tokens], a row contiguous."""
    shape = positions.shape if isinstance(positions, torch.Tensor) else ()
    if not (1 <= len(shape) <= 2 and positions.dtype is torch.int64 and positions.device == device and shape[-1] == tokens and
            (tokens <= 1 or positions.stride(-1) == 1)):
        _fail(ERR_ARGUMENT, "Rotation expects int64 positions [tokens] or [axes, tokens]")
    if len(shape) == 1:
        return 1, 0, positions.data_ptr()
    return shape[0], positions.stride(0) if shape[0] > 1 else 0, positions.data_ptr()


def rotate(x, positions, plan, transposed=False, out=None):
    """x (BF16 [tokens, heads, head_dim], last dimension contiguous) rotated by a
    RotaryPlan at positions (int64 [tokens] or [axes, tokens]) (fp8lin_rotate);
    transposed: turned back (times the magnitude), which is also the gradient
    with respect to x of one with respect to the result.  Returns BF16 [tokens,
    heads, head_dim]: `out` if given, which may be x and overlaps no other input."""
    if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dim() == 3 and x.dtype is torch.bfloat16 and x.stride(2) == 1):
        _fail(ERR_ARGUMENT, "Rotation expects BF16 heads [tokens, heads, head_dim]")
    device, (tokens, heads, dim) = x.device, x.shape
    record = plan_record(plan, device)
    axes, axis, at = positions_of(positions, tokens, device)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif not (isinstance(out, torch.Tensor) and out.shape == x.shape and out.dtype is torch.bfloat16 and out.device == device and
              out.stride(2) == 1):
        _fail(ERR_ARGUMENT, "Rotation expects a BF16 output as the input")
    xs, os = x.stride(), out.stride()
    call("fp8lin_rotate", device, ctypes.byref(record), x.data_ptr(), xs[0], xs[1], tokens, heads, dim, at, axes, axis, bool(transposed),
         out.data_ptr(), os[0], os[1])
    return out
