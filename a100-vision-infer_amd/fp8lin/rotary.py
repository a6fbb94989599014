"""Rotary positions: plans of frequencies, scaled for long contexts or not, and
the rotation of heads by them (include/fp8lin.h describes the operators).

`fused_rope` and `qk_norm_rope` are the reference's form: half layout, FP32
angles, BF16 between the products.  Here pairs are halves or neighbours, a
position times a plan's step is exact modulo a turn (a step is its frequency in
units of 2^-62 turns a position), and the result is rounded once.
"""
import ctypes
import math
from collections import namedtuple
from collections.abc import Mapping

import torch

from ._lib import ERR_ARGUMENT, ERR_SHAPE, RotaryRecord, check, lib
from .ops import _fail, call

RotaryPlan = namedtuple("RotaryPlan", "steps magnitude neighbours")
RotaryPlan.__doc__ = """What rotates heads: steps int64 [rotary / 2] on the device (4 * round(frequency / 2 pi * 2^62) + axis of each pair, as
rotary_plan makes them), magnitude of the cosines and sines, and whether pairs are neighbours (2j, 2j + 1) or halves (j, j + rotary / 2)."""

_SCALINGS = {"default": 0, "linear": 1, "ntk": 2, "yarn": 3, "wavelength": 4}
# A config's keys that a plan of any kind reads, and those that its kind reads beside them.
_KEYS = {"rope_type", "type", "attention_factor", "original_max_position_embeddings", "rope_theta", "partial_rotary_factor", "mrope_section",
         "mrope_interleaved"}
_KEYS_OF = {"default": set(), "linear": {"factor"}, "ntk": {"factor"},
            "yarn": {"factor", "beta_slow", "beta_fast", "mscale", "mscale_all_dim", "truncate"},
            "wavelength": {"factor", "low_freq_factor", "high_freq_factor"}}


def _read_scaling(scaling):
    """(kind, the dict without its null values): every key is one that the kind reads."""
    if not isinstance(scaling, Mapping):
        _fail(ERR_ARGUMENT, "A rotary scaling is a dict")
    scaling = {key: value for key, value in scaling.items() if value is not None}
    kinds = [scaling[key] for key in ("rope_type", "type") if key in scaling] or ["default"]
    kind = kinds[0]
    if not isinstance(kind, str) or kind not in _SCALINGS or kinds[-1] != kind:
        _fail(ERR_ARGUMENT, f"Unknown rotary scaling {' and '.join(map(repr, kinds))}: one of {', '.join(_SCALINGS)}")
    unread = [str(key) for key in scaling if key not in _KEYS and key not in _KEYS_OF[kind]]
    if unread:
        _fail(ERR_ARGUMENT, f"A rotary scaling {kind!r} does not read {', '.join(unread)} (frequencies= and magnitude= take any form)")
    if not scaling.get("truncate", True):
        _fail(ERR_ARGUMENT, "A rotary scaling 'yarn' rounds its borders to whole pairs: truncate must be true (frequencies= takes any form)")
    if kind != "default" and "factor" not in scaling:
        _fail(ERR_ARGUMENT, f"A rotary scaling {kind!r} needs a factor")
    if ("mscale" in scaling) != ("mscale_all_dim" in scaling) or ("mscale" in scaling and "attention_factor" in scaling):
        _fail(ERR_ARGUMENT, "A rotary scaling's magnitude is its attention_factor, or mscale and mscale_all_dim")
    return kind, scaling


def _number(scaling, key, default=None, positive=False):
    try:
        value = float(scaling.get(key, default))
    except (TypeError, ValueError):
        value = math.nan
    if math.isnan(value) or (positive and not 0 < value < math.inf):
        _fail(ERR_ARGUMENT, f"A rotary scaling's {key} must be a {'positive ' if positive else ''}number")
    return value


def _sections_of(scaling, sections):
    """The sections: the argument's, or the dict's, which have to be the same."""
    lists = [s for s in (sections, scaling.get("mrope_section")) if s is not None]
    try:
        lists = [[int(n) for n in s] for s in lists]
    except (TypeError, ValueError):
        lists = [[]]
    if any(len(s) != 3 or s != lists[0] for s in lists):
        _fail(ERR_ARGUMENT, "Sections are of three axes, and the config's are those given")
    if not scaling.get("mrope_interleaved", sections is not None or not lists):
        _fail(ERR_ARGUMENT, "Sections are interleaved: mrope_interleaved must be true, or the sections given")
    return lists[0] if lists else None


def rotary_plan(rotary, theta=None, scaling=None, neighbours=False, sections=None, frequencies=None, magnitude=None, device="cuda", head_dim=None):
    """A RotaryPlan of the first `rotary` dimensions of a head, with frequencies
    theta^(-2j / rotary) (theta: by default the config's rope_theta, or 10000)
    scaled by `scaling`, a model config's dict, or with the given `frequencies`
    (rotary / 2 numbers, radians per position).  fp8lin_rotary_frequencies has
    the formulas.  The dict's keys, null ones being those that are not there:
    - rope_type (or type) "default", "linear", "ntk", "yarn" or "wavelength",
      and for all but the first its factor;
    - original_max_position_embeddings, and the turns between which "yarn"
      (beta_slow, beta_fast) and "wavelength" (low_freq_factor,
      high_freq_factor) blend;
    - the magnitude of a plan, unless `magnitude` is given: attention_factor, or
      of "yarn" mscale and mscale_all_dim together, the ratio of the two
      magnitudes 0.1 mscale ln(factor) + 1;
    - rope_theta and mrope_section, which may not differ from the arguments, and
      partial_rotary_factor: with head_dim given, rotary has to be that part of
      it (without, that is the caller's to see to);
    - what has one form here: truncate true, mrope_interleaved true (needed
      where the dict has sections and the call none).
    Any other key is refused, as it may change the formula.
    sections: the config's mrope_section of three axes (pair j takes axis 1
    where j % 3 == 1 and j < 3 sections[1], axis 2 where j % 3 == 2 and j < 3
    sections[2], else axis 0)."""
    rotary = int(rotary)
    if rotary <= 0 or rotary % 2:
        _fail(ERR_SHAPE, "A rotary plan needs an even, positive number of dimensions")
    half = rotary // 2
    freq, mag = (ctypes.c_double * half)(), ctypes.c_double(1.0)
    if frequencies is not None and scaling is not None:
        _fail(ERR_ARGUMENT, "A rotary plan takes rotary / 2 frequencies, or a scaling")
    kind, scaling = _read_scaling({} if scaling is None else scaling)
    sections = _sections_of(scaling, sections)
    part = _number(scaling, "partial_rotary_factor", 1.0, positive=True)
    if part > 1 or (head_dim is not None and (rotary > head_dim or ("partial_rotary_factor" in scaling and rotary != int(head_dim * part)))):
        _fail(ERR_SHAPE, "A rotary plan's dimensions are not the config's partial_rotary_factor of the head's")
    if frequencies is not None:
        values = [float(f) for f in frequencies]
        if len(values) != half:
            _fail(ERR_ARGUMENT, "A rotary plan takes rotary / 2 frequencies, or a scaling")
        freq[:] = values
    else:
        base = _number(scaling, "rope_theta", 10000.0 if theta is None else theta, positive=True)
        if theta is not None and float(theta) != base:
            _fail(ERR_ARGUMENT, "A rotary plan's theta is not the config's rope_theta")
        low, high = ("low_freq_factor", "high_freq_factor") if kind == "wavelength" else ("beta_slow", "beta_fast")
        # 0: the usual border, which a dict cannot ask for
        low, high = [_number(scaling, key, positive=True) if key in scaling else 0.0 for key in (low, high)]
        factor = _number(scaling, "factor", 1.0)
        check(lib().fp8lin_rotary_frequencies(rotary, base, _SCALINGS[kind], factor, _number(scaling, "original_max_position_embeddings", 0.0), low, high,
                                              freq, ctypes.byref(mag)))
        if "attention_factor" in scaling:
            mag.value = _number(scaling, "attention_factor")
        elif "mscale" in scaling:
            of, all_dim = [0.1 * _number(scaling, key, positive=True) * math.log(max(factor, 1.0)) + 1 for key in ("mscale", "mscale_all_dim")]
            mag.value = of / all_dim
    if magnitude is not None:
        mag.value = float(magnitude)
    axes = None
    if sections is not None:
        axes = (ctypes.c_int32 * half)(*[j % 3 if j % 3 and j < 3 * sections[j % 3] else 0 for j in range(half)])
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
