"""Rotation by positions and the append with block scales in 64 bits, written
from their definitions with loops over pairs, rows and blocks, on the CPU."""
import math

import torch

BF16_HALF = torch.finfo(torch.bfloat16).eps / 2
F32_HALF = torch.finfo(torch.float32).eps / 2
E4M3_HALF = torch.finfo(torch.float8_e4m3fn).eps / 2
E4M3_SMALL = 2.0 ** -10  # half the step of the codes below 2^-6


def frequencies(rotary, theta, scaling=None):
    """([rotary / 2] radians per position, magnitude)."""
    scaling = scaling or {}
    kind, s = scaling.get("rope_type", "default"), scaling.get("factor", 1.0)
    length = scaling.get("original_max_position_embeddings")
    got, magnitude = [], 1.0
    for j in range(rotary // 2):
        f = theta ** (-2 * j / rotary)
        if kind == "linear":
            f = f / s
        elif kind == "ntk":
            f = (theta * s ** (rotary / max(rotary - 2, 1))) ** (-2 * j / rotary)
        elif kind == "wavelength":
            low, high = scaling.get("low_freq_factor", 1), scaling.get("high_freq_factor", 4)
            turns = length * f / (2 * math.pi)
            kept = min(max((turns - low) / (high - low), 0), 1)
            f = f * kept + f / s * (1 - kept)
        elif kind == "yarn":
            slow, fast = scaling.get("beta_slow", 1), scaling.get("beta_fast", 32)
            first, last = [rotary * math.log(length / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (fast, slow)]
            first, last = max(math.floor(first), 0), min(math.ceil(last), rotary - 1)
            stretched = min(max((j - first) / max(last - first, 0.001), 0), 1)
            f = f * (1 - stretched) + f / s * stretched
            magnitude = 0.1 * math.log(s) + 1
        got.append(f)
    return got, magnitude


def steps(freq, axes=None):
    """The plan's integers, by exact fractions of the frequency's turns."""
    got = []
    for j, f in enumerate(freq):
        turns = f / (2 * math.pi)
        at = round((turns - math.floor(turns)) * 2 ** 62) * 4 + (axes[j] if axes else 0)
        got.append(at % 2 ** 64)
    return got


def pair(j, half, neighbours):
    return (2 * j, 2 * j + 1) if neighbours else (j, j + half)


def rotate(x, positions, freq, magnitude=1.0, neighbours=False, axes=None, transposed=False):
    """(y, reach): x [tokens, heads, dim] rotated in 64 bits, and magnitude (|x_a| + |x_b|) of each value's pair (0 behind the pairs).
    positions [tokens] or [axes, tokens]; angles by whole-number arithmetic modulo a turn (2^-75)."""
    x = x.double()
    y, reach = x.clone(), torch.zeros_like(x)
    rows = positions.tolist() if positions.dim() == 2 else [positions.tolist()]
    for j, f in enumerate(freq):
        a, b = pair(j, len(freq), neighbours)
        unit = round(f / (2 * math.pi) * 2 ** 75)
        at = rows[min(axes[j] if axes else 0, len(rows) - 1)]
        angle = torch.tensor([2 * math.pi * ((p * unit) % 2 ** 75) / 2 ** 75 for p in at], dtype=torch.float64)[:, None]
        c, s = magnitude * torch.cos(angle), magnitude * torch.sin(angle) * (-1 if transposed else 1)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        reach[..., a] = reach[..., b] = abs(magnitude) * (x[..., a].abs() + x[..., b].abs())
    return y, reach


def norm(x, weight, eps, centered=True):
    x = x.double()
    if weight is None:
        return x
    w = weight.double() + (1 if centered else 0)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w


# Half steps of FP32 that a rotated value may be off, of its pair's reach: the angle's conversion to FP32 and the constant (2, of at
# most pi / 4), the series' next term (under 1) and its evaluation (3), the magnitude's own rounding and its product (2), the products
# and the sum (3).  And of a normed value: half of the sum of squares (at most 16 terms in a row and 6 joins: 11), its scaling and eps (2), the
# reciprocal root (2), the weight, its product and the value's (3).
TURN, NORM = 11, 18


def row_bound(y, reach, normed):
    """How far the FP32 value may be from y."""
    flat = torch.where(reach > 0, reach, y.abs())
    return 1.01 * F32_HALF * flat * (TURN + (NORM if normed else 0)) if normed else 1.01 * F32_HALF * reach * TURN


def power(top):
    """The exponent of the least 2^e, e of -120 .. 119, with top <= 448 2^e."""
    e = -120
    while top > 448.0 * 2.0 ** e and e < 119:
        e += 1
    return e


def append_blocks(rows, bounds, slots, cache, powers, block):
    """rows [tokens, heads, dim] (64 bits, each off by at most bounds) into cache (codes [pages, page, heads, dim], float8) with the bytes
    powers [pages, blocks, heads]: (values of the codes before their rounding [pages, page, heads, dim], bound of them, bytes, other bytes
    that rounding may give).  Rows of one block stand side by side."""
    pages, page, heads, dim = cache.shape
    flat = cache.double().reshape(pages * page, heads, dim).clone()
    off = torch.zeros_like(flat)
    bytes_ = powers.reshape(-1, heads).int().clone()
    other = bytes_.clone()
    t = 0
    while t < len(slots):
        if not 0 <= slots[t] < pages * page:
            t += 1
            continue
        at, end = slots[t] // block, t
        while end < len(slots) and 0 <= slots[end] < pages * page and slots[end] // block == at:
            end += 1
        mine = {slots[i]: i for i in range(t, end)}
        fresh = any(s % block == 0 for s in mine)
        for h in range(heads):
            x = rows[t:end, h]
            fine = torch.isfinite(x)
            tops = [float((x.abs() + d * bounds[t:end, h])[fine].max()) if bool(fine.any()) else 0.0 for d in (-1, 0, 1)]
            low, e, high = [power(max(v, 0.0)) for v in tops]
            old = int(bytes_[at, h]) - 127
            if not fresh:
                low, e, high = max(low, old), max(e, old), max(high, old)
                for s in range(at * block, (at + 1) * block):
                    if s not in mine:
                        flat[s, h] *= 2.0 ** (old - e)
            bytes_[at, h] = e + 127
            other[at, h] = (high if high != e else low) + 127
            for s, i in mine.items():
                flat[s, h] = (rows[i, h] * 2.0 ** -e).clamp(-448, 448)
                off[s, h] = bounds[i, h] * 2.0 ** -e
        t = end
    return flat.view(cache.shape), off.view(cache.shape), bytes_.view(powers.shape), other.view(powers.shape)


def code_bound(values, off):
    """How far a code may be from the value that it rounds: the value's own error and half a step."""
    return off * 1.01 + (values.abs() + off) * E4M3_HALF + E4M3_SMALL
