"""The angle of a rotation on the GPU at positions up to the ends of their type.

Pairs whose rotated value is next to 0 (x_a cos = x_b sin): what is left is the
angle's error times the pair's length, which an output in BF16 shows in full,
where any other value's rounding hides it."""
import math

import pytest
import torch

import rotary_oracle as RO
from test_gpu_rotary import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("position", [1, -1, 1500001, (1 << 40) + 1, 2 ** 63 - 1, -2 ** 63 + 1])
def test_angle_where_a_pair_cancels(fp8lin, gpu, position, neighbours):
    g = torch.Generator().manual_seed(abs(position) % 1000003)
    half = 64
    for _ in range(5):
        x = torch.randn(1, 1, 2 * half, generator=g).to(torch.bfloat16)
        pairs = [RO.pair(j, half, neighbours) for j in range(half)]
        # the phase that turns x_a to 0, at this position: an odd number has an inverse modulo 2^64
        phases = [round(math.atan2(float(x[0, 0, a]), float(x[0, 0, b])) / (2 * math.pi) * 2 ** 64) for a, b in pairs]
        steps = [p * pow(position % 2 ** 64, -1, 2 ** 64) % 2 ** 64 for p in phases]
        plan = fp8lin.RotaryPlan(torch.tensor([s - 2 ** 64 if s >= 2 ** 63 else s for s in steps], dtype=torch.int64).to(gpu), 1.0, neighbours)
        got = fp8lin.rotate(x.to(gpu), torch.tensor([position], device=gpu), plan)
        want, reach = x.double(), torch.zeros(x.shape, dtype=torch.float64)
        for (a, b), s in zip(pairs, steps):
            angle = 2 * math.pi * (position * s % 2 ** 64) / 2 ** 64
            u, v = float(x[0, 0, a]), float(x[0, 0, b])
            want[0, 0, a], want[0, 0, b] = u * math.cos(angle) - v * math.sin(angle), v * math.cos(angle) + u * math.sin(angle)
            reach[0, 0, a] = reach[0, 0, b] = abs(u) + abs(v)
        assert all(abs(float(want[0, 0, a])) < 1e-14 * float(reach[0, 0, a]) for a, _ in pairs)
        check(got, want, RO.row_bound(want, reach, False))
