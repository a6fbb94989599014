"""Dimensions behind the rotated ones, on the GPU: as they are, bit for bit,
whatever the others of their group of pairs hold (infinities, NaN, zeros below 0).

A pair that is not turned must not be multiplied by a turn of 0 either: 0 times
an infinity is NaN, and -0 + 0 is 0."""
import math

import pytest
import torch

import rotary_oracle as RO
from test_gpu_rotary import check, plan_of

pytestmark = pytest.mark.gpu

ODD = [math.inf, -math.inf, math.nan, -0.0, 3.3e38, 0.0]
# head_dim, rotary: groups of 8 pairs that end in ones that are not turned, and (64 of 256, 16 of 48) that do not
SHAPES = [(16, 8), (16, 4), (48, 20), (64, 20), (96, 24), (256, 84), (6, 4), (50, 22), (48, 16), (256, 64)]


def rows(tokens, heads, dim, rotary, seed):
    """Heads whose dimensions behind the rotated ones hold ODD values, each head one more of them than the last."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g).to(torch.bfloat16)
    for t in range(tokens):
        for h in range(heads):
            for i in range((t + h) % len(ODD) + 1):
                d = rotary + int(torch.randint(0, dim - rotary, (1,), generator=g))
                x[t, h, d] = ODD[(t + i) % len(ODD)]
    return x


def same(got, want):
    """Bit for bit, but for the payload of NaN."""
    odd = want.float().isnan()
    assert torch.equal(got.float().isnan(), odd)
    whole = torch.int16 if want.element_size() == 2 else torch.uint8
    assert torch.equal(got.view(whole)[~odd], want.view(whole)[~odd])


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("dim,rotary", SHAPES)
def test_rotate_leaves_them(fp8lin, gpu, dim, rotary, neighbours):
    plan, how = plan_of(fp8lin, gpu, rotary, neighbours=neighbours, magnitude=1.25)
    x = rows(7, 5, dim, rotary, dim + rotary)
    at = torch.tensor([0, 1, 2, 3, 1000, 65537, 1 << 20])
    for transposed in (False, True):
        got = fp8lin.rotate(x.to(gpu), at.to(gpu), plan, transposed=transposed).cpu()
        same(got[..., rotary:], x[..., rotary:])
        y, reach = RO.rotate(x, at, transposed=transposed, **how)
        y, reach = y[..., :rotary], reach[..., :rotary]
        check(got[..., :rotary], y, RO.row_bound(y, reach, False))


@pytest.mark.parametrize("kind", ["bf16", "heads", "blocks"])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("dim,rotary", [(16, 8), (64, 20), (96, 24), (256, 84), (256, 64)])
def test_append_leaves_them(fp8lin, gpu, dim, rotary, neighbours, kind):
    """Queries, and keys of one row, a few and many rows a block, without a norm: what lies behind comes to the cache as a value does,
    rounded once, an infinity as the largest code, NaN as NaN."""
    plan, _ = plan_of(fp8lin, gpu, rotary, neighbours=neighbours)
    page, heads, hk = 64, 3, 2
    slots = [5] + list(range(64, 67)) + list(range(130, 170))
    t = len(slots)
    q, k = rows(t, heads, dim, rotary, 1), rows(t, hk, dim, rotary, 2)
    if kind == "blocks":  # 3.3e38 in a block would leave nothing of the others
        k = torch.where(k.float().abs() > 1e30, torch.where(k.isinf() | k.isnan(), k, torch.ones_like(k)), k)
    v = torch.randn(t, hk, dim, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    dtype = torch.bfloat16 if kind == "bf16" else torch.float8_e4m3fn
    caches = [torch.zeros(3, page, hk, dim, dtype=dtype, device=gpu) for _ in range(2)]
    scale = {}
    if kind == "heads":
        scale = {n: torch.tensor([0.5, 0.0078125], device=gpu) for n in ("k_scale", "v_scale")}
    elif kind == "blocks":
        scale = {n: torch.zeros(3, 1, hk, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu) for n in ("k_scale", "v_scale")}
    at = torch.arange(t) * 97
    got = fp8lin.paged_rotate_append(q.to(gpu), k.to(gpu), v.to(gpu), at.to(gpu), torch.tensor(slots, device=gpu), *caches, plan, **scale).cpu()
    same(got[..., rotary:], q[..., rotary:])
    have = caches[0].cpu().flatten(0, 1)[slots][..., rotary:]
    want = k[..., rotary:]
    if kind != "bf16":
        by = scale["k_scale"].cpu()[:, None] if kind == "heads" else \
            torch.exp2(scale["k_scale"].view(torch.uint8).cpu().float() - 127)[[s // page for s in slots], 0][..., None]
        want = (want.float() / by).clamp(-448, 448).to(dtype)
    same(have, want)
