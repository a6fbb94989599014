"""Rotation, rotated append and caches with block scales on the GPU against
their plain 64-bit forms (rotary_oracle): values within a bound that counts
their roundings, scales and untouched memory exactly."""
import math
import random

import pytest
import torch

import paged_oracle as PO
import rotary_oracle as RO

pytestmark = pytest.mark.gpu


def plan_of(fp8lin, dev, rotary, theta=10000.0, scaling=None, neighbours=False, axes=None, magnitude=None):
    """(plan, oracle's arguments): the steps are the oracle's own."""
    freq, mag = RO.frequencies(rotary, theta, scaling)
    mag = mag if magnitude is None else magnitude
    steps = torch.tensor([s - 2 ** 64 if s >= 2 ** 63 else s for s in RO.steps(freq, axes)], dtype=torch.int64)
    return fp8lin.RotaryPlan(steps.to(dev), mag, neighbours), dict(freq=freq, magnitude=mag, neighbours=neighbours, axes=axes)


def check(got, y, bound, what=""):
    err = (got.double().cpu() - y).abs() - bound - RO.BF16_HALF * (y.abs() + bound) * 1.01 - 1e-38
    assert torch.isfinite(got.float()).all() and float(err.max()) <= 0, f"{what}: {float(err.max())} beyond the bound"


SHAPES = [(1, 1, 64, 64), (1, 24, 256, 64), (5, 3, 128, 128), (37, 8, 128, 64), (3, 5, 80, 80), (9, 7, 96, 20), (2, 1, 16, 16), (65, 12, 256, 64),
          (4, 2, 1024, 512), (7, 3, 6, 4), (3, 2, 2, 2), (6, 40, 64, 32), (11, 2, 528, 528), (130, 33, 32, 32), (2, 3, 250, 62)]


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rotate(fp8lin, gpu, shape, neighbours):
    tokens, heads, dim, rotary = shape
    rng = random.Random(f"{shape}{neighbours}")
    g = torch.Generator().manual_seed(rng.randrange(1 << 20))
    axes = [rng.randrange(3) for _ in range(rotary // 2)] if rng.random() < 0.5 else None
    plan, how = plan_of(fp8lin, gpu, rotary, rng.choice([1e4, 1e7]), neighbours=neighbours, axes=axes)
    x = torch.randn(tokens, heads, dim, generator=g).to(torch.bfloat16)
    at = torch.randint(0, 1 << rng.choice([4, 12, 20, 30]), (3, tokens) if axes else (tokens,), generator=g)
    for transposed in (False, True):
        y, reach = RO.rotate(x, at, transposed=transposed, **how)
        got = fp8lin.rotate(x.to(gpu), at.to(gpu), plan, transposed=transposed)
        check(got, y, RO.row_bound(y, reach, False))
        assert torch.equal(got.cpu()[..., rotary:], x[..., rotary:])


@pytest.mark.parametrize("scaling", ["linear", "ntk", "yarn", "wavelength"])
def test_rotate_scaled_far_positions(fp8lin, gpu, scaling):
    """A library plan, positions up to the ends of their type (also below 0)."""
    g = torch.Generator().manual_seed(2)
    scaling = {"rope_type": scaling, "factor": 8.0, "original_max_position_embeddings": 32768}
    plan = fp8lin.rotary_plan(64, 10000000.0, scaling, device=gpu)
    freq, mag = RO.frequencies(64, 10000000.0, scaling)
    x = torch.randn(8, 4, 128, generator=g).to(torch.bfloat16)
    at = torch.tensor([0, 1, 31, 65537, 1500001, (1 << 24) + 1, 1 << 26, -77])
    # the library's powers may be 64 half steps of 2^-53 from the oracle's: of the turns that the position makes
    turns = at.abs().double()[:, None, None] * max(freq) / (2 * math.pi) * 64 * 2 ** -53 * 2 * math.pi
    y, reach = RO.rotate(x, at, freq, mag)
    check(fp8lin.rotate(x.to(gpu), at.to(gpu), plan), y, RO.row_bound(y, reach, False) + turns * reach)
    # with the plan's own integers the angle is exact at any position
    plan, how = plan_of(fp8lin, gpu, 4, 1e4)
    at = torch.tensor([2 ** 63 - 1, -2 ** 63, 2 ** 62 + 12345, -1, 10 ** 15, 7, 0, 2 ** 40 + 1])
    steps = [s % 2 ** 64 for s in plan.steps.tolist()]
    want = x.double().clone()
    reach = torch.zeros_like(want)
    for j, s in enumerate(steps):
        angle = torch.tensor([2 * math.pi * ((p * s) % 2 ** 64) / 2 ** 64 for p in at.tolist()], dtype=torch.float64)[:, None]
        a, b = x[..., j].double(), x[..., j + 2].double()
        want[..., j], want[..., j + 2] = a * torch.cos(angle) - b * torch.sin(angle), b * torch.cos(angle) + a * torch.sin(angle)
        reach[..., j] = reach[..., j + 2] = a.abs() + b.abs()
    check(fp8lin.rotate(x.to(gpu), at.to(gpu), plan), want, RO.row_bound(want, reach, False))


@pytest.mark.parametrize("pad", [0, 1, 3, 8])
def test_rotate_views(fp8lin, gpu, pad):
    """Views off 16 bytes, transposed layouts, in place, an output beside its input; what lies around stays."""
    g = torch.Generator().manual_seed(3)
    plan, how = plan_of(fp8lin, gpu, 64)
    t, h, d = 13, 5, 128
    at = torch.randint(0, 9999, (t,), generator=g)
    wide = torch.randn(t, h, 2 * d + 2 * pad, generator=g).to(torch.bfloat16)
    x = wide[..., pad:pad + d]
    y, reach = RO.rotate(x, at, **how)
    bound = RO.row_bound(y, reach, False)
    up = wide.to(gpu)
    view = up[..., pad:pad + d]
    check(fp8lin.rotate(view, at.to(gpu), plan), y, bound)
    out = torch.full((h, t, d + pad), 7.0, dtype=torch.bfloat16, device=gpu)
    got = fp8lin.rotate(view, at.to(gpu), plan, out=out.transpose(0, 1)[..., pad:])
    check(got, y, bound)
    assert (out[..., :pad] == 7.0).all() and torch.equal(up.cpu(), wide)
    got = fp8lin.rotate(view, at.to(gpu), plan, out=view)
    assert got.data_ptr() == view.data_ptr()
    check(view, y, bound)
    keep = up.cpu()
    keep[..., pad:pad + d] = x
    assert torch.equal(keep, wide)
    # heads that a token shares (a stride of 0), positions of one row expanded over the axes
    many = wide.to(gpu)[:, :1, pad:pad + d].expand(t, 4, d)
    got = fp8lin.rotate(many, at.to(gpu)[None].expand(3, t), plan)
    for i in range(4):
        check(got[:, i], y[:, 0], bound[:, 0])


def test_rotate_positions_of_fewer_axes(fp8lin, gpu):
    """A pair whose axis the positions do not have takes the last one."""
    g = torch.Generator().manual_seed(4)
    axes = [0, 1, 2, 3] * 2
    plan, how = plan_of(fp8lin, gpu, 16, axes=axes)
    x = torch.randn(6, 2, 16, generator=g).to(torch.bfloat16)
    for n in (1, 2, 3, 4):
        at = torch.randint(0, 1000, (n, 6), generator=g)
        y, reach = RO.rotate(x, at, **{**how, "axes": [min(a, n - 1) for a in axes]})
        check(fp8lin.rotate(x.to(gpu), at.to(gpu), plan), y, RO.row_bound(y, reach, False))


def test_rotate_values(fp8lin, gpu):
    """Infinities and NaN stay in their pairs; the largest values do not overflow on the way of a turn of 0."""
    plan, _ = plan_of(fp8lin, gpu, 8)
    x = torch.ones(1, 1, 16, dtype=torch.bfloat16)
    x[0, 0, 1], x[0, 0, 6], x[0, 0, 9] = math.nan, math.inf, 3.3e38
    got = fp8lin.rotate(x.to(gpu), torch.tensor([5], device=gpu), plan).cpu()[0, 0]
    assert torch.isnan(got[[1, 5]]).all() and not torch.isfinite(got[[2, 6]]).any()
    assert torch.isfinite(got[[0, 3, 4, 7]]).all() and torch.equal(got[8:], x[0, 0, 8:])
    big = torch.full((1, 1, 8), 3.3e38, dtype=torch.bfloat16)
    assert torch.equal(fp8lin.rotate(big.to(gpu), torch.tensor([0], device=gpu), plan).cpu(), big)


def test_rotate_gradient(fp8lin, gpu):
    """The transposed rotation of a gradient, against differences of the rotation in 64 bits."""
    g = torch.Generator().manual_seed(5)
    plan, how = plan_of(fp8lin, gpu, 12, magnitude=1.25, neighbours=True)
    x, w = [torch.randn(3, 2, 20, generator=g).to(torch.bfloat16) for _ in range(2)]
    at = torch.tensor([2, 900, 123456])
    got = fp8lin.rotate(w.to(gpu), at.to(gpu), plan, transposed=True)
    want = torch.zeros(x.numel(), dtype=torch.float64)
    for i in range(x.numel()):
        d = torch.zeros(x.numel(), dtype=torch.float64)
        d[i] = 2.0 ** -10
        up, down = [(RO.rotate(x.double() + e * d.view(x.shape), at, **how)[0] * w.double()).sum() for e in (1, -1)]
        want[i] = (up - down) / 2 ** -9
    _, reach = RO.rotate(w, at, transposed=True, **how)
    check(got, want.view(x.shape), RO.row_bound(want.view(x.shape), reach, False) + 1e-10)


def test_rotate_past_32_bits(fp8lin, gpu):
    """More than 2^31 elements between a call's first and last token, and a grid of more than 2^20 workgroups."""
    plan, how = plan_of(fp8lin, gpu, 64)
    t = 1 << 22
    x = torch.empty(t, 1, 1032, dtype=torch.bfloat16, device=gpu)[..., 4:68]
    x.copy_(torch.randn(64, device=gpu).to(torch.bfloat16).expand(t, 1, 64))
    at = torch.arange(t, device=gpu)
    got = fp8lin.rotate(x, at, plan)
    for lo in (0, (1 << 21) + 5, t - 9):
        y, reach = RO.rotate(x[lo:lo + 9].cpu(), at[lo:lo + 9].cpu(), **how)
        check(got[lo:lo + 9], y, RO.row_bound(y, reach, False))
    plan, how = plan_of(fp8lin, gpu, 2)
    x = torch.randn(5 << 20, 1, 1, 2, device=gpu).to(torch.bfloat16).view(-1, 1, 2)
    at = torch.arange(x.size(0), device=gpu)
    got = fp8lin.rotate(x, at, plan)
    for lo in (0, (1 << 22) - 4, x.size(0) - 9):
        y, reach = RO.rotate(x[lo:lo + 9].cpu(), at[lo:lo + 9].cpu(), **how)
        check(got[lo:lo + 9], y, RO.row_bound(y, reach, False))


# ---- append ---------------------------------------------------------------------


class Step:
    """The new rows of requests (length before, new tokens) and a cache that holds what came before them."""

    def __init__(self, fp8lin, dev, held, heads, hk, dim, page, kind, block=16, rotary=None, neighbours=False, norm=True, axes=False, seed=0,
                 big=None, extra=0):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.block, self.dim, self.page = kind, block, dim, page
        need = [-(-(b + c) // page) for b, c in held]
        pages = sum(need) + 3
        ids = torch.randperm(pages, generator=g).tolist()
        self.slots, self.at = [], []
        for b, c in held:
            mine = [ids.pop() for _ in range(-(-(b + c) // page))]
            self.slots += [mine[p // page] * page + p % page for p in range(b, b + c)]
            self.at += list(range(b, b + c))
        self.slots += [-1, pages * page, -5, 1 << 40][:extra]
        self.at += [0] * extra
        t = len(self.slots)
        wide = torch.randn(t, (heads + 2 * hk) * dim + 8, generator=g).to(torch.bfloat16)
        if big is not None:
            wide *= torch.exp2(torch.randint(-big, big + 1, (t, 1), generator=g).float()).to(torch.bfloat16)
        self.wide = wide
        split = lambda w: [w[:, a * dim:(a + n) * dim].unflatten(1, (n, dim)) for a, n in ((0, heads), (heads, hk), (heads + hk, hk))]  # noqa: E731
        self.q, self.k, self.v = split(wide)
        self.up = split(wide.to(dev))
        # cast norms away from 0 and 1
        self.norms = [(0.4 * torch.randn(dim, generator=g)).to(torch.bfloat16) for _ in range(2)] if norm else [None, None]
        self.positions = torch.tensor(self.at)
        ax = None
        if rotary and axes:
            ax = [j % 3 for j in range(rotary // 2)]
            self.positions = torch.stack([self.positions, self.positions // 3, self.positions % 7])
        self.plan, self.how = plan_of(fp8lin, dev, rotary, neighbours=neighbours, axes=ax, magnitude=1.125) if rotary else (None, None)
        kv = [torch.randn(pages, page, hk, dim, generator=g) for _ in range(2)]
        if kind == "bf16":
            self.caches, self.scales = [x.to(torch.bfloat16) for x in kv], [None, None]
        elif kind == "heads":
            self.scales = [0.01 * (1 + torch.randint(0, 4, (hk,), generator=g).float()) for _ in range(2)]
            self.caches = [(x / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn) for x, s in zip(kv, self.scales)]
        else:
            self.scales = [torch.randint(115, 123, (pages, page // block, hk), generator=g).to(torch.uint8) for _ in range(2)]
            self.caches = [(x * 100).to(torch.float8_e4m3fn) for x in kv]
        self.dev = dev
        self.fp8lin = fp8lin

    def scale(self, s):
        return None if s is None else s.to(self.dev).view(torch.float8_e8m0fnu) if self.kind == "blocks" else s.to(self.dev)

    def run(self, **kw):
        caches, scales = [c.to(self.dev) for c in self.caches], [self.scale(s) for s in self.scales]
        q = self.fp8lin.paged_rotate_append(
            *self.up, self.positions.to(self.dev), torch.tensor(self.slots, device=self.dev), *caches, self.plan,
            **{**dict(q_norm=None if self.norms[0] is None else self.norms[0].to(self.dev),
                      k_norm=None if self.norms[1] is None else self.norms[1].to(self.dev), k_scale=scales[0], v_scale=scales[1]), **kw})
        return q, caches, scales

    def rows(self, x, weight, eps=1e-6, centered=True):
        y = RO.norm(x, weight, eps, centered)
        reach = torch.zeros_like(y)
        if self.plan is not None:
            y, reach = RO.rotate(y, self.positions, **self.how)
        return y, RO.row_bound(y, reach, weight is not None)

    def check(self, got, **kw):
        q, caches, scales = got
        y, bound = self.rows(self.q, self.norms[0], **kw)
        check(q, y, bound, "queries")
        for i, (x, w, name) in enumerate(((self.k, self.norms[1], "keys"), (self.v, None, "values"))):
            y, bound = self.rows(x, w, **kw) if i == 0 else (x.double(), torch.zeros(x.shape).double())
            cache = caches[i].cpu()
            if self.kind == "blocks":
                values, off, want, other = RO.append_blocks(y, bound, self.slots, self.caches[i], self.scales[i], self.block)
                have = scales[i].cpu().view(torch.uint8).int()
                assert ((have == want) | (have == other)).all(), name
                # a scale that rounding decides: the codes under the other power of two
                shift = torch.exp2((want - have).double()).repeat_interleave(self.block, 1)[..., None]
                values, off = values * shift, off * shift
                # a NaN code that the cache held stays NaN, under any scale
                odd = torch.isnan(values)
                assert torch.equal(torch.isnan(cache.double()), odd), name
                err = ((cache.double() - values.clamp(-448, 448)).abs() - RO.code_bound(values, off))[~odd]
                assert float(err.max()) <= 0, f"{name}: {float(err.max())}"
                # untouched blocks bit for bit
                touched = {s // self.block for s in self.slots if 0 <= s < cache.size(0) * self.page}
                same = torch.tensor([b not in touched for b in range(cache.size(0) * self.page // self.block)])
                bits = [c.view(torch.uint8).reshape(same.numel(), -1) for c in (cache, self.caches[i])]
                assert torch.equal(bits[0][same], bits[1][same])
                if i == 1:  # values come as they are: bit for bit
                    for b in touched:
                        for s in range(b * self.block, (b + 1) * self.block):
                            if s in self.slots:
                                row = (x[self.slots.index(s)].float() * torch.exp2(127 - have.reshape(-1, have.size(2))[b].float())[:, None])
                                assert torch.equal(cache.reshape(-1, *cache.shape[2:])[s].float(), row.clamp(-448, 448).to(torch.float8_e4m3fn).float())
                continue
            flat = self.caches[i].double().flatten(0, 1)
            err_at = torch.zeros_like(flat)
            for r, s in enumerate(self.slots):
                if 0 <= s < flat.size(0):
                    if self.kind == "heads":
                        sc = self.scales[i].double()[:, None]
                        flat[s] = (y[r] / sc).clamp(-448, 448)
                        err_at[s] = RO.code_bound(flat[s], bound[r] / sc + F32 * flat[s].abs())
                    else:
                        flat[s] = y[r]
                        err_at[s] = bound[r] + RO.BF16_HALF * (y[r].abs() + bound[r]) * 1.01 if i == 0 else torch.zeros_like(y[r])
            err = (cache.double().flatten(0, 1) - flat).abs() - err_at
            assert float(err.max()) <= 0, f"{name}: {float(err.max())}"


F32 = RO.F32_HALF
HELD = {
    "one": [(40, 1)], "first": [(0, 1)], "batch": [(15, 1), (16, 1), (31, 1), (100, 1), (0, 1), (63, 1), (64, 1)],
    "drafts": [(14, 4), (32, 3), (0, 2), (61, 8)], "prompt": [(0, 150)], "chunk": [(37, 120)], "mixed": [(5, 1), (70, 90), (0, 33), (200, 2)],
}


@pytest.mark.parametrize("kind", ["bf16", "heads", "blocks"])
@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("heads", [(12, 2, 256, 64), (8, 8, 64, 64), (4, 1, 128, 32), (3, 3, 80, 20), (2, 1, 1024, 1024), (5, 2, 16, 16)], ids=str)
def test_append(fp8lin, gpu, heads, held, kind):
    rng = random.Random(f"{heads}{held}{kind}")
    page = rng.choice([16, 32, 64, 256])
    h, hk, dim, rotary = heads
    s = Step(fp8lin, gpu, HELD[held], h, hk, dim, page, kind, block=rng.choice([b for b in (16, 32, 64, 128) if b <= page]),
             rotary=rng.choice([rotary, rotary, None]), neighbours=rng.random() < 0.5, norm=rng.random() < 0.6, axes=rng.random() < 0.4,
             seed=rng.randrange(1 << 20), big=rng.choice([None, 6]), extra=rng.choice([0, 4]))
    s.check(s.run())


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_append_long(fp8lin, gpu, block):
    """More rows than a launch's small path takes, blocks whose first row is not their first slot, rows that belong to nobody behind."""
    s = Step(fp8lin, gpu, [(33, 700), (0, 1), (130, 1), (17, 3)], 2, 2, 64, 128, "blocks", block=block, rotary=64, seed=7, big=3, extra=4)
    s.check(s.run())


def test_append_norm_forms(fp8lin, gpu):
    """Weights that are not centered, another eps, one norm without the other."""
    for centered, eps, which in ((False, 1e-2, 2), (True, 0.0, 0), (True, 1e-6, 1)):
        s = Step(fp8lin, gpu, [(20, 30)], 4, 2, 128, 32, "blocks", block=32, rotary=64, seed=8)
        if which < 2:
            s.norms[which] = None
        s.check(s.run(eps=eps, centered=centered), eps=eps, centered=centered)


def test_append_without_rotation_is_paged_append(fp8lin, gpu):
    """Keys and values alone: paged_append over each cache, the same codes."""
    for kind in ("bf16", "heads", "blocks"):
        s = Step(fp8lin, gpu, [(10, 40), (3, 1)], 1, 2, 64, 32, kind, rotary=None, norm=False, seed=9)
        _, caches, scales = s.run()
        again, sc = [c.to(gpu) for c in s.caches], [s.scale(x) for x in s.scales]
        fp8lin.paged_append(s.up[1], s.up[2], torch.tensor(s.slots, device=gpu), *again, k_scale=sc[0], v_scale=sc[1])
        for x, y in zip(caches, again):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        if kind == "blocks":
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(scales, sc))


def test_append_token_by_token(fp8lin, gpu):
    """A prompt in one piece, in pieces and a token at a time: the same scales (the largest value decides), and values that are one
    rounding, or where a block grew two, from the rows'."""
    g = torch.Generator().manual_seed(10)
    t, hk, d, block = 75, 2, 64, 32
    rows = (torch.randn(t, hk, d, generator=g) * torch.exp2(torch.linspace(-8, 8, t))[:, None, None]).to(torch.bfloat16).to(gpu)
    got = []
    for piece in (t, 10, 1):
        cache = [torch.zeros(3, 32, hk, d, dtype=torch.float8_e4m3fn, device=gpu) for _ in range(2)]
        scale = [torch.zeros(3, 1, hk, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu) for _ in range(2)]
        for lo in range(0, t, piece):
            part = rows[lo:lo + piece]
            fp8lin.paged_append(part, part, torch.arange(lo, lo + part.size(0), device=gpu), *cache, k_scale=scale[0], v_scale=scale[1])
        assert torch.equal(cache[0].view(torch.uint8), cache[1].view(torch.uint8))
        power = torch.exp2(scale[0].view(torch.uint8).double() - 127).repeat_interleave(block, 1)[..., None]
        got.append((scale[0].view(torch.uint8).cpu(), (cache[0].double() * power).flatten(0, 1)[:t].cpu(), power.flatten(0, 1)[:t].cpu()))
    for scale, values, power in got:
        assert torch.equal(scale, got[0][0])
        x = rows.double().cpu()
        # one rounding each time the scale grows past a value's 2^-6, at most 17 times; above that one in all
        assert float(((values - x).abs() - x.abs() * RO.E4M3_HALF - 18 * RO.E4M3_SMALL * power).max()) <= 0


def test_append_of_all_rows_to_one_slot(fp8lin, gpu):
    """More rows in a block than it has slots: a scale that holds them all, one of the rows in the slot, nothing else."""
    g = torch.Generator().manual_seed(11)
    rows = torch.randn(300, 1, 64, generator=g).to(torch.bfloat16)
    cache = [torch.zeros(2, 16, 1, 64, dtype=torch.float8_e4m3fn, device=gpu) for _ in range(2)]
    scale = [torch.full((2, 1, 1), 100, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu) for _ in range(2)]
    fp8lin.paged_append(rows.to(gpu), rows.to(gpu), torch.full((300,), 21, device=gpu), *cache, k_scale=scale[0], v_scale=scale[1])
    e = RO.power(float(rows.float().abs().max()))
    assert scale[0].view(torch.uint8).flatten().tolist() == [100, e + 127]
    want = (rows.float() * 2.0 ** -e).to(torch.float8_e4m3fn).float()[:, 0]
    have = cache[0].float().cpu()[1, 5, 0]
    assert ((want[:, None, :] == have).any(0)).all()
    assert (cache[0].float().cpu().flatten(0, 1)[[i for i in range(32) if i != 21]] == 0).all()


def test_append_values(fp8lin, gpu):
    """Infinities at the block's end of range, NaN as NaN, zeros, and the smallest scale."""
    x = torch.zeros(4, 1, 16, dtype=torch.bfloat16)
    x[0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    x[2, 0, 0], x[3, 0, 1] = 1e-39, math.inf
    cache = [torch.full((4, 16, 1, 16), 5.0, device=gpu).to(torch.float8_e4m3fn) for _ in range(2)]
    scale = [torch.full((4, 1, 1), 120, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu) for _ in range(2)]
    fp8lin.paged_append(x.to(gpu), x.to(gpu), torch.tensor([0, 16, 32, 48], device=gpu), *cache, k_scale=scale[0], v_scale=scale[1])
    c = cache[0].float().cpu()
    e = RO.power(3.0)
    assert scale[0].view(torch.uint8).flatten().tolist() == [e + 127, 7, 7, 7]
    assert c[0, 0, 0, :2].tolist() == [448.0, -448.0] and math.isnan(c[0, 0, 0, 2]) and float(c[0, 0, 0, 3]) == 3.0 * 2.0 ** -e
    assert (c[1, 0] == 0).all() and float(c[3, 0, 0, 1]) == 448.0 and float(c[3, 0, 0, 0]) == 0.0
    assert torch.equal(c[2, 0], (x[2].float() * 2.0 ** 120).to(torch.float8_e4m3fn).float()) and float(c[2, 0, 0, 0]) == 2.0 ** -9
    # the largest finite values saturate, as their block's range ends at 448 2^119
    big = torch.full((1, 1, 16), 3.38e38, dtype=torch.bfloat16, device=gpu)
    fp8lin.paged_append(big, -big, torch.tensor([48], device=gpu), *cache, k_scale=scale[0], v_scale=scale[1])
    assert [int(x.view(torch.uint8)[3, 0, 0]) for x in scale] == [246, 246]
    assert [x.float()[3, 0, 0].unique().tolist() for x in cache] == [[448.0], [-448.0]]
    # a later token: the codes of the slots before it, and NaN, under the greater scale
    y = torch.full((1, 1, 16), 1000.0, dtype=torch.bfloat16, device=gpu)
    fp8lin.paged_append(y, y, torch.tensor([1], device=gpu), *cache, k_scale=scale[0], v_scale=scale[1])
    grown = RO.power(1000.0)
    c = cache[0].float().cpu()
    assert int(scale[0].view(torch.uint8)[0, 0, 0]) == grown + 127
    want = (torch.tensor([448.0, -448.0, math.nan, 3.0 * 2.0 ** -e]) * 2.0 ** (e - grown)).to(torch.float8_e4m3fn).float()
    assert torch.equal(c[0, 0, 0, :4].isnan(), want.isnan()) and torch.equal(c[0, 0, 0, :4].nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("bits", [0x7f81, 0x7fc1, 0xff85])
def test_append_nan_beside_large_values(fp8lin, gpu, bits):
    """Quiet and signalling NaN count for nothing in their block's scale, wherever they stand, and stay NaN."""
    g = torch.Generator().manual_seed(15)
    for rows in (1, 3, 40):
        x = torch.randn(rows, 2, 64, generator=g).to(torch.bfloat16)
        x[0, :, 5], x[rows - 1, :, 44] = 70.0, -90.0
        for r, d in ((0, 0), (0, 6), (rows - 1, 43), (rows // 2, 63)):
            x.view(torch.int16)[r, :, d] = bits - (1 << 16 if bits >> 15 else 0)
        cache = [torch.zeros(3, 32, 2, 64, dtype=torch.float8_e4m3fn, device=gpu) for _ in range(2)]
        scale = [torch.full((3, 1, 2), 7, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu) for _ in range(2)]
        fp8lin.paged_append(x.to(gpu), x.to(gpu), torch.arange(rows, device=gpu), *cache, k_scale=scale[0], v_scale=scale[1])
        fine = x.float().nan_to_num(0.0)
        for c, s in zip(cache, scale):
            for lo in range(0, rows, 32):
                e = [RO.power(float(fine[lo:lo + 32, h].abs().max())) for h in range(2)]
                assert s.view(torch.uint8)[lo // 32, 0].tolist() == [p + 127 for p in e]
                want = (x[lo:lo + 32].float() / torch.tensor([2.0 ** p for p in e])[:, None]).to(torch.float8_e4m3fn).float()
                have = c.float().cpu()[lo // 32, :want.size(0)]
                assert torch.equal(have.isnan(), want.isnan()) and torch.equal(have.nan_to_num(), want.nan_to_num())


def test_append_strided_caches_and_outputs(fp8lin, gpu):
    """Caches [pages, kv_heads, page_size, dim] in memory, keys and values in one tensor, queries turned in place."""
    s = Step(fp8lin, gpu, [(7, 40), (64, 1)], 4, 2, 64, 32, "blocks", block=16, rotary=32, seed=12)
    both = torch.stack([c.view(torch.uint8) for c in s.caches], 1).permute(0, 1, 3, 2, 4).contiguous().to(gpu)
    caches = [both[:, i].transpose(1, 2).view(torch.float8_e4m3fn) for i in range(2)]
    scales = [s.scale(x) for x in s.scales]
    q = s.up[0].clone()
    norms = [w.to(gpu) for w in s.norms]
    got = fp8lin.paged_rotate_append(q, s.up[1], s.up[2], s.positions.to(gpu), torch.tensor(s.slots, device=gpu), *caches, s.plan, q_norm=norms[0],
                                     k_norm=norms[1], k_scale=scales[0], v_scale=scales[1], out=q)
    assert got.data_ptr() == q.data_ptr()
    s.check((q, [c.contiguous() for c in caches], scales))
    none = torch.empty(len(s.slots), 0, 64, dtype=torch.bfloat16, device=gpu)
    fresh, sc = [c.to(gpu) for c in s.caches], [s.scale(x) for x in s.scales]
    assert fp8lin.paged_rotate_append(none, s.up[1], s.up[2], s.positions.to(gpu), torch.tensor(s.slots, device=gpu), *fresh, s.plan,
                                      k_norm=norms[1], k_scale=sc[0], v_scale=sc[1]).shape == none.shape
    assert torch.equal(fresh[0].view(torch.uint8), caches[0].contiguous().view(torch.uint8))


def test_append_cache_past_32_bits(fp8lin, gpu):
    """Slots whose elements lie beyond 2^31, in the last page of a large cache."""
    pages, page, hk, d = 2200, 1024, 8, 128
    cache = torch.zeros(pages, page, hk, d, dtype=torch.uint8, device=gpu)
    scale = [torch.full((pages, page // 64, hk), 90, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu) for _ in range(2)]
    x = torch.randn(3, hk, d, device=gpu).to(torch.bfloat16)
    slots = [pages * page - 1, pages * page - 64, 5]
    small = torch.zeros(pages, page, hk, d, dtype=torch.uint8, device=gpu)
    two = x[[0, 2]].contiguous()
    fp8lin.paged_append(two, two, torch.tensor([slots[0], slots[2]], device=gpu), cache, small, k_scale=scale[0], v_scale=scale[1])
    for i, s in ((0, slots[0]), (2, slots[2])):
        power = scale[0].view(torch.uint8)[s // page, s % page // 64].float() - 127
        want = (x[i].float() * torch.exp2(-power)[:, None]).to(torch.float8_e4m3fn)
        assert torch.equal(cache[s // page, s % page], want.view(torch.uint8)) and torch.equal(small[s // page, s % page], want.view(torch.uint8))
    assert int((cache != 0).flatten(1).any(1).sum()) == 2


def test_refused_tensors(fp8lin, gpu):
    s = Step(fp8lin, gpu, [(4, 6)], 2, 2, 64, 32, "blocks", rotary=32, seed=13)
    q, k, v = s.up
    pos, slots = s.positions.to(gpu), torch.tensor(s.slots, device=gpu)
    caches, scales = [c.to(gpu) for c in s.caches], [s.scale(x) for x in s.scales]

    def call(**kw):
        d = dict(q=q, k=k, v=v, positions=pos, slots=slots, k_cache=caches[0], v_cache=caches[1], plan=s.plan, k_scale=scales[0], v_scale=scales[1])
        return fp8lin.paged_rotate_append(**{**d, **kw})

    call()
    plan = s.plan
    for kw in (dict(q=q.float()), dict(q=q[:-1]), dict(k=k[:, :1]), dict(v=v.float()), dict(v=v[..., :32]), dict(positions=pos.int()),
               dict(positions=pos[:-1]), dict(positions=pos.cpu()), dict(positions=torch.zeros(5, 6, dtype=torch.int64, device=gpu)),
               dict(positions=torch.zeros(6, 2, dtype=torch.int64, device=gpu)[:, 0]), dict(slots=slots.int()), dict(slots=slots[1:]),
               dict(plan=plan.steps), dict(plan=plan._replace(steps=plan.steps.cpu())), dict(plan=plan._replace(steps=plan.steps.int())),
               dict(plan=plan._replace(magnitude=math.nan)), dict(plan=plan._replace(steps=plan.steps.repeat(3))), dict(q_norm=q[0, 0].float()),
               dict(k_norm=k[0, 0, :32]), dict(k_norm=s.norms[0]), dict(eps=-1.0), dict(out=torch.empty(6, 2, 64, device=gpu)), dict(out=k),
               dict(k_scale=None), dict(v_scale=None), dict(k_scale=scales[0].view(torch.uint8)), dict(k_scale=scales[0][:-1]),
               dict(v_scale=scales[1][:, :, :1]), dict(k_scale=scales[0].cpu()), dict(k_cache=caches[0].to(torch.bfloat16), v_cache=caches[1].to(torch.bfloat16)),
               dict(k_cache=caches[0].to(torch.bfloat16)), dict(k_scale=scales[0], v_scale=scales[0])):
        with pytest.raises(fp8lin.Fp8linError):
            call(**kw)
    for kw in (dict(x=q.float()), dict(positions=pos.int()), dict(positions=pos[1:]), dict(plan=None), dict(out=q[..., :32]), dict(out=q.cpu()),
               dict(plan=plan._replace(steps=plan.steps.repeat(3)))):
        with pytest.raises(fp8lin.Fp8linError):
            fp8lin.rotate(**{**dict(x=q, positions=pos, plan=plan), **kw})
    wide = torch.zeros(6, 5, 64, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(fp8lin.Fp8linError):  # an output that lies one head off its input
        fp8lin.rotate(wide[:, :2], pos, plan, out=wide[:, 1:3])
    fp8lin.rotate(wide[:, :2], pos, plan, out=wide[:, 2:4])


def test_calls_without_tokens(fp8lin, gpu):
    plan, _ = plan_of(fp8lin, gpu, 32)
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=gpu)
    at = torch.empty(0, dtype=torch.int64, device=gpu)
    assert fp8lin.rotate(none, at, plan).shape == (0, 2, 64)
    assert fp8lin.rotate(torch.empty(3, 0, 64, dtype=torch.bfloat16, device=gpu), torch.zeros(3, dtype=torch.int64, device=gpu), plan).shape == (3, 0, 64)
    cache = torch.full((2, 16, 2, 64), 3, dtype=torch.uint8, device=gpu)
    scale = [torch.full((2, 1, 2), 99, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu) for _ in range(2)]
    assert fp8lin.paged_rotate_append(none, none, none, at, at, cache, cache.clone(), plan, k_scale=scale[0], v_scale=scale[1]).shape == (0, 2, 64)
    x = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=gpu)
    fp8lin.paged_append(x, x, torch.tensor([-1, 32, 1 << 50], device=gpu), cache, cache.clone(), k_scale=scale[0], v_scale=scale[1])
    assert (cache == 3).all() and (scale[0].view(torch.uint8) == 99).all()


def test_captured_and_on_another_stream(fp8lin, gpu):
    """A rotated append as a HIP graph, replayed with other inputs between the program's own work; and the same on a side stream."""
    s = Step(fp8lin, gpu, [(14, 3), (40, 1), (0, 20)], 4, 2, 64, 32, "blocks", rotary=64, seed=14)
    caches, scales = [c.to(gpu) for c in s.caches], [s.scale(x) for x in s.scales]
    wide, pos, slots = s.wide.to(gpu), s.positions.to(gpu), torch.tensor(s.slots, device=gpu)
    norms = [w.to(gpu) for w in s.norms]
    split = lambda w: [w[:, a * 64:(a + n) * 64].unflatten(1, (n, 64)) for a, n in ((0, 4), (4, 2), (6, 2))]  # noqa: E731

    def one():
        return fp8lin.paged_rotate_append(*split(wide), pos, slots, *caches, s.plan, q_norm=norms[0], k_norm=norms[1], k_scale=scales[0],
                                          v_scale=scales[1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = one()
    for i in range(5):
        s.wide = (torch.randn(wide.shape, generator=torch.Generator().manual_seed(i)) * 2.0 ** (i - 2)).to(torch.bfloat16)
        wide.copy_(s.wide)
        s.q, s.k, s.v = split(s.wide)
        for to, x in zip((*caches, *scales), (*s.caches, *s.scales)):
            to.view(torch.uint8).copy_(x.view(torch.uint8))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        s.check((q, caches, scales))
