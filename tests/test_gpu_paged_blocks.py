"""Attention over a paged cache in 8 bits with a power of two per block of
tokens and head, on the GPU, against its plain 64-bit form on the values that
the codes stand for; and the operators of a serving step over such a cache
together."""
import math
import random

import pytest
import torch

import paged_oracle as PO
import paged_values as PV
import rotary_oracle as RO
from test_gpu_paged import HEADS, HELD, Batch, compare

pytestmark = pytest.mark.gpu


class Blocks(Batch):
    """A Batch over a cache with scales of blocks, from 2^-4 to 2^4 of each other; the bytes of blocks without a token are NaN's."""

    def __init__(self, held, heads, kv_heads, dim, page, block, seed=0, low=-4, high=4, **kw):
        super().__init__(held, heads, kv_heads, dim, page, fp8=True, seed=seed, **kw)
        g = torch.Generator().manual_seed(seed + 1)
        pages = self.k.size(0)
        self.block = block
        used = torch.zeros(pages, page // block, dtype=torch.bool)
        for b, n in enumerate(self.lengths):
            for j in range(-(-n // page)):
                used[self.table[b, j], :-(-min(page, n - j * page) // block)] = True
        # codes of about +-16
        self.k_scale, self.v_scale = [torch.where(used[..., None], torch.randint(low, high + 1, (pages, page // block, kv_heads), generator=g) + 123, 255)
                                      .to(torch.uint8) for _ in range(2)]
        self.k, self.v = [(c.float() / 4).to(torch.float8_e4m3fn) for c in (self.k, self.v)]

    def up(self, dev):
        got = super().up(dev)
        got["k_scale"], got["v_scale"] = [s.to(dev).view(torch.float8_e8m0fnu) for s in (self.k_scale, self.v_scale)]
        return got

    def values(self):
        """The caches in 64 bits; NaN where no token is."""
        return [c.double() * torch.exp2(torch.where(s == 255, math.nan, s.double()) - 127).repeat_interleave(self.block, 1)[..., None]
                for c, s in ((self.k, self.k_scale), (self.v, self.v_scale))]

    def expect(self, **kw):
        """As PO.attention.  A row's maximum may stand 12 powers of two above its largest score, so that weights below 2^-126 of it,
        2^-114 of the largest weight, are lost: of each key at most that part of its value."""
        out, bound = PO.attention(self.q, *self.values(), self.table, self.offsets, self.lengths, gate=self.gate, **kw)
        top = max([float(v[torch.isfinite(v)].abs().max()) for v in self.values()[1:] if bool(torch.isfinite(v).any())], default=0.0)
        return out, torch.where(bound > 0, bound + 2.0 ** -114 * max(self.lengths) * top, bound)


def sizes(rng):
    page = rng.choice([16, 32, 64, 128, 256])
    return page, rng.choice([b for b in (16, 32, 64, 128) if b <= page])


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("held", HELD)
def test_attention(fp8lin, gpu, held, heads):
    rng = random.Random(f"{held}{heads}")
    for _ in range(2):
        page, block = sizes(rng)
        b = Blocks(HELD[held], *heads, page, block, gate=rng.random() < 0.5, seed=rng.randrange(1 << 20), order=rng.choice(["page", "head"]))
        compare(fp8lin.paged_attention(max_count=b.max_count, **b.up(gpu)), b.expect(), f"{held} {page} {block}")


@pytest.mark.parametrize("held", [[(5000, 1), (1, 1)], [(4500, 3)], [(4300, 150)]], ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_long(fp8lin, gpu, dim, held):
    """Keys beyond the scales that one load of a wave brings, with blocks of every size."""
    for page, block in ((16, 16), (256, 128), (64, 32)):
        b = Blocks(held, 2, 1, dim, page, block, seed=page, gate=True)
        compare(fp8lin.paged_attention(max_count=b.max_count, **b.up(gpu)), b.expect(), f"{page} {block}")


@pytest.mark.parametrize("heads", [(12, 2, 256), (4, 4, 64), (6, 1, 128)], ids=str)
def test_attention_of_all_keys(fp8lin, gpu, heads):
    b = Blocks([(70, 20), (5, 5), (200, 1), (0, 2)], *heads, 32, 16, gate=True, seed=3)
    compare(fp8lin.paged_attention(max_count=20, causal=False, scale=0.05, **b.up(gpu)), b.expect(causal=False, scale=0.05))


@pytest.mark.parametrize("count", [1, 5, 1000])
def test_attention_expects_any_count(fp8lin, gpu, count):
    b = Blocks([(150, 40), (33, 1), (90, 9)], 12, 2, 256, 16, 16, gate=True, seed=4)
    compare(fp8lin.paged_attention(max_count=count, **b.up(gpu)), b.expect())


@pytest.mark.parametrize("count", [2, 70])
def test_attention_of_far_scales(fp8lin, gpu, count):
    """Scales from 2^-100 to 2^100 of values, and keys whose scores they lift or lower: one block rules a head."""
    b = Blocks([(150, count), (300, 1)], 4, 2, 128, 64, 16, seed=5, low=0, high=0)
    g = torch.Generator().manual_seed(6)
    b.v_scale = torch.where(b.v_scale == 255, b.v_scale, (127 + torch.randint(-100, 101, b.v_scale.shape, generator=g)).to(torch.uint8))
    b.k_scale = torch.where(b.k_scale == 255, b.k_scale, (123 + torch.randint(-60, 3, b.k_scale.shape, generator=g)).to(torch.uint8))
    compare(fp8lin.paged_attention(max_count=count, **b.up(gpu)), b.expect())


@pytest.mark.parametrize("count", [2, 70])
def test_attention_bad_pages_read_as_zeros(fp8lin, gpu, count):
    b = Blocks([(100, count), (40, 1)], 4, 2, 64, 16, 16, seed=6)
    pages = b.k.size(0)
    b.table[0, 1], b.table[0, 3], b.table[1, 0] = -1, pages, 1 << 30
    compare(fp8lin.paged_attention(max_count=count, **b.up(gpu)), b.expect())


@pytest.mark.parametrize("heads", [(12, 2, 256), (8, 8, 64), (16, 1, 128)], ids=str)
@pytest.mark.parametrize("held", [[(40, 4), (9, 9)], [(70, 70)], [(300, 100), (33, 3), (1, 1)]], ids=str)
def test_attention_hides_what_a_row_may_not_see(fp8lin, gpu, held, heads):
    """NaN codes in keys and values of later tokens reach the rows that see them alone (which are summed a key at a time)."""
    b = Blocks(held, *heads, 32, 16, gate=True, seed=7)
    last = b.lengths[0] - 1
    at = b.table[0, last // 32], last % 32
    b.v[at][:, 5] = math.nan
    b.k[at][0, 3] = math.nan
    k, v = b.values()
    want = PV.attention(b.q, k, v, b.table, b.offsets, b.lengths, gate=b.gate)
    assert PV.compare(fp8lin.paged_attention(max_count=b.max_count, **b.up(gpu)), want) > 0


def test_attention_equals_that_of_the_values(fp8lin, gpu):
    """Scales of blocks that are all one power of two: the same as scales of heads, of few rows bit for bit (the product with the
    scale is exact); for many rows the kernel keeps another distance to a row's maximum."""
    for count in (1, 3, 90):
        b = Blocks([(400, count), (33, 1)], 12, 2, 256, 64, 32, seed=8, gate=True, low=0, high=0)
        up = b.up(gpu)
        got = fp8lin.paged_attention(max_count=count, **up)
        one = torch.full((2,), 2.0 ** -4, device=gpu)
        again = fp8lin.paged_attention(max_count=count, **{**up, "k_scale": one, "v_scale": one})
        compare(got, b.expect())
        compare(again, b.expect())
        assert count > 3 or torch.equal(got, again)


def test_attention_cache_past_32_bits(fp8lin, gpu):
    """Codes beyond 2^32 bytes, in the last pages of a large cache, with scales beyond 2^16 of them."""
    pages, page, hk, d = 5200, 1024, 8, 128
    k, v = [torch.zeros(pages, page, hk, d, dtype=torch.uint8, device=gpu) for _ in range(2)]
    scale = [torch.full((pages, page // 16, hk), 255, dtype=torch.uint8, device=gpu) for _ in range(2)]
    g = torch.Generator(device=gpu).manual_seed(9)
    ids = [pages - 1, 0, pages - 2]
    for x, s in zip((k, v), scale):
        for i in ids:
            x[i] = torch.randn(page, hk, d, device=gpu, generator=g).to(torch.float8_e4m3fn).view(torch.uint8)
            s[i] = torch.randint(125, 129, (page // 16, hk), device=gpu, generator=g).to(torch.uint8)
    n, count = 2 * page + 77, 2
    q = torch.randn(count, 16, d, device=gpu, generator=g).to(torch.bfloat16)
    ints = dict(dtype=torch.int32, device=gpu)
    got = fp8lin.paged_attention(q, k, v, torch.tensor([ids], **ints), torch.tensor([0, count], **ints), torch.tensor([n], **ints), max_count=count,
                                 k_scale=scale[0].view(torch.float8_e8m0fnu), v_scale=scale[1].view(torch.float8_e8m0fnu))
    values = [x[ids].view(torch.float8_e4m3fn).double().cpu() * torch.exp2(s[ids].double().cpu() - 127).repeat_interleave(16, 1)[..., None]
              for x, s in zip((k, v), scale)]
    compare(got, PO.attention(q.cpu(), *values, torch.tensor([[0, 1, 2]]), [0, count], [n]))


@pytest.mark.parametrize("held", ["all", "last"])
def test_attention_of_the_most_requests(fp8lin, gpu, held):
    n = 4096
    lengths = [(1 + i % 20, 1) for i in range(n)] if held == "all" else [(0, 0)] * (n - 1) + [(500, 3)]
    b = Blocks(lengths, 4, 2, 64, 16, 16, seed=10, spare=1)
    compare(fp8lin.paged_attention(max_count=b.max_count, **b.up(gpu)), b.expect())


def test_attention_captured_and_at_once(fp8lin, gpu):
    """Repeated, replayed from a graph between other work, and on two streams at once: the same bits."""
    b = Blocks([(700, 2), (90, 1), (33, 2)], 12, 2, 256, 32, 32, gate=True, seed=11)
    c = Blocks([(300, 120)], 4, 2, 128, 64, 16, seed=12)
    ups = [b.up(gpu), c.up(gpu)]
    want = [fp8lin.paged_attention(max_count=x.max_count, **u) for x, u in zip((b, c), ups)]
    compare(want[0], b.expect())
    compare(want[1], c.expect())
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, x, u in zip(streams, (b, c), ups):
            with torch.cuda.stream(s):
                got.append(fp8lin.paged_attention(max_count=x.max_count, **u))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2])
    graphs = []
    for x, u in zip((b, c), ups):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0][0].pool() if graphs else None):
            y = fp8lin.paged_attention(max_count=x.max_count, **u)
        graphs.append((graph, y))
    # graphs of one memory pool run one after the other: each result is read before the next
    for _ in range(3):
        for i, (graph, y) in enumerate(graphs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want[i])
            fp8lin.paged_attention(max_count=b.max_count, **ups[0])


def test_refused_tensors(fp8lin, gpu):
    b = Blocks([(40, 2)], 4, 2, 64, 32, 16, seed=13)
    up = b.up(gpu)
    fp8lin.paged_attention(max_count=2, **up)
    k, v = up["k_scale"], up["v_scale"]
    thirds = torch.zeros(k.size(0), 3, 2, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu)
    eights = torch.zeros(k.size(0), 4, 2, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu)
    for ks, vs in ((k, None), (None, v), (k, v[:, :1]), (k[:, :1], v[:, :1]), (k[:-1], v[:-1]), (k.view(torch.uint8), v.view(torch.uint8)), (k.cpu(), v),
                   (thirds, thirds), (eights, eights), (k.transpose(0, 1).contiguous().transpose(0, 1), v), (k, torch.ones(2, device=gpu)),
                   (k.flatten(1), v.flatten(1)), (k[:, :0], v[:, :0])):
        with pytest.raises(fp8lin.Fp8linError):
            fp8lin.paged_attention(max_count=2, **{**up, "k_scale": ks, "v_scale": vs})
    for cache in (up["k_cache"].to(torch.bfloat16),):
        with pytest.raises(fp8lin.Fp8linError):
            fp8lin.paged_attention(max_count=2, **{**up, "k_cache": cache, "v_cache": cache})
    none = {**up, "q": up["q"][:0], "offsets": torch.zeros(2, dtype=torch.int32, device=gpu)}
    assert fp8lin.paged_attention(max_count=2, **none).shape == (0, 4, 64)


# ---- the operators together -----------------------------------------------------


@pytest.mark.parametrize("dim,rotary,neighbours", [(256, 64, False), (128, 128, True), (64, 20, False)])
def test_serving_steps(fp8lin, gpu, dim, rotary, neighbours):
    """Prompts in chunks, then drafts of which some are rejected, over a cache with scales of blocks: after each step the caches
    and the attention's output against 64 bits of what went in."""
    heads, hk, page, block, n = 4, 2, 32, 16, 3
    g = torch.Generator().manual_seed(dim)
    ints = dict(dtype=torch.int32, device=gpu)
    plan = fp8lin.rotary_plan(rotary, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}, neighbours=neighbours,
                              device=gpu)
    freq, mag = RO.frequencies(rotary, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64})
    norms = [(0.3 * torch.randn(dim, generator=g)).to(torch.bfloat16) for _ in range(2)]
    pages = 40
    caches = [torch.full((pages, page, hk, dim), 0x7f, dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.full((pages, page // block, hk), 255, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu) for _ in range(2)]
    table, lengths = torch.full((n, 12), -1, **ints), torch.zeros(n, **ints)
    free, cursor = torch.randperm(pages, generator=g).to(**ints), torch.zeros(1, **ints)
    kept = [[] for _ in range(n)]  # (key, its bound, value) of each token in 64 bits
    # new tokens of each request, and how many of them stay
    steps = [([70, 5, 33], [70, 5, 33]), ([40, 1, 1], [40, 1, 1]), ([1, 4, 3], [1, 2, 1]), ([3, 3, 0], [1, 3, 0]), ([1, 1, 40], [1, 1, 40]), ([2, 2, 2], [2, 1, 1])]
    for step, (counts, stay) in enumerate(steps):
        total, extra = sum(counts), 2
        x = torch.randn(total + extra, (heads + 2 * hk) * dim, generator=g) * 2.0 ** ((step % 3) - 1)
        x = x.to(torch.bfloat16)
        q, k, v = [x[:, a * dim:(a + m) * dim].unflatten(1, (m, dim)) for a, m in ((0, heads), (heads, hk), (heads + hk, hk))]
        lay = fp8lin.paged_layout(lengths, torch.tensor(counts, **ints), table, free, total + extra, page, cursor=cursor, out=table)
        cursor.copy_(lay.cursor)
        up = x.to(gpu)
        uq, uk, uv = [up[:, a * dim:(a + m) * dim].unflatten(1, (m, dim)) for a, m in ((0, heads), (heads, hk), (heads + hk, hk))]
        turned = fp8lin.paged_rotate_append(uq, uk, uv, lay.positions, lay.slots, *caches, plan, q_norm=norms[0].to(gpu), k_norm=norms[1].to(gpu),
                                            k_scale=scales[0], v_scale=scales[1])
        got = fp8lin.paged_attention(turned, *caches, lay.block_table, lay.offsets, lay.lengths, max_count=max(counts), k_scale=scales[0],
                                     v_scale=scales[1])
        pos = lay.positions.cpu()
        yk, reach = RO.rotate(RO.norm(k, norms[1], 1e-6), pos, freq, mag, neighbours)
        bound = RO.row_bound(yk, reach, True)
        yq, qreach = RO.rotate(RO.norm(q, norms[0], 1e-6), pos, freq, mag, neighbours)
        off = RO.row_bound(yq, qreach, True)
        assert float(((turned.double().cpu() - yq).abs() - off - RO.BF16_HALF * (yq.abs() + off) * 1.01).max()) <= 0
        # the attention of what is in the caches
        values = [c.double().cpu() * torch.exp2(s.view(torch.uint8).double().cpu() - 127).repeat_interleave(block, 1)[..., None]
                  for c, s in zip(caches, scales)]
        compare(got, PO.attention(turned.cpu(), *values, lay.block_table.cpu(), lay.offsets.tolist(), lay.lengths.tolist()), f"step {step}")
        # and what is in the caches: each token's values to half a step of its block's scale (and half a step more for each growth past it)
        o = lay.offsets.tolist()
        now = [kept[b] + [(yk[i], bound[i], v[i].double()) for i in range(o[b], o[b + 1])] for b in range(n)]
        for b in range(n):
            for p, (key, err, value) in enumerate(now[b]):
                at, slot = int(lay.block_table[b, p // page]), p % page
                for i, (want, e) in enumerate(((key, err), (value, 0))):
                    unit = torch.exp2(scales[i].view(torch.uint8)[at, slot // block].double().cpu() - 127)[:, None]
                    have = values[i][at, slot]
                    assert float(((have - want).abs() - e - (want.abs() + e) * RO.E4M3_HALF - 6 * RO.E4M3_SMALL * unit).max()) <= 0, (step, b, p)
        kept = [now[b][:len(kept[b]) + s] for b, s in enumerate(stay)]
        lengths.add_(torch.tensor(stay, **ints))
    assert lengths.tolist() == [len(k) for k in kept]


@pytest.mark.parametrize("power", [20, 27, 36, 38, 200, 220])
@pytest.mark.parametrize("count", [2, 70, 200])
def test_attention_of_small_and_large_values(fp8lin, gpu, count, power):
    """Values of one size, from 2^-107 to 2^93 times their codes: the same relative precision (the bound's absolute part is far below)."""
    b = Blocks([(260, count), (90, 1)], 4, 2, 128, 32, 16, seed=14, low=0, high=0)
    b.v_scale = torch.where(b.v_scale == 255, b.v_scale, power).to(torch.uint8)
    b.k_scale = torch.where(b.k_scale == 255, b.k_scale, 124).to(torch.uint8)
    unit = 2.0 ** (power - 127)
    got = fp8lin.paged_attention(max_count=count, **b.up(gpu)).double().cpu() / unit
    # as bounded for values of size 1, where 1e-37 is nothing
    b.v_scale = torch.where(b.v_scale == 255, b.v_scale, 127).to(torch.uint8)
    want, bound = b.expect()
    rows = bound > 0
    # a product with a weight below the least normal number may be lost
    bound = bound + 260 * 2.0 ** -126 / unit
    assert float(((got - want).abs() - bound)[rows].max()) <= 0
