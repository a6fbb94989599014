"""The paged-cache operators on the GPU against their plain 64-bit forms
(paged_oracle): layouts and drawn tokens exactly, the cache's contents bit for
bit, attention within a bound that counts its roundings."""
import math
import random

import pytest
import torch

import paged_oracle as PO

pytestmark = pytest.mark.gpu


class Batch:
    """Requests of given (length, new tokens) over a shuffled cache whose unused slots and pages hold NaN."""

    def __init__(self, held, heads, kv_heads, dim, page, fp8=False, gate=False, seed=0, spare=3, extra_rows=0, order="page"):
        g = torch.Generator().manual_seed(seed)
        self.lengths = [n for n, _ in held]
        counts = [c for _, c in held]
        self.offsets = [sum(counts[:i]) for i in range(len(counts) + 1)]
        self.tokens, self.max_count = self.offsets[-1] + extra_rows, max(counts)
        width = max(1, max(-(-n // page) for n in self.lengths)) + 1
        need = [-(-n // page) for n in self.lengths]
        pages = sum(need) + spare
        ids = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((len(held), width), -1, dtype=torch.int32)
        shape = (pages, page, kv_heads, dim)
        kv = [torch.full(shape, math.nan) for _ in range(2)]
        for b, n in enumerate(self.lengths):
            for j in range(need[b]):
                at = ids.pop()
                self.table[b, j] = at
                there = min(page, n - j * page)
                for x in kv:
                    x[at, :there] = torch.randn(there, kv_heads, dim, generator=g)
        if fp8:
            self.k_scale, self.v_scale = [0.01 * (1 + torch.randint(0, 4, (kv_heads,), generator=g).float()) for _ in range(2)]
            self.k, self.v = [(x / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn) for x, s in zip(kv, (self.k_scale, self.v_scale))]
        else:
            self.k_scale = self.v_scale = None
            self.k, self.v = [x.to(torch.bfloat16) for x in kv]
        self.order = order
        self.q = (2 * torch.randn(self.tokens, heads, dim, generator=g)).to(torch.bfloat16)
        self.gate = torch.randn(self.tokens, heads, dim, generator=g).to(torch.bfloat16) if gate else None

    def up(self, dev):
        def cache(x):
            if self.order == "head":  # [pages, kv_heads, page_size, dim] in memory
                return x.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
            return x.to(dev)
        ints = dict(dtype=torch.int32, device=dev)
        return dict(q=self.q.to(dev), k_cache=cache(self.k), v_cache=cache(self.v), block_table=self.table.to(dev),
                    offsets=torch.tensor(self.offsets, **ints), lengths=torch.tensor(self.lengths, **ints),
                    gate=None if self.gate is None else self.gate.to(dev),
                    k_scale=None if self.k_scale is None else self.k_scale.to(dev),
                    v_scale=None if self.v_scale is None else self.v_scale.to(dev))

    def expect(self, **kw):
        return PO.attention(self.q, self.k, self.v, self.table, self.offsets, self.lengths, gate=self.gate,
                            k_scale=self.k_scale, v_scale=self.v_scale, **kw)


def compare(got, want, what=""):
    out, bound = want
    rows = ~torch.isnan(bound) & (bound > 0)
    g = got.double().cpu()
    nan = torch.isnan(out) & rows
    assert torch.equal(torch.isnan(g) & rows, nan), f"{what}: NaN in other places"
    inf = torch.isinf(out) & rows
    assert torch.equal(g[inf], out[inf]), f"{what}: other infinities"
    err = ((g - out).abs() - bound)[rows & ~nan & ~inf]
    assert not err.numel() or float(err.max()) <= 0, f"{what}: {float(err.max())} beyond the bound"


HEADS = [(12, 2, 256), (8, 8, 64), (7, 1, 128), (16, 1, 128), (6, 2, 64), (2, 2, 256)]
HELD = {
    "one": [(1, 1)],
    "tile": [(16, 1), (32, 1), (64, 1)],
    "around": [(15, 1), (17, 1), (31, 1), (33, 1), (63, 1), (65, 1), (129, 1)],
    "ragged": [(700, 1), (3, 1), (1, 1), (250, 1), (1025, 1)],
    "drafts": [(300, 4), (5, 5), (77, 2), (1, 1), (513, 8)],
    "empty": [(0, 0), (40, 0), (0, 1), (2, 5), (90, 3), (0, 0)],
    "chunk": [(333, 70)],
    "prompt": [(200, 200), (129, 129), (1, 1)],
    "mixed": [(400, 1), (450, 90), (64, 64), (3, 0), (100, 2)],
}


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("held", HELD)
def test_attention(fp8lin, gpu, held, heads, fp8):
    rng = random.Random(f"{held}{heads}{fp8}")
    b = Batch(HELD[held], *heads, page=rng.choice([16, 32, 64, 256]), fp8=fp8, gate=rng.random() < 0.5,
              seed=rng.randrange(1 << 20), order=rng.choice(["page", "head"]))
    got = fp8lin.paged_attention(max_count=b.max_count, **b.up(gpu))
    compare(got, b.expect(), held)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(12, 2, 256), (4, 4, 64), (6, 1, 128)], ids=str)
def test_attention_of_all_keys(fp8lin, gpu, heads, fp8):
    """causal=False: every row sees all keys of its request; and another softmax scale."""
    b = Batch([(70, 20), (5, 5), (200, 1), (0, 2)], *heads, page=16, fp8=fp8, gate=True, seed=3)
    got = fp8lin.paged_attention(max_count=20, causal=False, scale=0.05, **b.up(gpu))
    compare(got, b.expect(causal=False, scale=0.05))


@pytest.mark.parametrize("count", [1, 5, 1000])
def test_attention_expects_any_count(fp8lin, gpu, count):
    """max_count picks the kernel; requests with more rows than it come out right as well."""
    b = Batch([(150, 40), (33, 1), (90, 9)], 12, 2, 256, page=16, gate=True, seed=4)
    compare(fp8lin.paged_attention(max_count=count, **b.up(gpu)), b.expect())


@pytest.mark.parametrize("count", [3, 50])
def test_attention_strided_operands(fp8lin, gpu, count):
    """Queries, gate and output as views that start off 16 (8) bytes; rows behind the last request stay."""
    b = Batch([(60, count), (130, 1)], 6, 2, 128, page=16, gate=True, seed=5, extra_rows=4)
    up = b.up(gpu)
    t = b.tokens
    for pad in (1, 4, 8):
        wide = torch.zeros(t, 6, 256 + 2 * pad, dtype=torch.bfloat16, device=gpu)
        q, gate = wide[..., pad:pad + 128], wide[..., pad + 128:pad + 256]
        q.copy_(up["q"])
        gate.copy_(up["gate"])
        out = torch.full((t, 7, 128 + pad), 7.0, dtype=torch.bfloat16, device=gpu)
        view = out[:, 1:, pad:]
        got = fp8lin.paged_attention(max_count=count, out=view, **{**up, "q": q, "gate": gate})
        assert got.data_ptr() == view.data_ptr()
        compare(got, b.expect())
        keep = out.clone()
        keep[:t - 4, 1:, pad:] = 7.0
        assert (keep == 7.0).all(), "wrote outside the rows of the requests"


@pytest.mark.parametrize("count", [2, 70])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_bad_pages_read_as_zeros(fp8lin, gpu, fp8, count):
    b = Batch([(200, count), (100, 1), (150, 2)], 6, 2, 128, page=32, fp8=fp8, seed=6)
    b.table[0, 1], b.table[0, 4], b.table[2, 0], b.table[1, 2] = -1, b.k.size(0), 1 << 30, -(1 << 31)
    compare(fp8lin.paged_attention(max_count=count, **b.up(gpu)), b.expect())


def test_attention_lengths_beyond_the_table(fp8lin, gpu):
    """Lengths are cut to the table's width, offsets to the rows that are there; negative ones count as none."""
    b = Batch([(64, 1), (48, 2)], 4, 2, 64, page=16, seed=7)
    up = b.up(gpu)
    up["block_table"] = up["block_table"][:, :3].contiguous()  # 48 tokens
    got = fp8lin.paged_attention(max_count=2, **up)
    b.lengths = [48, 48]
    compare(got, b.expect())
    up["lengths"] = torch.tensor([-5, 48], dtype=torch.int32, device=gpu)
    up["offsets"] = torch.tensor([-3, 1, 1000], dtype=torch.int32, device=gpu)
    b.lengths = [0, 48]
    compare(fp8lin.paged_attention(max_count=2, **up), b.expect())


@pytest.mark.parametrize("count", [1, 4, 90])
@pytest.mark.parametrize("heads", [(12, 2, 256), (4, 4, 64)], ids=str)
def test_attention_extreme_scores(fp8lin, gpu, heads, count):
    """Scores of some thousands either way, rising and falling along the keys: the running maximum moves by any amount."""
    b = Batch([(500, count), (333, 1)], *heads, page=16, seed=8)
    for at in range(b.k.size(0)):
        b.k[at] = (b.k[at].float() * (1 + 40 * (at % 5))).to(torch.bfloat16)
    compare(fp8lin.paged_attention(max_count=count, **b.up(gpu)), b.expect())
    b.q = -b.q
    compare(fp8lin.paged_attention(max_count=count, **b.up(gpu)), b.expect())


@pytest.mark.parametrize("dim,fp8", [(256, False), (128, True)])
def test_attention_cache_past_32_bits(fp8lin, gpu, dim, fp8):
    """Pages whose offset passes 2^31 elements (and 2^32 bytes)."""
    page, hk = 256, 8
    pages = (1 << 32) // (page * hk * dim) + 40
    held, top = [(600, 1), (300, 80)], pages - 1
    b = Batch(held, hk, hk, dim, page, fp8=fp8, seed=9)
    up = b.up(gpu)
    big = [torch.empty(pages, page, hk, dim, dtype=x.dtype, device=gpu) for x in (b.k, b.v)]
    n = b.k.size(0)
    for x, name in zip(big, ("k_cache", "v_cache")):
        x.view(torch.uint8)[pages - n:] = up[name].view(torch.uint8)
    table = torch.where(up["block_table"] >= 0, up["block_table"] + (pages - n), up["block_table"])
    assert int(table.max()) <= top
    got = fp8lin.paged_attention(max_count=80, **{**up, "k_cache": big[0], "v_cache": big[1], "block_table": table})
    compare(got, b.expect())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(12, 2, 256), (8, 8, 64), (16, 1, 128)], ids=str)
@pytest.mark.parametrize("held", [[(40, 4), (9, 9)], [(70, 70)], [(300, 100), (33, 3), (1, 1)]], ids=str)
def test_attention_hides_what_a_row_may_not_see(fp8lin, gpu, held, heads, fp8):
    """Infinities and NaN in keys and values of later tokens of a chunk: the rows before them are as if they were not there, the
    rows that see them get them."""
    b = Batch(held, *heads, page=16, fp8=fp8, gate=True, seed=13)
    g = torch.Generator().manual_seed(14)
    nan, inf = math.nan, math.inf
    for r, (n, c) in enumerate(held):
        if c < 3:
            continue
        for at, cache, values in ((n - 1, b.v, [nan, 3.0]), (n - c // 2, b.v, [inf, -inf]), (n - 1 - c // 4, b.k, [nan, 1.0])):
            if cache.dtype != torch.bfloat16:
                values = [nan, nan]  # E4M3FN has no infinities
            row = cache[int(b.table[r, at // 16]), at % 16]
            where = torch.randint(0, row.size(1), (row.size(0), 2), generator=g)
            for h in range(row.size(0)):
                for d, x in zip(where[h].tolist(), values):
                    row[h, d] = x
    got = fp8lin.paged_attention(max_count=b.max_count, **b.up(gpu))
    compare(got, b.expect())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(12, 2, 256), (8, 8, 64), (16, 1, 128)], ids=str)
@pytest.mark.parametrize("held", [(61, 61), (301, 193), (20, 33)], ids=str)
def test_attention_hides_each_later_token(fp8lin, gpu, held, heads, fp8):
    """A NaN in the values of one token of a chunk: the rows that see it have it, all others, of its tiles and of others, what
    they have without it."""
    n, c = held
    b = Batch([held], *heads, page=16, fp8=fp8, gate=True, seed=15)
    up = b.up(gpu)
    out, bound = b.expect()
    for at in range(max(n - c, 0), n, 3):
        v, dim = up["v_cache"].clone(), at % heads[2]
        v[int(b.table[0, at // 16]), at % 16, :, dim] = math.nan
        want = out.clone()
        want[at - (n - c):, :, dim] = math.nan
        compare(fp8lin.paged_attention(max_count=c, **{**up, "v_cache": v}), (want, bound), f"token {at}")


@pytest.mark.parametrize("count", [1, 400])
@pytest.mark.parametrize("held", ["all", "last"])
def test_attention_of_the_most_requests(fp8lin, gpu, held, count):
    """4096 requests, most of a few keys, or none but the last of any length; both kernels."""
    rng = random.Random(held)
    n = 4096
    sizes = [(0, rng.choice([0, 1]))] * (n - 1) + [(3000, 2)]
    if held == "all":
        sizes = [(rng.choice([0, 1, 15, 16, 17, 40]), rng.choice([0, 1, 1, 2, 9])) for _ in range(n - 1)] + [(2000, 3)]
    b = Batch(sizes, 2, 1, 64, page=16, seed=21)
    compare(fp8lin.paged_attention(max_count=count, **b.up(gpu)), b.expect(), held)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(128, 1, 64), (96, 1, 256), (65, 1, 128), (40, 40, 64), (64, 16, 128)], ids=str)
def test_attention_many_heads(fp8lin, gpu, heads, fp8):
    """More rows of one token than the few-rows kernel takes, many kv heads."""
    b = Batch([(130, 1), (77, 3), (1, 1)], *heads, page=64, fp8=fp8, gate=True, seed=22)
    want = b.expect()
    for count in (1, 3, 300):
        compare(fp8lin.paged_attention(max_count=count, **b.up(gpu)), want, str(count))


def test_attention_one_page(fp8lin, gpu):
    """The largest page: a request's keys in a row."""
    g = torch.Generator().manual_seed(23)
    k, v = [torch.randn(1, 1 << 20, 1, 64, generator=g).to(torch.bfloat16) for _ in range(2)]
    q = torch.randn(4, 2, 64, generator=g).to(torch.bfloat16)
    table, offsets, lengths = torch.zeros(2, 1, dtype=torch.int32), [0, 1, 4], [70001, 333]
    want = PO.attention(q, k, v, table, offsets, lengths)
    ints = dict(dtype=torch.int32, device=gpu)
    for count in (1, 500):
        got = fp8lin.paged_attention(q.to(gpu), k.to(gpu), v.to(gpu), table.to(gpu), torch.tensor(offsets, **ints),
                                     torch.tensor(lengths, **ints), max_count=count)
        compare(got, want, str(count))


def test_attention_is_repeatable_and_capturable(fp8lin, gpu):
    """Bit-equal calls; a captured call replayed with other lengths, queries and cache contents equals the eager one."""
    b = Batch([(300, 2), (50, 1), (90, 3)], 12, 2, 256, page=16, gate=True, seed=10)
    for count in (3, 200):
        up = b.up(gpu)
        first = fp8lin.paged_attention(max_count=count, **up)
        assert torch.equal(first, fp8lin.paged_attention(max_count=count, **up))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fp8lin.paged_attention(max_count=count, **up)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fp8lin.paged_attention(max_count=count, **up)
        for i in range(4):
            up["lengths"].copy_(torch.tensor([300 - 60 * i, 50 - i, 90 + i], dtype=torch.int32))
            up["q"].mul_(0.9)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            # lengths past what was written read NaN slots: compare the bits
            assert torch.equal(out.view(torch.int16), fp8lin.paged_attention(max_count=count, **up).view(torch.int16)), i


def test_attention_on_two_streams(fp8lin, gpu):
    a, b = Batch([(900, 1)] * 5, 12, 2, 256, page=16, seed=11), Batch([(400, 60)], 12, 2, 256, page=16, seed=12)
    ua, ub = a.up(gpu), b.up(gpu)
    wa, wb = fp8lin.paged_attention(max_count=1, **ua), fp8lin.paged_attention(max_count=60, **ub)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(s):
            ga = fp8lin.paged_attention(max_count=1, **ua)
        with torch.cuda.stream(t):
            gb = fp8lin.paged_attention(max_count=60, **ub)
        torch.cuda.synchronize()
        assert torch.equal(ga, wa) and torch.equal(gb, wb)


# ---- append -------------------------------------------------------------------


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tokens,hk,dim,page,pad", [(1, 2, 256, 16, 0), (27, 2, 256, 16, 8), (300, 8, 128, 64, 1), (65, 3, 48, 32, 3),
                                                    (1000, 1, 64, 256, 0)])
def test_append(fp8lin, gpu, tokens, hk, dim, page, pad, fp8):
    g = torch.Generator().manual_seed(tokens)
    pages = tokens // page + 3
    x = (3 * torch.randn(2, tokens, hk, dim + pad, generator=g)).to(torch.bfloat16)
    x[0, 0, 0, pad], x[1, 0, 0, pad], x[0, -1, -1, -1], x[1, -1, -1, -1] = math.nan, math.inf, -math.inf, 3e38
    if tokens > 2:
        x[0, 1, 0, pad:pad + 6] = torch.tensor([0.0, -0.0, 1e-40, -1e-3, 1e-2, 5e-3], dtype=torch.bfloat16)
    k, v = x[0, ..., pad:], x[1, ..., pad:]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[tokens // 2] = -1
    if tokens > 3:
        slots[3], slots[2] = pages * page, -(1 << 40)
    dtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
    caches = [torch.randn(pages, page, hk, dim, generator=g).to(dtype) for _ in range(2)]
    scales = [0.01 + torch.rand(hk, generator=g) / 50 for _ in range(2)] if fp8 else [None, None]
    up = [c.to(gpu) for c in caches]
    ks, vs = [s.to(gpu) if s is not None else None for s in scales]
    xg = x.to(gpu)
    fp8lin.paged_append(xg[0, ..., pad:], xg[1, ..., pad:], slots.to(gpu), *up, k_scale=ks, v_scale=vs)
    for cache, got, rows, s in zip(caches, up, (k, v), scales):
        want = cache.clone().view(torch.uint8 if fp8 else torch.int16).view(pages * page, hk, dim)
        vals = rows if s is None else (rows.float() / s[:, None]).clamp(-448, 448).to(dtype)
        for t, at in enumerate(slots.tolist()):
            if 0 <= at < pages * page:
                want[at] = vals[t].contiguous().view(want.dtype)
        got = got.cpu().view(want.dtype).view(want.shape)
        same = got == want
        if fp8:  # a NaN of either sign
            same |= ((got & 0x7F) == 0x7F) & ((want & 0x7F) == 0x7F)
        assert same.all()


def test_append_strided_caches(fp8lin, gpu):
    """Caches [pages, kv_heads, page_size, dim] in memory, K and V interleaved in one buffer, codes as uint8."""
    tokens, hk, dim, page, pages = 40, 2, 64, 16, 5
    k, v = [torch.randn(tokens, hk, dim, device=gpu, dtype=torch.bfloat16) for _ in range(2)]
    slots = torch.randperm(pages * page, device=gpu)[:tokens]
    plain = [torch.zeros(pages, page, hk, dim, dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    fp8lin.paged_append(k, v, slots, *plain)
    both = torch.zeros(pages, 2, hk, page, dim, dtype=torch.bfloat16, device=gpu)
    kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    fp8lin.paged_append(k, v, slots, kc, vc)
    assert torch.equal(kc, plain[0]) and torch.equal(vc, plain[1])
    scale = torch.full((hk,), 0.01, device=gpu)
    codes = [torch.zeros(pages, page, hk, dim, dtype=torch.uint8, device=gpu) for _ in range(2)]
    fp8lin.paged_append(k, v, slots, *codes, k_scale=scale, v_scale=scale)
    floats = [c.view(torch.float8_e4m3fn).clone().zero_() for c in codes]
    fp8lin.paged_append(k, v, slots, *floats, k_scale=scale, v_scale=scale)
    assert torch.equal(codes[0], floats[0].view(torch.uint8)) and torch.equal(codes[1], floats[1].view(torch.uint8))
    fp8lin.paged_append(k[:0], v[:0], slots[:0], *plain)  # nothing to write


# ---- layout -------------------------------------------------------------------


def _random_layout(rng, requests, page, width, long=False):
    lengths = [rng.choice([0, page, rng.randrange(page * width)]) for _ in range(requests)]
    counts = [rng.choice([0, 1, 1, 4, rng.randrange(1, page * (width if long else 2))]) for _ in range(requests)]
    if requests > 3:
        lengths[1], counts[2] = -7, -2
    ids = list(range(requests * width))
    rng.shuffle(ids)
    table = [[ids.pop() if j * page < n + rng.choice([0, 0, page]) else -1 - j for j in range(width)] for n in lengths]
    free = ids[:rng.randrange(len(ids) + 1)]
    return lengths, counts, table, free


@pytest.mark.parametrize("requests", [1, 2, 3, 64, 257, 1024, 1500])
def test_layout(fp8lin, gpu, requests):
    rng = random.Random(requests)
    for round_ in range(4):
        page, width = rng.choice([16, 64, 256]), rng.choice([1, 5, 33]) if requests > 3 else rng.choice([1, 40, 700])
        lengths, counts, table, free = _random_layout(rng, requests, page, width, long=requests < 64)
        total = sum(max(c, 0) for c in counts)
        tokens = max(0, total + rng.choice([0, 0, 5, 300, -2]))
        cursor = rng.randrange(0, 4)
        want = PO.layout(lengths, counts, table, free, tokens, page, cursor)
        ints = dict(dtype=torch.int32, device=gpu)
        wide = torch.full((requests, width + 3), 99, **ints)
        args = (torch.tensor(lengths, **ints), torch.tensor(counts, **ints))
        free_t = torch.tensor(free, **ints)
        for form in ("new", "view", "in place"):
            t = torch.tensor(table, **ints).view(requests, width)
            kw = {}
            if form == "view":
                wide[:, :width] = t
                t = wide[:, :width]
            elif form == "in place":
                kw["out"] = t
            got = fp8lin.paged_layout(*args, t, free_t, tokens, page, cursor=torch.tensor([cursor], **ints), **kw)
            assert got.offsets.tolist() == want[0] and got.lengths.tolist() == want[1]
            assert got.slots.tolist() == want[2] and got.positions.tolist() == want[3]
            assert got.block_table.tolist() == want[4] and got.cursor.tolist() == [want[5]]
            if form == "in place":
                assert got.block_table.data_ptr() == t.data_ptr()
            else:
                assert t.tolist() == table, "the input table changed"


def test_layout_without_cursor_or_pages(fp8lin, gpu):
    ints = dict(dtype=torch.int32, device=gpu)
    got = fp8lin.paged_layout(torch.tensor([0, 3], **ints), torch.tensor([20, 1], **ints), torch.full((2, 4), -1, **ints),
                              torch.empty(0, **ints), 21, 16)
    assert got.slots.tolist() == [-1] * 21 and got.cursor.tolist() == [3]
    assert got.positions.tolist() == list(range(20)) + [3] and got.offsets.tolist() == [0, 20, 21]
    none = fp8lin.paged_layout(torch.tensor([5], **ints), torch.tensor([0], **ints), torch.full((1, 4), -1, **ints),
                               torch.arange(4, **ints), 0, 16)
    assert none.cursor.tolist() == [0] and none.slots.numel() == 0 and none.block_table.tolist() == [[-1] * 4]


# ---- verification -------------------------------------------------------------


def _drafted(rng, requests, drafts, vocab, probs, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    counts = [rng.choice([0, 1, drafts + 1, rng.randint(1, drafts + 1)]) if requests > 1 else drafts + 1 for _ in range(requests)]
    offsets = [sum(counts[:i]) for i in range(requests + 1)]
    rows = offsets[-1]
    logits = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    near, tokens = [], torch.randint(0, vocab, (rows,), generator=g)
    for b in range(requests):
        for i in range(counts[b] - 1):
            x = logits[offsets[b] + i].float() + 0.7 * torch.randn(vocab, generator=g)
            q = torch.softmax(x, 0)
            near.append(q)
            tokens[offsets[b] + i + 1] = int(torch.multinomial(q, 1, generator=g)) if probs else int(x.argmax())
    q = torch.stack(near) if near else torch.zeros(0, vocab)
    return logits, tokens, torch.rand(rows, generator=g), offsets, q if probs else None


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("requests,drafts,vocab", [(1, 0, 1), (1, 3, 7), (5, 2, 1000), (9, 5, 2049), (3, 4, 40001), (40, 1, 513),
                                                   (2, 7, 24000)])
def test_verify(fp8lin, gpu, requests, drafts, vocab, probs, dtype):
    rng = random.Random(f"{requests}{drafts}{vocab}{probs}{dtype}")
    for round_ in range(3):
        logits, tokens, u, offsets, q = _drafted(rng, requests, drafts, vocab, probs, dtype, rng.randrange(1 << 20))
        if logits.size(0) == 0:
            continue
        temperature = torch.tensor([rng.choice([0.0, 1.0, 0.3, 2.5]) for _ in range(requests)]) if round_ else None
        want = PO.verify(logits, tokens, u, offsets, q, temperature)
        pad = torch.zeros(logits.size(0), vocab + 5, dtype=dtype)
        pad[:, 5:] = logits
        for x in (logits.to(gpu), pad.to(gpu)[:, 5:]):
            got = fp8lin.verify_drafts(x, tokens.to(gpu), u.to(gpu), torch.tensor(offsets, dtype=torch.int32, device=gpu),
                                       draft_probs=None if q is None else q.to(gpu),
                                       temperature=None if temperature is None else temperature.to(gpu))
            assert got[0].tolist() == want[0] and got[1].tolist() == want[1]


def test_verify_masked_and_broken_rows(fp8lin, gpu):
    """-inf logits (a top-k cut), rows of NaN, +inf or nothing, equal logits, drafts outside the vocabulary, rows behind the
    last request."""
    v = 5000
    x = torch.randn(12, v)
    x[0, 100:] = -math.inf
    x[1, :] = -math.inf
    x[1, 4321] = 2.0
    x[2, 17] = math.nan
    x[3, 18] = math.inf
    x[4, :] = -math.inf
    x[5, :] = 1.5
    x[6, :] = -3e38
    tokens = torch.tensor([0, 50, 4321, 17, 1, 1, 0, 4999, 0, -1, v, 0])
    u = torch.tensor([0.0, 0.5, 0.1, 0.1, 0.1, 0.9999, 0.3, 0.999999, 0.0, 0.0, 0.999, 0.5])
    for offsets in ([0, 3, 4, 5, 6, 8, 11], [0, 1, 2, 3, 5, 7, 9], [0, 0, 0, 2, 11, 11, 12]):
        for t in (None, torch.tensor([1.0, 0.0, 0.5, 0.0, 2.0, 0.7])):
            want = PO.verify(x, tokens, u, offsets, None, t)
            got = fp8lin.verify_drafts(x.to(gpu), tokens.to(gpu), u.to(gpu), torch.tensor(offsets, dtype=torch.int32, device=gpu),
                                       temperature=None if t is None else t.to(gpu))
            assert got[0].tolist() == want[0] and got[1].tolist() == want[1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [40, 9001, 248320])
def test_verify_refuses_likely_drafts(fp8lin, gpu, vocab, dtype):
    """Drafts of nearly all probability that the largest number below 1 refuses, and certain ones that it does not: the token is
    drawn from what little is left."""
    g = torch.Generator().manual_seed(vocab)
    rows = 24
    x = torch.randn(rows, vocab, generator=g)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    for i in range(0, rows, 2):  # row i decides on the draft tokens[i + 1]
        x[i, tokens[i + 1]] = math.log(vocab) + 4 + i / 2
    x[22, :] = -math.inf
    x[22, tokens[23]] = 1.0
    x = x.to(dtype)
    u = torch.rand(rows, generator=g)
    u[::2] = 1 - 2.0 ** -24
    offsets = list(range(0, rows + 1, 2))
    want = PO.verify(x, tokens, u, offsets, None, None)
    got = fp8lin.verify_drafts(x.to(gpu), tokens.to(gpu), u.to(gpu), torch.tensor(offsets, dtype=torch.int32, device=gpu))
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    assert 0 < sum(want[0]) < 12


def test_verify_draws_the_distribution(fp8lin, gpu):
    """Over an even grid of numbers every token is drawn as often as its share of the residual weight says, to one draw."""
    v, n = 300, 4096
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, v, generator=g).expand(n, v).contiguous().to(gpu)
    u = ((torch.arange(n) + 0.5) / n).float().to(gpu)
    offsets = torch.arange(n + 1, dtype=torch.int32, device=gpu)
    drawn = fp8lin.verify_drafts(x, torch.zeros(n, dtype=torch.int64, device=gpu), u, offsets)[1]
    share = torch.bincount(drawn, minlength=v).cpu().double()
    assert float((share - torch.softmax(x[0].double().cpu(), 0) * n).abs().max()) <= 1.0 + 1e-6


def test_verify_numbers_outside_the_interval(fp8lin, gpu):
    """Numbers that are no uniforms stay inside the row: the first token with weight, or the last one."""
    x = torch.randn(6, 700)
    x[:, :3], x[:, 690:] = -math.inf, -math.inf
    u = torch.tensor([-1.0, -math.inf, 1.0, 7.0, math.inf, math.nan])
    offsets = torch.arange(7, dtype=torch.int32, device=gpu)
    out = fp8lin.verify_drafts(x.to(gpu), torch.zeros(6, dtype=torch.int64, device=gpu), u.to(gpu), offsets)[1].tolist()
    assert out[:5] == [3, 3, 689, 689, 689] and 3 <= out[5] <= 689


def test_verify_past_32_bits(fp8lin, gpu):
    """Logits of more than 2^31 values: the last rows as by themselves."""
    rows, vocab = 9000, 248320
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=gpu)
    x[-300:].normal_(0, 3)
    tokens, u = torch.randint(0, vocab, (rows,), device=gpu), torch.rand(rows, device=gpu)
    tokens[-299:] = x[-300:-1].argmax(1)
    offsets = torch.arange(0, rows + 1, 3, dtype=torch.int32, device=gpu)
    taken, out = fp8lin.verify_drafts(x, tokens, u, offsets)
    last = fp8lin.verify_drafts(x[-300:], tokens[-300:], u[-300:], (offsets[-101:] - offsets[-101]))
    assert torch.equal(taken[-100:], last[0]) and torch.equal(out[-300:], last[1]) and int(taken[-100:].sum()) > 0


# ---- refusals on the device -----------------------------------------------------


def test_refused_tensors(fp8lin, gpu):
    """Each tensor of another type, shape, place or stride than a call takes raises; nothing reaches a kernel."""
    def alike(t):
        yield t.cpu()
        yield t.double() if t.is_floating_point() else t.to(torch.int16)
        yield t[:-1] if t.dim() == 1 else t[..., :-1]
        yield t.unsqueeze(0)
        if t.dim() == 1 and t.numel() > 1:
            yield torch.stack([t, t], 1)[:, 0]
        elif t.dim() > 1:
            yield t.transpose(-1, -2).contiguous().transpose(-1, -2)

    b = Batch([(40, 3), (20, 2)], 4, 2, 64, page=16, gate=True, fp8=True)
    ints = dict(dtype=torch.int32, device=gpu)
    attention = dict(b.up(gpu), out=torch.empty(5, 4, 64, dtype=torch.bfloat16, device=gpu))
    append = dict(k=attention["q"][:, :2], v=attention["q"][:, 2:], slots=torch.full((5,), -1, dtype=torch.int64, device=gpu),
                  **{n: attention[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")})
    layout = dict(lengths=torch.tensor([40, 20], **ints), counts=torch.tensor([1, 2], **ints), block_table=attention["block_table"],
                  free_pages=torch.arange(3, **ints), cursor=torch.zeros(1, **ints), out=torch.empty_like(attention["block_table"]))
    verify = dict(logits=torch.zeros(5, 90, device=gpu), tokens=torch.zeros(5, dtype=torch.int64, device=gpu),
                  uniforms=torch.zeros(5, device=gpu), offsets=torch.tensor([0, 3, 5], **ints),
                  draft_probs=torch.zeros(3, 90, device=gpu), temperature=torch.ones(2, device=gpu))
    calls = [(fp8lin.paged_attention, attention, {}), (fp8lin.paged_append, append, {}),
             (fp8lin.paged_layout, layout, dict(tokens=5, page_size=16)), (fp8lin.verify_drafts, verify, {})]
    # of any length or width, of which a shorter one is as good
    free = {("paged_layout", "free_pages"): (2,), ("paged_attention", "block_table"): (2,)}
    for call, good, plain in calls:
        call(**good, **plain)
        for name, t in good.items():
            for i, bad in enumerate(alike(t)):
                if i in free.get((call.__name__, name), ()):
                    continue
                with pytest.raises(fp8lin.Fp8linError):
                    call(**{**good, name: bad}, **plain)
                    pytest.fail(f"{call.__name__}: {name} {i}")
    for plain in (dict(tokens=-1, page_size=16), dict(tokens=5, page_size=24), dict(tokens=5, page_size=8)):
        with pytest.raises(fp8lin.Fp8linError):
            fp8lin.paged_layout(**layout, **plain)
    for change in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(k_scale=None), dict(v_scale=None)):
        with pytest.raises(fp8lin.Fp8linError):
            fp8lin.paged_attention(**{**attention, **change})
    none = attention["k_cache"][:, :, :0]
    with pytest.raises(fp8lin.Fp8linError):
        fp8lin.paged_attention(**{**attention, "k_cache": none, "v_cache": none, "k_scale": attention["k_scale"][:0],
                                  "v_scale": attention["v_scale"][:0]})
    torch.cuda.synchronize()


def test_calls_without_tokens(fp8lin, gpu):
    b = Batch([(40, 3), (20, 2)], 4, 2, 64, page=16)
    up = b.up(gpu)
    none = up["q"][:0]
    out = fp8lin.paged_attention(**{**up, "q": none, "offsets": torch.zeros_like(up["offsets"])})
    assert out.shape == none.shape
    before = up["k_cache"].clone()
    fp8lin.paged_append(none[:, :2], none[:, :2], torch.zeros(0, dtype=torch.int64, device=gpu), up["k_cache"], up["v_cache"])
    assert torch.equal(before.view(torch.int16), up["k_cache"].view(torch.int16))
    taken, out = fp8lin.verify_drafts(torch.zeros(0, 50, device=gpu), torch.zeros(0, dtype=torch.int64, device=gpu),
                                      torch.zeros(0, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu))
    assert taken.tolist() == [0, 0] and out.numel() == 0


def test_verify_captured(fp8lin, gpu):
    rng = random.Random(7)
    logits, tokens, u, offsets, q = _drafted(rng, 6, 3, 9000, True, torch.bfloat16, 5)
    args = [logits.to(gpu), tokens.to(gpu), u.to(gpu), torch.tensor(offsets, dtype=torch.int32, device=gpu), q.to(gpu)]
    fp8lin.verify_drafts(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fp8lin.verify_drafts(*args)
    for i in range(4):
        args[2].copy_(torch.rand(u.shape, generator=torch.Generator().manual_seed(i)))
        args[0].mul_(0.9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = fp8lin.verify_drafts(*args)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_at_once_and_graphs_of_one_pool(fp8lin, gpu):
    """Layout, a mixed batch's attention and verification without probabilities: on two streams at once, and in two captured graphs
    that share a memory pool, replayed in turn with eager calls between, as by themselves."""
    rng = random.Random(31)
    sets = []
    for seed in (1, 2):
        b = Batch([(300, 90), (50, 1), (90, 30), (7, 0)], 12, 2, 256, page=16, gate=True, seed=seed)
        up = b.up(gpu)
        logits, tokens, u, offsets, _ = _drafted(rng, 6, 3, 9000, False, torch.bfloat16, seed)
        ints = dict(dtype=torch.int32, device=gpu)
        verify = [logits.to(gpu), tokens.to(gpu), u.to(gpu), torch.tensor(offsets, **ints)]
        layout = [torch.tensor([3, 40, 16, 0], **ints), torch.tensor([2, 1, 17, 5], **ints),
                  torch.where(torch.arange(8, device=gpu)[None] < torch.tensor([1, 3, 1, 0], device=gpu)[:, None], 9, -1).int(),
                  torch.randperm(20, device=gpu).int(), 25, 16]

        def call(up=up, verify=verify, layout=layout):
            return (*fp8lin.paged_layout(*layout), fp8lin.paged_attention(max_count=90, **up), *fp8lin.verify_drafts(*verify))
        sets.append((call, [x.clone() for x in call()], up, verify))

    def same(got, want):
        return all(torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x, y.view(torch.int16) if y.dtype == torch.bfloat16 else y)
                   for x, y in zip(got, want))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, (call, *_rest) in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(call())
        torch.cuda.synchronize()
        assert all(same(x, w) for x, (_, w, *_rest) in zip(got, sets))
    graphs, outs = [], []
    for call, *_rest in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(call())
        graphs.append(graph)
    for i in range(4):
        for graph, out, (call, _, up, verify) in zip(graphs, outs, sets):
            up["q"].mul_(0.9)
            verify[2].copy_(torch.rand(verify[2].shape, generator=torch.Generator().manual_seed(i)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = [x.clone() for x in out]
            assert same(got, call()), i


# ---- a run of them together -----------------------------------------------------


class _Server:
    """Two requests and one layer: prompts in chunks, then steps of drafted tokens that are verified, every length on the GPU."""

    H, HK, D, K, V, PAGE = 4, 2, 64, 256, 1000, 16
    ROPE = {"partial_rotary_factor": 0.25, "mrope_section": [3, 3, 2], "rope_theta": 10000}
    P = "model.language_model.layers.3.self_attn"

    def __init__(self, F, dev, requests, fp8):
        self.F, self.dev = F, dev
        self.eng = F.LinearEngine(F.LinearOptions())
        for i, (name, n, k) in enumerate((("q_proj", self.H * 2 * self.D, self.K), ("k_proj", self.HK * self.D, self.K),
                                          ("v_proj", self.HK * self.D, self.K), ("o_proj", self.K, self.H * self.D))):
            self.eng.add(f"{self.P}.{name}.weight", *F.gen_weights(n, k, seed=5, tag=10 + i, std=0.06, device=dev))
        self.eng.fuse_weights(self.P + ".qkv_gate", [self.P + "." + n for n in ("q_proj", "k_proj", "v_proj")])
        self.eng.add("lm_head.weight", *F.gen_weights(self.V, self.K, seed=5, tag=20, std=0.2, device=dev))
        g = torch.Generator().manual_seed(2)
        self.embed = torch.randn(self.V, self.K, generator=g).to(torch.bfloat16).to(dev)
        self.norms = [(0.1 * torch.randn(self.D, generator=g)).to(torch.bfloat16).to(dev) for _ in range(2)]
        width, pages = 12, 12 * requests
        shape = (pages, self.PAGE, self.HK, self.D)
        dtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
        self.caches = [torch.full(shape, math.nan, device=dev).to(dtype) for _ in range(2)]
        self.scales = dict(k_scale=torch.full((self.HK,), 0.01, device=dev), v_scale=torch.full((self.HK,), 0.01, device=dev)) if fp8 else {}
        ints = dict(dtype=torch.int32, device=dev)
        self.table = torch.full((requests, width), -1, **ints)
        self.free = torch.randperm(pages, generator=g).int().to(dev)
        self.lengths, self.cursor = torch.zeros(requests, **ints), torch.zeros(1, **ints)

    def step(self, tokens, counts, max_count):
        """The layer's output rows of a step, and its layout."""
        lay = self.F.paged_layout(self.lengths, counts, self.table, self.free, tokens.size(0), self.PAGE, cursor=self.cursor, out=self.table)
        y = self.eng.full_attention(self.embed[tokens], self.P, lay, *self.caches, *self.norms, self.H, self.HK, self.D, self.ROPE, 1e-6,
                                    max_count=max_count, **self.scales)
        self.cursor.copy_(lay.cursor)
        return y, lay


@pytest.mark.parametrize("fp8", [False, True])
def test_serving_steps(fp8lin, gpu, fp8):
    """Chunked prompts, then drafted steps with rejected drafts: the cache at the end holds what one prompt of the tokens that
    were kept puts there, up to the roundings of two ways through the same arithmetic."""
    s = _Server(fp8lin, gpu, 2, fp8)
    ints = dict(dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, s.V, (n,), generator=g) for n in (45, 18)]
    kept = [list(p.tolist()) for p in prompts]
    for at in range(0, 45, 20):  # chunks of 20, the shorter prompt done after the first
        parts = [p[at:at + 20] for p in prompts]
        counts = torch.tensor([len(p) for p in parts], **ints)
        _, lay = s.step(torch.cat(parts).to(gpu), counts, 20)
        s.lengths.copy_(lay.lengths)
    last = [k.pop() for k in kept]
    s.lengths.sub_(1)  # the last prompt token is fed again as each request's current one
    temperature = torch.tensor([1.0, 0.0], device=gpu)
    rejected = 0
    for i in range(12):
        drafts = [3, (2, 0, 3)[i % 3]]
        rows = [[last[b]] + torch.randint(0, s.V, (drafts[b],), generator=g).tolist() for b in range(2)]
        tokens = torch.tensor(sum(rows, []), device=gpu)
        counts = torch.tensor([len(r) for r in rows], **ints)
        y, lay = s.step(tokens, counts, 4)
        logits = s.eng.linear(y, "lm_head")
        if i % 2:  # let some drafts through: they are the likely tokens of their rows
            likely = logits.float().argmax(1)
            tokens = torch.where(torch.rand(tokens.shape, generator=g).to(gpu) < 0.7, likely.roll(1), tokens)
            first = lay.offsets[:-1].long()
            tokens[first] = torch.tensor(last, device=gpu)
            y, lay = s.step(tokens, counts, 4)  # same step again with other drafts: same pages, new contents
            logits = s.eng.linear(y, "lm_head")
        u = torch.rand(tokens.shape, generator=g).to(gpu)
        accepted, out = fp8lin.verify_drafts(logits, tokens, u, lay.offsets, temperature=temperature)
        want = PO.verify(logits.cpu(), tokens.cpu(), u.cpu(), lay.offsets.tolist(), None, temperature.cpu())
        assert accepted.tolist() == want[0] and out.tolist() == want[1]
        s.lengths.add_(1 + accepted)
        for b in range(2):
            a, n = int(lay.offsets[b]), int(accepted[b])
            kept[b] += [last[b]] + out[a:a + n].tolist()
            last[b] = int(out[a + n])
            rejected += drafts[b] - n
    assert rejected and s.lengths.tolist() == [len(k) for k in kept]
    # the same tokens in one piece, in a fresh cache
    t = _Server(fp8lin, gpu, 2, fp8)
    y, lay = t.step(torch.tensor(kept[0] + kept[1], device=gpu), torch.tensor([len(k) for k in kept], **ints), max(map(len, kept)))
    # keys and values: one projection row through GEMMs of other row counts, so a BF16 (E4M3) step apart here and there
    step_rel = torch.finfo(torch.float8_e4m3fn).eps if fp8 else torch.finfo(torch.bfloat16).eps
    for b in range(2):
        for cache, other in zip(s.caches, t.caches):
            x, z = [PO.keys_of(c.cpu(), None, tab[b].cpu(), len(kept[b]), 1) for c, tab in ((cache, s.table), (other, lay.block_table))]
            assert torch.isfinite(x).all()
            assert float((x - z).norm() / z.norm()) <= step_rel
    # nothing of a request's cache is in another's pages: the pages that were taken are distinct
    used = s.table[s.table >= 0].tolist()
    assert len(used) == len(set(used)) == int(s.cursor)


def test_serving_step_captured(fp8lin, gpu):
    """One decode step as a HIP graph: layout, projection, epilogue, append, attention, head and verification, the lengths
    advanced by the graph itself; every replay equals the eager step from the same state."""
    state = []
    for form in ("eager", "graph"):
        s = _Server(fp8lin, gpu, 3, False)
        ints = dict(dtype=torch.int32, device=gpu)
        g = torch.Generator().manual_seed(4)
        _, lay = s.step(torch.randint(0, s.V, (60,), generator=g).to(gpu), torch.tensor([33, 16, 11], **ints), 33)
        s.lengths.copy_(lay.lengths)
        tokens = torch.randint(0, s.V, (9,), generator=g).to(gpu)
        counts, u = torch.full((3,), 3, **ints), torch.empty(9, device=gpu)
        heads = torch.arange(0, 9, 3, device=gpu)

        def one():
            y, lay = s.step(tokens, counts, 3)
            logits = s.eng.linear(y, "lm_head")
            accepted, out = fp8lin.verify_drafts(logits, tokens, u, lay.offsets)
            s.lengths.add_(1 + accepted)
            tokens[heads] = out[heads + accepted]
            return logits, accepted, out

        saved = [x.clone() for x in (s.lengths, s.cursor, s.table, tokens, *s.caches)]
        if form == "graph":
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                u.fill_(0.5)
                one()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                res = one()
            for x, y in zip((s.lengths, s.cursor, s.table, tokens, *s.caches), saved):
                x.copy_(y)
        got = []
        for i in range(8):
            u.copy_(torch.rand(9, generator=torch.Generator().manual_seed(i)))
            torch.cuda.synchronize()
            if form == "graph":
                graph.replay()
            else:
                res = one()
            torch.cuda.synchronize()
            got += [x.clone().cpu() for x in (*res, s.lengths, s.cursor, s.table)]
        state.append(got)
    for x, y in zip(*state):
        assert torch.equal(x, y)
