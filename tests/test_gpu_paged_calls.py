"""Calls of the paged-cache operators on the GPU that a server makes beside the plain ones: operands that share memory, batches
with rows of no request, prompts beside drafted requests."""
import math
import random

import pytest
import torch

import paged_oracle as PO
import paged_values as PV
from test_gpu_paged import _drafted, _Server

pytestmark = pytest.mark.gpu


def test_layout_refuses_a_table_over_its_inputs(fp8lin, gpu):
    """An output table that overlaps the input table elsewhere than at its beginning, or another input, raises; side by side rows
    of one buffer are taken."""
    ints = dict(dtype=torch.int32, device=gpu)
    lengths, counts, free = torch.tensor([3, 40], **ints), torch.tensor([1, 2], **ints), torch.arange(20, **ints)
    buf = torch.full((5, 8), -1, **ints)
    wide = torch.full((2, 16), -1, **ints)
    for table, out in ((buf[1:3], buf[2:4]), (buf[1:3], buf[:2]), (buf[1:3], free[:16].view(2, 8)), (wide[:, :8], wide[:, 4:12])):
        with pytest.raises(fp8lin.Fp8linError):
            fp8lin.paged_layout(lengths, counts, table, free, 3, 16, out=out)
    got = fp8lin.paged_layout(lengths, counts, wide[:, :8], free, 3, 16, out=wide[:, 8:])
    # one page for position 3, then entry 2 for positions 40 and 41
    assert got.block_table.tolist() == [[0] + [-1] * 7, [-1, -1, 1] + [-1] * 5] and got.slots.tolist() == [3, 24, 25]
    assert (wide[:, :8] == -1).all()


def _verify(fp8lin, logits, tokens, u, offsets, q=None, temperature=None):
    """fp8lin_verify_drafts into memory that holds other numbers."""
    rows, vocab = logits.shape
    dev, requests = logits.device, len(offsets) - 1
    off = torch.tensor(offsets, dtype=torch.int32, device=dev)
    accepted, out = torch.full((requests,), 77, dtype=torch.int32, device=dev), torch.full((rows,), 77, dtype=torch.int64, device=dev)
    need = fp8lin.lib().fp8lin_verify_drafts_workspace_bytes(requests, rows, vocab)
    ws = torch.full((need,), 0x7f, dtype=torch.uint8, device=dev)
    rc = fp8lin.lib().fp8lin_verify_drafts(
        logits.data_ptr(), int(logits.dtype == torch.float32), logits.stride(0), None if q is None else q.data_ptr(), vocab,
        0 if q is None else q.size(0), tokens.data_ptr(), u.data_ptr(), off.data_ptr(),
        None if temperature is None else temperature.data_ptr(), requests, rows, vocab, accepted.data_ptr(), out.data_ptr(),
        ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return accepted.tolist(), out.tolist()


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("before,behind", [(0, 3), (1, 0), (5, 2), (200, 1)])
def test_verify_rows_of_no_request(fp8lin, gpu, before, behind, probs):
    """Rows before the first request and behind the last one: token -1, and the draft model's rows are those of the requests."""
    rng = random.Random(before)
    logits, tokens, u, offsets, q = _drafted(rng, 6, 3, 700, probs, torch.float32, 40 + before)
    g = torch.Generator().manual_seed(3)
    pad = lambda x, n: torch.rand(n, *x.shape[1:], generator=g).to(x.dtype)
    logits, tokens, u = [torch.cat([pad(x, before), x, pad(x, behind)]) for x in (logits, tokens, u)]
    offsets = [before + o for o in offsets]
    want = PO.verify(logits, tokens, u, offsets, q, None)
    got = _verify(fp8lin, logits.to(gpu), tokens.to(gpu), u.to(gpu), offsets, None if q is None else q.to(gpu))
    assert got == want


@pytest.mark.parametrize("probs", [False, True])
def test_verify_offsets_past_the_rows(fp8lin, gpu, probs):
    """A last request that is cut by the number of rows (a layout of fewer token rows than new tokens) is one of the rows that are
    there: its last row draws, over all columns."""
    vocab, rows = 5000, 7
    g = torch.Generator().manual_seed(6)
    x = torch.randn(rows, vocab, generator=g)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    for i in range(rows):  # each row's own token is likely: where it is taken for the row's draft, its weight is missing
        x[i, tokens[i]] = 12.0
    x[[3, 4, 5], tokens[4:7]] = 30.0
    q = torch.softmax(torch.randn(rows - 2, vocab, generator=g), 1) if probs else None
    for i in range(8):
        u = torch.rand(rows, generator=g)
        want = PO.verify(x, tokens, u, [0, 3, rows], q, None)
        for end in (rows + 1, rows + 5, 1 << 30):
            got = _verify(fp8lin, x.to(gpu), tokens.to(gpu), u.to(gpu), [0, 3, end], None if q is None else q.to(gpu))
            assert got == want, (i, end)
        assert want[0][1] == 3 or probs


@pytest.mark.parametrize("rows,given", [(4, 1), (4, 2), (6, 3), (2, 1)])
def test_verify_drafts_without_a_row(fp8lin, gpu, rows, given):
    """Fewer rows of draft probabilities than drafts: a draft without one is refused and the token drawn from p, as if the request
    ended there."""
    vocab = 900
    g = torch.Generator().manual_seed(rows)
    for i in range(12):
        x = torch.randn(rows, vocab, generator=g)
        tokens, u = torch.randint(0, vocab, (rows,), generator=g), torch.rand(rows, generator=g)
        x[torch.arange(rows - 1), tokens[1:]] = 9.0
        q = torch.softmax(x[:-1] + 0.5 * torch.randn(rows - 1, vocab, generator=g), 1)
        short = u[:given + 1].clone()
        short[given] = u[-1]
        kept, out = PO.verify(x[:given + 1], tokens[:given + 1], short, [0, given + 1], q, None)
        want = kept, out + [-1] * (rows - given - 1)
        got = _verify(fp8lin, x.to(gpu), tokens.to(gpu), u.to(gpu), [0, rows], q[:given].contiguous().to(gpu))
        assert got == want, i


@pytest.mark.parametrize("fp8", [False, True])
def test_full_attention_is_its_parts(fp8lin, gpu, fp8):
    """LinearEngine.full_attention of prompts, then of drafted tokens with rows of no request, against q, gate, k and v from
    full_attention_inputs: the cache's contents, 64-bit attention and a 64-bit product with o_proj's weights; rows of no request
    give zeros, whatever the memory held."""
    s = _Server(fp8lin, gpu, 3, fp8)
    H, HK, D = s.H, s.HK, s.D
    ints = dict(dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(8)
    codes, scale = s.eng.weights[s.P + ".o_proj.weight"].data, s.eng.weights[s.P + ".o_proj.weight"].scale
    w = codes.cpu().view(torch.float8_e4m3fn).double() * scale.cpu().double().view(codes.size(0), -1).repeat_interleave(128, 1)[:, :H * D] \
        if scale.dim() == 2 else codes.cpu().view(torch.float8_e4m3fn).double() * scale.cpu().double()[:, None]
    slots = {}
    for counts, extra in (([40, 17, 5], 0), ([3, 1, 4], 6), ([0, 1, 1], 30)):
        tokens = torch.randint(0, s.V, (sum(counts) + extra,), generator=g).to(gpu)
        x = s.embed[tokens]
        lay = fp8lin.paged_layout(s.lengths, torch.tensor(counts, **ints), s.table, s.free, tokens.numel(), s.PAGE, cursor=s.cursor, out=s.table)
        s.cursor.copy_(lay.cursor)
        junk = [torch.full((tokens.numel(), H, D), math.nan, dtype=torch.bfloat16, device=gpu) for _ in range(8)]
        del junk  # what the next tensors of this size hold
        args = (lay, *s.caches, *s.norms, H, HK, D, s.ROPE, 1e-6)
        y = s.eng.full_attention(x, s.P, *args, max_count=max(counts), **s.scales)
        pos = lay.positions.repeat(3, 1)
        again = s.eng.full_attention(x, s.P, *args, max_count=max(counts), positions=pos, **s.scales)
        assert torch.equal(y.view(torch.int16), again.view(torch.int16))
        q, gate, k, v = [t.cpu() for t in s.eng.full_attention_inputs(x, s.P, pos, *s.norms, H, HK, D, s.ROPE, 1e-6)]
        total = sum(counts)
        for i, slot in enumerate(lay.slots.tolist()[:total]):
            slots[slot] = k[i], v[i]
        caches = [c.cpu() for c in s.caches]
        for slot, rows in slots.items():
            for cache, row, name in zip(caches, rows, ("k_scale", "v_scale")):
                if fp8:
                    row = (row.float() / s.scales[name].cpu()[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
                assert torch.equal(cache[slot // s.PAGE, slot % s.PAGE].float(), row.float())
        sc = {n: t.cpu() for n, t in s.scales.items()}
        core, bound, rows = PV.attention(q, *caches, lay.block_table.cpu(), lay.offsets.tolist(), lay.lengths.tolist(),
                                         gate=gate.view(-1, H, D), **sc)
        assert rows.tolist() == [True] * total + [False] * extra
        core, bound = core.flatten(1), bound.flatten(1)
        # the operand's own bound; weights rounded to BF16 by some paths, FP32 sums, the result's rounding
        mass = core.abs() @ w.abs().t()
        off = bound @ w.abs().t() + (PO.BF16_HALF + 2 * PO.F32_HALF * H * D) * mass * 1.01

        def beyond(core):
            want = core @ w.t()
            return float(((y.double().cpu() - want).abs() - off - PO.BF16_HALF * want.abs() * 1.02)[:total].max())
        assert beyond(core) <= 0
        # a mistake of the heads' order, or of the dimensions', would show
        assert beyond(core.view(-1, H, D).roll(1, 1).flatten(1)) > 0 and beyond(core.view(-1, H, D).roll(1, 2).flatten(1)) > 0
        assert (y[total:] == 0).all()
        s.lengths.copy_(lay.lengths)


@pytest.mark.parametrize("heads,tokens", [((4, 2, 64), 1), ((4, 2, 64), 3), ((12, 2, 256), 70), ((12, 2, 256), 2000)], ids=str)
def test_positions_of_one_row(fp8lin, gpu, heads, tokens):
    """Positions expanded over the axes: the same bits as three rows of them, and no copy of them is made."""
    H, HK, D = heads
    g = torch.Generator().manual_seed(tokens)
    projected = torch.randn(tokens, 2 * (H + HK) * D, generator=g).to(torch.bfloat16).to(gpu)
    norms = [(0.1 * torch.randn(D, generator=g)).to(torch.bfloat16).to(gpu) for _ in range(2)]
    pos = torch.randint(0, 100000, (tokens,), generator=g).to(gpu)
    rest = (H, HK, D, D // 4, 10000.0, D // 32 - 1, D // 32, 1e-6)
    want = fp8lin.qk_norm_rope(projected, *norms, pos.repeat(3, 1), *rest)
    got = fp8lin.qk_norm_rope(projected, *norms, pos.expand(3, tokens), *rest)
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(got, want))
    expanded = pos.expand(3, tokens)
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    got = fp8lin.qk_norm_rope(projected, *norms, expanded, *rest)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] - before == 2  # q and k, no positions
    # a row that is no row of its own, strided: copied
    two = torch.stack([pos, pos + 1], 1)
    got = fp8lin.qk_norm_rope(projected, *norms, two[:, 0].expand(3, tokens), *rest)
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(got, want))


class _Loop:
    """A server's step of chunks and drafted requests together, every length on the GPU."""

    def __init__(self, F, dev, requests):
        self.s = _Server(F, dev, requests, False)
        self.F, self.u = F, None

    def step(self, tokens, counts, is_chunk, deciding, deciding_offsets, max_count):
        s = self.s
        layout = self.F.paged_layout(s.lengths, counts, s.table, s.free, tokens.numel(), s.PAGE, cursor=s.cursor)
        x = s.eng.full_attention(s.embed[tokens], s.P, layout, *s.caches, *s.norms, s.H, s.HK, s.D, s.ROPE, 1e-6, max_count=max_count)
        logits = s.eng.linear(x[deciding], "lm_head")
        taken, out = self.F.verify_drafts(logits, tokens[deciding], self.u, deciding_offsets)
        s.lengths.copy_(torch.where(is_chunk, layout.lengths, s.lengths + taken + (counts > 0)))
        s.cursor.copy_(layout.cursor)
        s.table.copy_(layout.block_table)
        return logits, taken, out


def test_chunks_beside_drafted_requests(fp8lin, gpu):
    """Prompts that arrive in chunks while other requests verify drafts: every request's cache holds at the end what one prompt
    of its tokens puts there."""
    n, chunk = 3, 24
    loop = _Loop(fp8lin, gpu, n)
    s = loop.s
    ints = dict(dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(12)
    prompts = [torch.randint(0, s.V, (c,), generator=g).tolist() for c in (100, 30, 7)]
    fed, last, kept = [0] * n, [None] * n, [[] for _ in range(n)]
    drafted_beside_chunk = 0
    for i in range(10):
        rows, deciding, parts, ends = [], [], [], []
        for b in range(n):
            a = sum(map(len, rows))
            if fed[b] < len(prompts[b]):
                new = prompts[b][fed[b]:fed[b] + chunk]
                ends.append(fed[b] + len(new) == len(prompts[b]))
                mine = [a + len(new) - 1] if ends[-1] else []
            else:
                new = [last[b]] + torch.randint(0, s.V, ((i + b) % 4,), generator=g).tolist()
                ends.append(None)
                mine = list(range(a, a + len(new)))
            rows.append(new)
            deciding += mine
            parts.append(len(mine))
        tokens = torch.tensor(sum(rows, []), device=gpu)
        offsets = [sum(parts[:b]) for b in range(n + 1)]
        counts = torch.tensor([len(r) for r in rows], **ints)
        loop.u = torch.rand(len(deciding), generator=g).to(gpu)
        logits, taken, out = loop.step(tokens, counts, torch.tensor([e is not None for e in ends], device=gpu),
                                       torch.tensor(deciding, dtype=torch.int64, device=gpu), torch.tensor(offsets, **ints), chunk)
        want = PO.verify(logits.cpu(), tokens[deciding].cpu(), loop.u.cpu(), offsets, None, None)
        assert taken.tolist() == want[0] and out.tolist() == want[1]
        drafted_beside_chunk += None in ends and any(e is not None for e in ends)
        for b in range(n):
            t, o = int(taken[b]), out.tolist()[offsets[b]:offsets[b + 1]]
            if ends[b] is None:
                kept[b] += [last[b]] + o[:t]
                last[b] = o[t]
            else:
                kept[b] += rows[b]
                fed[b] += len(rows[b])
                if ends[b]:
                    assert t == 0
                    last[b] = o[0]
        assert s.lengths.tolist() == [len(k) for k in kept]
    assert drafted_beside_chunk > 2
    t = _Server(fp8lin, gpu, n, False)
    _, lay = t.step(torch.tensor(sum(kept, []), device=gpu), torch.tensor([len(k) for k in kept], **ints), max(map(len, kept)))
    for b in range(n):
        for cache, other in zip(s.caches, t.caches):
            x, z = [PO.keys_of(c.cpu(), None, tab[b].cpu(), len(kept[b]), 1) for c, tab in ((cache, s.table), (other, lay.block_table))]
            assert torch.isfinite(x).all()
            assert float((x - z).norm() / z.norm()) <= torch.finfo(torch.bfloat16).eps


def test_chunk_and_drafts_captured(fp8lin, gpu):
    """The same step as one graph, replayed: the lengths advance by it, a chunk's by all its tokens, and equal the eager steps'."""
    states = []
    for form in ("eager", "graph"):
        loop = _Loop(fp8lin, gpu, 2)
        s = loop.s
        ints = dict(dtype=torch.int32, device=gpu)
        g = torch.Generator().manual_seed(5)
        loop.u = torch.full((3,), 0.5, device=gpu)
        tokens = torch.randint(0, s.V, (20 + 3 + 2,), generator=g).to(gpu)  # two rows of no request
        args = (tokens, torch.tensor([20, 3], **ints), torch.tensor([True, False], device=gpu),
                torch.tensor([20, 21, 22], device=gpu), torch.tensor([0, 0, 3], **ints), 20)
        saved = [x.clone() for x in (s.lengths, s.cursor, s.table, *s.caches)]
        if form == "graph":
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                loop.step(*args)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                res = loop.step(*args)
            for x, y in zip((s.lengths, s.cursor, s.table, *s.caches), saved):
                x.copy_(y)
        got = []
        for i in range(5):
            gi = torch.Generator().manual_seed(i)
            loop.u.copy_(torch.rand(3, generator=gi))
            tokens.copy_(torch.randint(0, s.V, (25,), generator=gi))
            torch.cuda.synchronize()
            if form == "graph":
                graph.replay()
            else:
                res = loop.step(*args)
            torch.cuda.synchronize()
            got += [x.clone().cpu() for x in (*res, s.lengths, s.cursor, s.table)]
            assert int(s.lengths[0]) == 20 * (i + 1) and int(s.lengths[1]) > i
        states.append(got)
    for x, y in zip(*states):
        assert torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x, y.view(torch.int16) if y.dtype == torch.bfloat16 else y)
