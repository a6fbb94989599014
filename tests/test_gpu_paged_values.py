"""Paged attention over caches and queries that hold infinities and NaN, on the GPU against paged_values: every row of every
request is compared."""
import math

import pytest
import torch

import paged_values as PV
from test_gpu_paged import Batch

pytestmark = pytest.mark.gpu

NAN, INF = math.nan, math.inf


def expect(b, **kw):
    return PV.attention(b.q, b.k, b.v, b.table, b.offsets, b.lengths, gate=b.gate, k_scale=b.k_scale, v_scale=b.v_scale, **kw)


def put(b, cache, request, at, head, dim, x):
    cache[int(b.table[request, at // b.k.size(1)]), at % b.k.size(1), head, dim] = x


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(12, 2, 256), (8, 8, 64), (16, 1, 128)], ids=str)
@pytest.mark.parametrize("held", [[(40, 4), (9, 9)], [(70, 70)], [(300, 100), (33, 3), (1, 1)]], ids=str)
@pytest.mark.parametrize("where", ["keys", "values", "both"])
def test_attention_of_values_that_some_rows_see(fp8lin, gpu, where, held, heads, fp8):
    """Infinities and NaN in keys and values of later tokens of a chunk, in every other head: the rows before them are as if they
    were not there, the rows that see them get them."""
    b = Batch(held, *heads, page=16, fp8=fp8, gate=True, seed=13)
    h, hk, dim = heads
    odd = torch.zeros(b.tokens, h, dim, dtype=torch.bool)
    for r, (n, c) in enumerate(held):
        first, row0 = n - c, b.offsets[r]
        if c < 3:
            continue
        for head in range(0, hk, 2):
            mine = slice(head * h // hk, (head + 1) * h // hk)
            if where != "values":
                at = n - 1 - c // 4
                put(b, b.k, r, at, head, (7 * head + r) % dim, NAN)
                odd[row0 + at - first:row0 + c, mine] = True
            if where != "keys":
                for at, d, x in ((n - 1, 3, NAN), (n - c // 2, 5, INF), (n - c // 2, dim - 1, -INF)):
                    put(b, b.v, r, at, head, d, NAN if fp8 else x)  # E4M3FN has no infinities
                    odd[row0 + at - first:row0 + c, mine, d] = True
    want = expect(b)
    for count in (b.max_count, 1000):
        got = fp8lin.paged_attention(max_count=count, **b.up(gpu))
        assert PV.compare(got, want, str(count)) == odd.numel() - int(odd.sum())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(12, 2, 256), (4, 4, 64), (6, 1, 128)], ids=str)
@pytest.mark.parametrize("count", [3, 1000])
@pytest.mark.parametrize("what", ["query", "keys", "far"])
def test_attention_keeps_nan(fp8lin, gpu, what, count, heads, fp8):
    """Rows that NaN reach stay NaN, in units that are cut into pieces and whole ones, in both kernels: a NaN in a query; in every
    key that a row sees; in one key (and one value) whose piece weighs nothing beside another piece's."""
    held = [(1500, 2), (700, 1), (9, 3), (16, 1)]
    if count > 3:
        held = [(1500, 300), (900, 70), (100, 100), (5, 2)]
    b = Batch(held, *heads, page=16, fp8=fp8, gate=True, seed=17)
    h, hk, dim = heads
    odd = torch.zeros(b.tokens, h, dim, dtype=torch.bool)
    for r, (n, c) in enumerate(held):
        row0, head = b.offsets[r], r % hk
        mine = slice(head * h // hk, (head + 1) * h // hk)
        if what == "query":
            b.q[row0 + c - 1, r % h, 3] = NAN
            odd[row0 + c - 1, r % h] = True
        elif what == "keys":
            for at in range(n):
                put(b, b.k, r, at, head, at % dim, NAN)
            odd[row0:row0 + c, mine] = True
        elif n > 600:
            # keys of 0 in front: scores of 0; the others' some hundreds
            for at in range(n - c - 300):
                put(b, b.k, r, at, slice(None), slice(None), 0.0)
            b.q[row0:row0 + c] *= 30
            put(b, b.k, r, 5, head, 2, NAN)
            odd[row0:row0 + c, mine] = True
            if hk > 1:
                put(b, b.v, r, 7, (head + 1) % hk, 1, NAN)
                other = slice((head + 1) % hk * h // hk, ((head + 1) % hk + 1) * h // hk)
                odd[row0:row0 + c, other, 1] = True
    want = expect(b)
    for causal in (True, False):
        if not causal:
            if what != "query":
                break
            want = expect(b, causal=False)
        got = fp8lin.paged_attention(max_count=count, causal=causal, **b.up(gpu))
        assert PV.compare(got, want, f"causal={causal}") == odd.numel() - int(odd.sum())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", [(12, 2, 256), (4, 4, 64), (6, 1, 128)], ids=str)
@pytest.mark.parametrize("count", [3, 1000])
def test_attention_of_infinite_scores_and_gates(fp8lin, gpu, count, heads, fp8):
    """Infinities in queries, keys (BF16) and gates: +inf among a row's scores makes it NaN, -inf a weight of 0, nothing but -inf a row
    of zeros; gates of either infinity and NaN."""
    held = [(900, 2), (40, 3), (1, 1), (300, 1)] if count == 3 else [(900, 200), (70, 70), (5, 2)]
    b = Batch(held, *heads, page=16, fp8=fp8, gate=True, seed=23)
    h, hk, dim = heads
    b.q[0, 0, 2] = INF                                   # every score an infinity of the key's sign, or NaN
    b.q[b.offsets[1], h - 1] = 0.0
    b.q[b.offsets[1], h - 1, 1] = -INF                   # infinities and, of the zeros, nothing else
    if not fp8:
        put(b, b.k, 0, 17, hk - 1, 3, INF)
        put(b, b.k, 1, 4, 0, 1, -INF)
        for at in range(held[-1][0]):                    # one head whose every key is infinite: scores of one sign a row
            put(b, b.k, len(held) - 1, at, 0, 0, -INF)
    b.gate[1, :, 0], b.gate[1, :, 1], b.gate[1, :, 2] = INF, -INF, NAN
    want = expect(b)
    got = fp8lin.paged_attention(max_count=count, **b.up(gpu))
    compared = PV.compare(got, want)
    assert 0 < compared < want[0][want[2]].numel()
    if not fp8:
        last = want[0][b.offsets[-2]:b.offsets[-1], :h // hk]
        assert ((last == 0).all(-1) | torch.isnan(last).all(-1)).all()
