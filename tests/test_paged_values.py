"""The 64-bit attention of paged_values and its comparison, without a GPU: right where PO.attention is (finite inputs), and a
wrong output does not pass."""
import math

import pytest
import torch

import paged_oracle as PO
import paged_values as PV


def case(held, heads=4, kv_heads=2, dim=16, page=16, seed=0):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n, _ in held]
    table = torch.full((len(held), max(need) + 1), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(n) + sum(need[:b])
    k, v = [torch.randn(sum(need), page, kv_heads, dim, generator=g).to(torch.bfloat16) for _ in range(2)]
    counts = [c for _, c in held]
    offsets = [sum(counts[:i]) for i in range(len(counts) + 1)]
    q, gate = [torch.randn(offsets[-1] + 2, heads, dim, generator=g).to(torch.bfloat16) for _ in range(2)]
    return dict(q=q, k_cache=k, v_cache=v, table=table, offsets=offsets, lengths=[n for n, _ in held], gate=gate)


@pytest.mark.parametrize("causal", [True, False])
def test_equals_the_plain_form_on_finite_inputs(causal):
    c = case([(40, 4), (9, 9), (3, 5), (0, 1)])
    out, bound, rows = PV.attention(**c, causal=causal)
    plain, plain_bound = PO.attention(**c, causal=causal)
    assert rows.tolist() == [True] * 19 + [False] * 2
    assert torch.allclose(out[rows], plain[rows], rtol=1e-12, atol=1e-300)
    # the plain form's bound counts the scores of a row's own keys as well
    assert torch.allclose(bound[rows], plain_bound[rows], rtol=1e-9, atol=0)


def planted():
    """Two requests; NaN in a key of the first, infinities and a NaN in its values, a NaN in a query of the second."""
    c = case([(40, 6), (9, 9)])
    page = lambda b, at: (int(c["table"][b, at // 16]), at % 16)
    c["k_cache"][page(0, 38)][1, 3] = math.nan      # key of the last token but one, kv head 1
    c["v_cache"][page(0, 36)][0, 5] = math.inf      # seen by rows 2 .. of the 6
    c["v_cache"][page(0, 37)][0, 5] = -math.inf     # rows 3 ..: inf - inf
    c["v_cache"][page(0, 39)][0, 7] = math.nan      # row 5
    c["q"][6 + 2, 3, 0] = math.nan
    return c


def test_what_a_row_sees():
    out, bound, rows = PV.attention(**planted())
    odd = torch.zeros_like(out, dtype=torch.bool)
    odd[4:6, 2:] = True         # rows that see the NaN key, heads 2 and 3 of kv head 1
    odd[2:6, :2, 5] = True
    odd[5, :2, 7] = True
    odd[8, 3] = True
    assert torch.equal(~torch.isfinite(out) & rows[:, None, None], odd)
    assert (out[2, :2, 5] == math.inf).all() and torch.isnan(out[3:6, :2, 5]).all()
    assert torch.isfinite(bound).all() and (bound[rows] > 0).all()
    assert PV.compare(out, (out, bound, rows)) == 15 * 4 * 16 - int(odd.sum())


def test_wrong_outputs_do_not_pass():
    out, bound, rows = want = PV.attention(**planted())

    def changed(at, x):
        y = out.clone()
        y[at] = x
        return y
    bad = [torch.full_like(out, 123.0), torch.zeros_like(out), torch.full_like(out, math.nan),
           changed((0, 0, 0), math.nan), changed((0, 0, 0), math.inf), changed((0, 0, 0), out[0, 0, 0] + 2 * bound[0, 0, 0]),
           changed((2, 0, 5), -math.inf), changed((2, 0, 5), math.nan), changed((2, 0, 5), 1.0), changed((5, 2, 0), 0.0),
           changed((8, 3), 0.0)]
    for i, y in enumerate(bad):
        with pytest.raises(AssertionError):
            PV.compare(y, want)
            pytest.fail(f"output {i}")
    PV.compare(changed(15, 55.0), want)  # a row of no request
