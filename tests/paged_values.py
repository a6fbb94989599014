"""Paged attention in 64 bits where keys, values and queries may hold infinities and NaN, on the CPU: what a row may not see
does not reach it, what it sees does.  And a comparison that checks every row of every request."""
import math

import torch

import paged_oracle as PO

BF16_HALF, F32_HALF = PO.BF16_HALF, PO.F32_HALF


def attention(q, k_cache, v_cache, table, offsets, lengths, gate=None, k_scale=None, v_scale=None, scale=None, causal=True):
    """(out, bound, rows): the result, how far the kernel's may be off (as PO.attention derives it; finite wherever the result is),
    and which rows belong to a request.

    A row's weights are exp(s - max) over the keys it may see: a NaN among those scores, or a +inf, makes the row NaN; scores
    of -inf alone, or no key, make it 0.  A value that is no finite number counts in the rows that may see its token."""
    t, h, d = q.shape
    group = h // k_cache.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out, bound = torch.zeros(t, h, d, dtype=torch.float64), torch.zeros(t, h, d, dtype=torch.float64)
    rows = torch.zeros(t, dtype=torch.bool)
    for b in range(len(lengths)):
        a, e, n = int(offsets[b]), int(offsets[b + 1]), int(lengths[b])
        rows[a:e] = True
        for g in range(h):
            k = PO.keys_of(k_cache, k_scale, table[b], n, g // group)
            v = PO.keys_of(v_cache, v_scale, table[b], n, g // group)
            for i in range(a, e):
                sees = min(max(n - (e - i) + 1, 0), n) if causal else n
                x, sig = q[i, g].double(), torch.ones(d).double() if gate is None else torch.sigmoid(gate[i, g].double())
                s = (k[:sees] * x).sum(1) * scale
                bound[i, g] = 1e-37
                if not sees or bool((s == -math.inf).all()):
                    continue
                if bool(torch.isnan(s).any()) or bool((s == math.inf).any()):
                    out[i, g] = math.nan
                    continue
                w = torch.exp(s - s.max())
                w = w / w.sum()
                vi = v[:sees]
                fine = torch.where(torch.isfinite(vi), vi, 0.0)
                o, mass = w @ fine, w @ fine.abs()
                odd = ~torch.isfinite(vi)
                for j in odd.any(1).nonzero()[:, 0].tolist():
                    o = torch.where(odd[j], o + w[j] * vi[j], o)
                spread = float((k[:sees].abs() * x.abs()).sum(1)[torch.isfinite(s)].max()) * scale
                weight = BF16_HALF + 2 * F32_HALF * ((d + 2) * spread + n + 600)
                out[i, g] = o * sig
                o, sig = torch.where(torch.isfinite(o * sig), o, 0.0), torch.where(torch.isfinite(o * sig), sig, 0.0)
                bound[i, g] += sig * (weight * mass + 8 * F32_HALF * o.abs()) * 1.01 + BF16_HALF * (o * sig).abs() * 1.01
    return out, bound, rows


def compare(got, want, what=""):
    """Every element of every request's rows: NaN and infinities where they should be, the rest within the bound.  Returns how many
    finite elements were compared."""
    out, bound, rows = want
    g, out, bound = got.double().cpu()[rows], out[rows], bound[rows]
    assert torch.isfinite(bound).all()
    assert torch.equal(torch.isnan(g), torch.isnan(out)), f"{what}: NaN in other places"
    inf = torch.isinf(out)
    assert torch.equal(torch.isinf(g), inf) and torch.equal(g[inf], out[inf]), f"{what}: other infinities"
    fine = torch.isfinite(out)
    err = ((g - out).abs() - bound)[fine]
    assert not err.numel() or float(err.max()) <= 0, f"{what}: {float(err.max())} beyond the bound"
    return int(fine.sum())
