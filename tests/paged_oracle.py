"""Plain 64-bit forms of the paged-cache operators, written from their
definitions with loops over requests, heads and tokens, on the CPU."""
import math

import torch

BF16_HALF = torch.finfo(torch.bfloat16).eps / 2
F32_HALF = torch.finfo(torch.float32).eps / 2


def layout(lengths, counts, table, free, tokens, page, cursor=0):
    """offsets, lengths, slots, positions, table, cursor as lists."""
    table = [list(r) for r in table]
    offsets, after, slots, positions = [0], [], [], []
    for b, (n, c) in enumerate(zip(lengths, counts)):
        n, c = max(n, 0), max(c, 0)
        for pos in range(n, n + c):
            j = pos // page
            if j < len(table[b]) and table[b][j] < 0 and (pos == n or pos % page == 0):
                table[b][j] = free[cursor] if cursor < len(free) else -1
                cursor += 1
            there = j < len(table[b]) and table[b][j] >= 0
            slots.append(table[b][j] * page + pos % page if there else -1)
            positions.append(pos)
        offsets.append(offsets[-1] + c)
        after.append(n + c)
    slots = (slots + [-1] * tokens)[:tokens]
    positions = (positions + [0] * tokens)[:tokens]
    return offsets, after, slots, positions, table, cursor


def keys_of(cache, scale, table, length, head):
    """[length, D] float64 keys (values) of a request; zeros where the page id is out of range."""
    pages, page, _, d = cache.shape
    got = torch.zeros(length, d, dtype=torch.float64)
    for j in range(0, length, page):
        n, at = min(page, length - j), int(table[j // page])
        if 0 <= at < pages:
            got[j:j + n] = cache[at, :n, head].double()
    return got * float(scale[head]) if scale is not None else got


def attention(q, k_cache, v_cache, table, offsets, lengths, gate=None, k_scale=None, v_scale=None, scale=None, causal=True):
    """(out, bound) in float64: the result, NaN in rows of no request, and how far the kernel's may be.

    The kernel rounds each weight to BF16 (half a step of its value), which moves the result by at most that part of the
    sum of |w v|, and the result once.  A score is a sum of D products in FP32, off by at most D + 2 half steps of the sum
    of |q k| (products are exact; scaling, the subtraction of the maximum and 2^x are in the 2, for arguments of the order
    of the score), in any order; a weight and the sum of weights are off by that part each.  The sums over the keys are in
    FP32: their own half steps, once per key and once more per join of two parts.  The gate's sigmoid and products: 8 half steps."""
    t, h, d = q.shape
    hk = k_cache.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((t, h, d), math.nan, dtype=torch.float64)
    bound = torch.zeros(t, h, d, dtype=torch.float64)
    for b in range(len(lengths)):
        a, e, n = int(offsets[b]), int(offsets[b + 1]), int(lengths[b])
        if e <= a:
            continue
        limit = [min(max(n - (e - a) + i + 1, 0), n) if causal else n for i in range(e - a)]
        open_ = torch.arange(n)[None, :] < torch.tensor(limit)[:, None]
        for g in range(h):
            k = keys_of(k_cache, k_scale, table[b], n, g // (h // hk))
            v = keys_of(v_cache, v_scale, table[b], n, g // (h // hk))
            x = q[a:e, g].double()
            s = (x @ k.t() * scale).masked_fill(~open_, -math.inf)
            top = s.amax(1, keepdim=True) if n else torch.zeros(e - a, 1, dtype=torch.float64)
            w = torch.where(open_, torch.exp(s - torch.where(top > -math.inf, top, 0.0)), 0.0)
            total = w.sum(1, keepdim=True)
            w = torch.where(total > 0, w / total, 0.0)
            clean = torch.where(torch.isfinite(v), v, 0.0)
            o, mass = w @ clean, w @ clean.abs()
            # an infinity or NaN only counts for the rows that may see it
            for j in (~torch.isfinite(v)).any(1).nonzero()[:, 0].tolist():
                sees = open_[:, j]
                o[sees] = o[sees] + w[sees, j, None] * torch.where(torch.isfinite(v[j]), 0.0, v[j])
            spread = ((x.abs() @ k.abs().t()) * scale * open_).amax(1, keepdim=True) if n else torch.zeros(e - a, 1).double()
            weight = BF16_HALF + 2 * F32_HALF * ((d + 2) * spread + n + 600)
            sig = torch.sigmoid(gate[a:e, g].double()) if gate is not None else torch.ones(())
            out[a:e, g] = o * sig
            bound[a:e, g] = sig * (weight * mass + 8 * F32_HALF * o.abs()) * 1.01 + BF16_HALF * (o * sig).abs() * 1.01 + 1e-37
    return out, bound


def verify(logits, tokens, uniforms, offsets, draft_probs=None, temperature=None):
    """accepted, out as lists."""
    rows, vocab = logits.shape
    accepted, out, drafts = [], [-1] * rows, 0
    for b in range(len(offsets) - 1):
        a, n = int(offsets[b]), int(offsets[b + 1] - offsets[b])
        if n == 0:
            accepted.append(0)
            continue
        t = 1.0 if temperature is None else float(temperature[b])
        kept = 0
        while True:
            x = logits[a + kept].double()
            ok = bool((x < math.inf).all()) and bool((x > -math.inf).any())
            if t <= 0:
                p = torch.zeros(vocab, dtype=torch.float64)
                if ok:
                    p[int((x == x.max()).nonzero()[0])] = 1
            else:
                p = torch.softmax((x - (x.max() if ok else 0)) / t, 0)
            if kept == n - 1:
                w = p
                break
            draft = int(tokens[a + kept + 1])
            if draft_probs is not None:
                q = draft_probs[drafts + kept].double()
            else:
                q = torch.zeros(vocab, dtype=torch.float64)
                if 0 <= draft < vocab:
                    q[draft] = 1
            if not (ok and 0 <= draft < vocab and float(uniforms[a + kept]) * float(q[draft]) < float(p[draft])):
                w = (p - q).clamp_min(0)
                w = w if float(w.sum()) > 0 else p
                break
            kept += 1
        sums = w.cumsum(0)
        target = float(uniforms[a + n - 1]) * float(sums[-1])
        pick = int((sums <= target).sum())
        positive = (w > 0).nonzero()
        pick = min(pick, int(positive[-1])) if ok else -1
        accepted.append(kept)
        for i in range(kept):
            out[a + i] = int(tokens[a + i + 1])
        out[a + kept] = pick
        drafts += n - 1
    return accepted, out
