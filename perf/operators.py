"""The operators of a serving step over a paged cache, as cases to time and
compare: the paged layout of a step, the append to the cache, the attention of
the new tokens over it, and the verification of drafted tokens.

`run` takes the state that a server holds before the call.  With `own` it makes
fp8lin's calls; without, the same in elementary torch operations.

Head layouts are one rank's of the shipped configuration (24/4 heads of 256
over two ranks, a gate per query head, vocabulary 248320) and generic ones.
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "a100-vision-infer_amd"))

own = False

RANK = {"heads": 12, "kv_heads": 2, "head_dim": 256}


def listed():
    return [
        # one request's next token, the smallest step: the call itself counts
        {"name": "layout_1", "kind": "layout", "requests": 1, "count_max": 1, "chunks": 0, "len_max": 4001, "width": 1280, "page": 16,
         "mix": 1},
        # a large batch: drafted tokens of most requests, prompt chunks of some
        {"name": "layout_509", "kind": "layout", "requests": 509, "count_max": 6, "chunks": 5, "len_max": 20000, "width": 1280,
         "page": 16, "mix": 2},
        # the new keys and values of a batched decode step
        {"name": "append_27", "kind": "append", "tokens": 27, "pages": 512, "page": 16, "cache": "bf16", **RANK},
        # a prompt in one piece into an 8-bit cache
        {"name": "append_fp8_3913", "kind": "append", "tokens": 3913, "pages": 512, "page": 64, "cache": "fp8", **RANK},
        # the decode loop of one request
        {"name": "decode_1", "kind": "attention", "requests": 1, "chunks": 0, "count_max": 1, "len_max": 4001, "page": 16,
         "cache": "bf16", "gate": True, "mix": 3, **RANK},
        # a batched decode step over contexts of all lengths, 8-bit cache
        {"name": "decode_fp8_61", "kind": "attention", "requests": 61, "chunks": 0, "count_max": 1, "len_max": 20480, "page": 64,
         "cache": "fp8", "gate": True, "mix": 4, **RANK},
        # drafted tokens of a few requests to verify, every head on one card
        {"name": "drafts_7", "kind": "attention", "requests": 7, "chunks": 0, "count_max": 4, "len_max": 12000, "page": 16,
         "cache": "bf16", "gate": True, "mix": 5, "heads": 24, "kv_heads": 4, "head_dim": 256},
        # a chunk of a long prompt
        {"name": "chunk_512", "kind": "attention", "requests": 1, "chunks": 1, "count_max": 512, "len_max": 7431, "page": 16,
         "cache": "bf16", "gate": True, "mix": 6, **RANK},
        # a prompt of text and image tokens in one piece, the largest call
        {"name": "prompt_3913", "kind": "attention", "requests": 1, "chunks": 1, "count_max": 3913, "len_max": 3913, "page": 16,
         "cache": "bf16", "gate": True, "mix": 7, **RANK},
        # prompt chunks beside decoding requests, generic heads of 128 without a gate
        {"name": "mixed_13", "kind": "attention", "requests": 13, "chunks": 3, "count_max": 700, "len_max": 6000, "page": 32,
         "cache": "bf16", "gate": False, "mix": 8, "heads": 32, "kv_heads": 8, "head_dim": 128},
        # three drafted tokens of one request, taken from a draft without probabilities
        {"name": "verify_1", "kind": "verify", "requests": 1, "drafts": 3, "vocab": 248320, "probs": False, "mix": 9},
        # a batch, drafted by a sampled draft model
        {"name": "verify_48", "kind": "verify", "requests": 48, "drafts": 5, "vocab": 248320, "probs": True, "mix": 10},
    ]


def _log_range(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["layout", "append", "attention", "attention", "attention", "verify"])
    mix = rng.randrange(1 << 30)
    if kind == "layout":
        requests = _log_range(rng, 1, 509)
        return {"kind": kind, "requests": requests, "count_max": rng.randint(1, 6), "chunks": rng.randint(0, min(5, requests)),
                "len_max": _log_range(rng, 16, 20000), "width": 1280, "page": rng.choice([16, 32, 64]), "mix": mix}
    if kind == "append":
        return {"kind": kind, "tokens": _log_range(rng, 1, 3913), "pages": 512, "page": rng.choice([16, 32, 64]),
                "cache": rng.choice(["bf16", "fp8"]), **_heads(rng)}
    if kind == "verify":
        return {"kind": kind, "requests": _log_range(rng, 1, 48), "drafts": rng.randint(0, 5), "vocab": _log_range(rng, 1000, 248320),
                "probs": rng.random() < 0.5, "mix": mix}
    case = {"kind": kind, "page": rng.choice([16, 32, 64, 128]), "cache": rng.choice(["bf16", "fp8"]), "gate": rng.random() < 0.5,
            "mix": mix, **_heads(rng)}
    form = rng.choice(["decode", "drafts", "chunk", "mixed"])
    if form == "decode":
        case.update(requests=_log_range(rng, 1, 61), chunks=0, count_max=1, len_max=_log_range(rng, 1, 20480))
    elif form == "drafts":
        case.update(requests=_log_range(rng, 1, 32), chunks=0, count_max=rng.randint(2, 8), len_max=_log_range(rng, 8, 12000))
    elif form == "chunk":
        count = _log_range(rng, 9, 3000)
        case.update(requests=1, chunks=1, count_max=count, len_max=_log_range(rng, count, 4 * count + 2000))
    else:
        case.update(requests=rng.randint(2, 13), chunks=rng.randint(1, 2), count_max=_log_range(rng, 9, 500),
                    len_max=_log_range(rng, 500, 4000))
    # no larger than the largest listed case, in bytes and operations
    while work(case)["flops"] > 9e10 or work(case)["bytes"] > 4.5e8:
        case["len_max"] = case["len_max"] * 3 // 4
        case["count_max"] = min(case["count_max"], case["len_max"])
    return case


def _heads(rng):
    heads, kv, dim = rng.choice([(12, 2, 256), (24, 4, 256), (32, 8, 128), (28, 4, 128), (8, 8, 64), (16, 2, 64)])
    return {"heads": heads, "kv_heads": kv, "head_dim": dim}


def _lengths(case):
    """The requests' (length before the step, new tokens): the first `chunks` requests bring up to count_max new tokens (one of
    them all), the others one to count_max (to four beside chunks), in a drawn order; the longest context is len_max."""
    rng, n, top = random.Random(case["mix"]), case["requests"], case["count_max"]
    few = min(top, 4) if case["chunks"] else top
    # a layout's chunks are prompts, of 64 times as many tokens as its drafts
    long = top * 64 if case["kind"] == "layout" else top
    got = []
    for i in range(n):
        count = long if i == 0 and case["chunks"] else rng.randint(max(1, long // 4), long) if i < case["chunks"] else rng.randint(1, few)
        room = max(0, case["len_max"] - count)
        before = room if i == 0 else int(room * rng.random() ** 1.5)
        got.append((before, count))
    rng.shuffle(got)
    return got


# ---- what a server holds before the call --------------------------------------


class _Inputs:
    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def bf16(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.bfloat16)

    def ints(self, lo, hi, *shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=self.gen, device="cuda").to(dtype)

    def perm(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _pages_of(length, page):
    return -(-length // page)


def _offsets(counts):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    return {"case": case, **{"layout": _layout_inputs, "append": _append_inputs, "attention": _attention_inputs,
                             "verify": _verify_inputs}[case["kind"]](case, _Inputs(seed))}


def _layout_inputs(case, r):
    """Block tables with the pages of the tokens that are there (and of a few rejected drafts), the rest of the pool free."""
    held, page, width = _lengths(case), case["page"], case["width"]
    before = torch.tensor([b for b, _ in held], device="cuda")
    counts = torch.tensor([c for _, c in held], device="cuda")
    have = (before + page - 1) // page + (r.ints(0, 4, len(held)) == 0)
    at = torch.arange(width, device="cuda")[None]
    ids = r.perm(len(held) * width).view(len(held), width)
    table = torch.where(at < have[:, None], ids, -1)
    free = ids[at >= have[:, None]]
    return {"lengths": before.int(), "counts": counts.int(), "block_table": table.int(), "free_pages": free.int().contiguous(),
            "cursor": torch.tensor([3], dtype=torch.int32, device="cuda"), "tokens": sum(c for _, c in held), "page_size": page}


def _scales(r, case):
    """An 8-bit cache's scale of each head: four standard deviations at the top of the range, more or less."""
    return 4.0 / 448 * (1 + 0.5 * r.ints(0, 5, case["kv_heads"]).float())


def _append_inputs(case, r):
    t, hk, d, page, pages = case["tokens"], case["kv_heads"], case["head_dim"], case["page"], case["pages"]
    projected = r.bf16(t, 2 * (case["heads"] + hk) * d)
    fp8 = case["cache"] == "fp8"
    caches = [r.bf16(pages, page, hk, d) for _ in range(2)]
    return {"k": r.bf16(t, hk, d), "v": projected[:, -hk * d:].unflatten(1, (hk, d)), "slots": r.perm(pages * page)[:t],
            "k_cache": caches[0].to(torch.float8_e4m3fn) if fp8 else caches[0],
            "v_cache": caches[1].to(torch.float8_e4m3fn) if fp8 else caches[1],
            "k_scale": _scales(r, case) if fp8 else None, "v_scale": _scales(r, case) if fp8 else None}


def _attention_inputs(case, r):
    held, page, hk, d = _lengths(case), case["page"], case["kv_heads"], case["head_dim"]
    counts, lengths = [c for _, c in held], [b + c for b, c in held]
    width = _pages_of(max(lengths), page)
    need = [_pages_of(n, page) for n in lengths]
    pages = sum(need) + 5
    ids = r.perm(pages).int()
    table = torch.full((len(held), width), -1, dtype=torch.int32, device="cuda")
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    at = torch.arange(width, device="cuda")
    there = at[None] < torch.tensor(need, device="cuda")[:, None]
    table[there] = ids[(first[:, None] + at[None])[there]]
    fp8 = case["cache"] == "fp8"
    k, v = r.bf16(pages, page, hk, d), r.bf16(pages, page, hk, d)
    scales = (_scales(r, case), _scales(r, case)) if fp8 else (None, None)
    if fp8:
        k, v = [(x / s[:, None].to(torch.bfloat16)).to(torch.float8_e4m3fn) for x, s in ((k, scales[0]), (v, scales[1]))]
    total = sum(counts)
    query_gate = r.bf16(total, case["heads"], 2 * d)
    # normed heads times a learned weight: scores with a standard deviation of about two
    return {"q": (2 * query_gate[..., :d]).contiguous(), "gate": query_gate[..., d:] if case["gate"] else None, "k_cache": k, "v_cache": v,
            "k_scale": scales[0], "v_scale": scales[1], "block_table": table, "offsets": _offsets(counts),
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "max_count": max(counts)}


def _verify_inputs(case, r):
    """Logits of a trained head (a few likely tokens above a wide floor), and drafts from a nearby distribution."""
    rng, v, n = random.Random(case["mix"]), case["vocab"], case["requests"]
    counts = [1 + (case["drafts"] if i == 0 else rng.randint(0, case["drafts"])) for i in range(n)]
    total = sum(counts)
    offsets = _offsets(counts)
    logits = r.normal(total, v)
    lift = r.ints(0, v, total, 12, dtype=torch.int64)
    logits.scatter_add_(1, lift, 8 + 3 * r.normal(total, 12))
    last = torch.zeros(total, dtype=torch.bool, device="cuda")
    last[offsets[1:].long() - 1] = True
    near = logits[~last]
    near = near + 0.5 * r.normal(*near.shape)
    if case["probs"]:
        noise = -torch.log(-torch.log(torch.rand(near.shape, generator=r.gen, device="cuda").clamp_min(1e-20)).clamp_min(1e-20))
        drafts = (near + noise).argmax(1)
    else:
        drafts = near.argmax(1)
    tokens = r.ints(0, v, total, dtype=torch.int64)
    first = torch.zeros(total, dtype=torch.bool, device="cuda")
    first[offsets[:-1].long()] = True
    tokens[~first] = drafts
    return {"logits": logits.to(torch.bfloat16), "tokens": tokens, "offsets": offsets, "draft_probs": near.softmax(1) if case["probs"] else None,
            "uniforms": torch.rand(total, generator=r.gen, device="cuda"), "temperature": 0.5 + 0.75 * torch.rand(n, generator=r.gen, device="cuda")}


# ---- one pass -------------------------------------------------------------------


def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        return _run_own(s, kind)
    return {"layout": _layout, "append": _append, "attention": _attention, "verify": _verify}[kind](s)


def _run_own(s, kind):
    import fp8lin
    if kind == "layout":
        return fp8lin.paged_layout(s["lengths"], s["counts"], s["block_table"], s["free_pages"], s["tokens"], s["page_size"],
                                   cursor=s["cursor"])
    if kind == "append":
        fp8lin.paged_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return s["k_cache"], s["v_cache"]
    if kind == "attention":
        return fp8lin.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["offsets"], s["lengths"],
                                      max_count=s["max_count"], gate=s["gate"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return fp8lin.verify_drafts(s["logits"], s["tokens"], s["uniforms"], s["offsets"], draft_probs=s["draft_probs"],
                                temperature=s["temperature"])


def _layout(s):
    """offsets, lengths after the step, slots, positions, the block table with the pages it takes, the pool's cursor."""
    before, counts, table, free, page = s["lengths"].long(), s["counts"].long(), s["block_table"], s["free_pages"], s["page_size"]
    width = table.size(1)
    offsets = torch.nn.functional.pad(counts.cumsum(0), (1, 0))
    after = before + counts
    at = torch.arange(width, device=table.device)[None]
    fresh = (at >= (before // page)[:, None]) & (at < ((after + page - 1) // page)[:, None]) & (counts > 0)[:, None] & (table < 0)
    rank = fresh.flatten().cumsum(0).view_as(table) - 1 + s["cursor"]
    taken = torch.where(rank < free.numel(), free[rank.clamp(0, free.numel() - 1)], table)
    table = torch.where(fresh, taken, table)
    rows = torch.arange(s["tokens"], device=table.device)
    req = torch.searchsorted(offsets[1:].contiguous(), rows, right=True).clamp_max(before.numel() - 1)
    pos = before[req] + rows - offsets[req]
    col = pos // page
    ids = table[req, col.clamp_max(width - 1)].long()
    slots = torch.where((col < width) & (ids >= 0), ids * page + pos % page, -1)
    return offsets.int(), after.int(), slots, pos, table, (s["cursor"] + fresh.sum()).int()


def _append(s):
    caches = s["k_cache"], s["v_cache"]
    rows = _rows(s["k"], s["k_scale"], caches[0].dtype), _rows(s["v"], s["v_scale"], caches[1].dtype)
    _store(caches[0], s["slots"], rows[0])
    _store(caches[1], s["slots"], rows[1])
    return caches


def _rows(x, scale, dtype):
    return x if scale is None else (x.float() / scale[:, None]).clamp(-448, 448).to(dtype)


def _store(cache, slots, rows):
    # one-byte types have no index_put: the same bytes as integers
    flat = cache.flatten(0, 1)
    as_int = torch.int16 if cache.element_size() == 2 else torch.uint8
    flat.view(as_int)[slots] = rows.contiguous().view(as_int)


def _attention(s):
    """softmax(q k^T / sqrt(d)) v over the keys up to each new token's own, times sigmoid(gate)."""
    q, table, lengths = s["q"], s["block_table"].long(), s["lengths"].long()
    heads, d = q.shape[1:]
    offsets = s["offsets"].long()
    counts = offsets.diff()
    page, hk = s["k_cache"].shape[1:3]
    most, longest = s["max_count"], table.size(1) * page
    # the requests' rows and keys, padded to the longest
    step = torch.arange(most, device=q.device)
    rows = (offsets[:-1, None] + step).clamp_max(q.size(0) - 1)
    kv = [c[table.clamp_min(0)].flatten(1, 2).float() if x is None else c[table.clamp_min(0)].flatten(1, 2).float() * x[:, None]
          for c, x in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]))]
    k, v = [x.permute(0, 2, 1, 3) for x in kv]
    group = heads // hk
    qp = q[rows].float().view(-1, most, hk, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = torch.matmul(qp, k.transpose(-1, -2).contiguous()) / math.sqrt(d)
    limit = (lengths - counts)[:, None] + step
    masked = torch.arange(longest, device=q.device) > limit[..., None]
    scores = scores.unflatten(2, (group, most)).masked_fill_(masked[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(weights.flatten(2, 3), v.contiguous()) / weights.sum(-1).flatten(2, 3)[..., None]
    out = out.unflatten(2, (group, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    owner = torch.searchsorted(offsets[1:].contiguous(), torch.arange(q.size(0), device=q.device), right=True)
    out = out[owner, torch.arange(q.size(0), device=q.device) - offsets[owner]]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].float())
    return out.to(torch.bfloat16)


def _verify(s):
    """Accepted drafts and the tokens of the step.  In 64 bits: a draw lies next to a border of the cumulative sum."""
    logits, tokens, offsets, u = s["logits"].double(), s["tokens"], s["offsets"].long(), s["uniforms"].double()
    total, vocab = logits.shape
    counts = offsets.diff()
    rows = torch.arange(total, device=logits.device)
    owner = torch.searchsorted(offsets[1:].contiguous(), rows, right=True)
    p = torch.softmax(logits / s["temperature"].double()[owner, None], -1)
    is_draft = rows + 1 < offsets[owner + 1]
    token = tokens[(rows + 1).clamp_max(total - 1)]
    p_at = p.gather(1, token[:, None])[:, 0]
    # a request's drafts are its rows but the last: the draft model's row of row t is t - owner
    if s["draft_probs"] is not None:
        q_row = (rows - owner).clamp_max(max(s["draft_probs"].size(0) - 1, 0))
        q_at = s["draft_probs"][q_row, token].double() if s["draft_probs"].size(0) else p_at
    else:
        q_at = 1.0
    refused = is_draft & ~(u * q_at < p_at)
    # the first refused row of each request, or its last
    stop = torch.where(refused | ~is_draft, rows, total)
    stop = torch.full_like(counts, total).scatter_reduce(0, owner, stop, "amin")
    short = is_draft[stop]
    w = p[stop]
    if s["draft_probs"] is None:
        less = torch.nn.functional.one_hot(token[stop], vocab).to(w.dtype) * w
    elif s["draft_probs"].size(0):
        less = s["draft_probs"][q_row[stop]].double()
    else:
        less = 0.0
    w = torch.where(short[:, None], (w - less).clamp_min(0), w)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p[stop])
    sums = w.cumsum(-1)
    pick = (sums <= u[offsets[1:] - 1][:, None] * sums[:, -1:]).sum(-1)
    highest = vocab - 1 - (w > 0).flip(-1).int().argmax(-1)
    pick = torch.minimum(pick, highest)
    accepted = stop - offsets[:-1]
    out = torch.where(rows < stop[owner], token, torch.where(rows == stop[owner], pick[owner], -1))
    return accepted.int(), out


# ---- what a pass cannot do without ----------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "layout":
        held = _lengths(case)
        tokens, n = sum(c for _, c in held), len(held)
        taken = sum(_pages_of(b + c, case["page"]) - _pages_of(b, case["page"]) for b, c in held)
        return {"bytes": 8 * n + 8 * n * case["width"] + 4 * taken + 4 * (n + 1) + 4 * n + 16 * tokens + 8, "flops": 0}
    if kind == "append":
        values = 2 * case["tokens"] * case["kv_heads"] * case["head_dim"]
        return {"bytes": values * (2 + (1 if case["cache"] == "fp8" else 2)) + 8 * case["tokens"], "flops": 0}
    if kind == "attention":
        held, h, hk, d = _lengths(case), case["heads"], case["kv_heads"], case["head_dim"]
        tokens, keys = sum(c for _, c in held), sum(b + c for b, c in held)
        pairs = sum(c * b + c * (c + 1) // 2 for b, c in held)
        return {"bytes": 2 * keys * hk * d * (1 if case["cache"] == "fp8" else 2) + 2 * tokens * h * d * (3 if case["gate"] else 2),
                "flops": 4.0 * pairs * h * d}
    rng, n = random.Random(case["mix"]), case["requests"]
    drafts = case["drafts"] + sum(rng.randint(0, case["drafts"]) for _ in range(n - 1))
    return {"bytes": case["vocab"] * (2 * (drafts + n) + (4 * drafts if case["probs"] else 0)) + 24 * (drafts + n),
            "flops": 4.0 * case["vocab"] * (drafts + n)}


# ---- the same in 64 bits ----------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"layout": _exact_layout, "append": _exact_append, "attention": _exact_attention, "verify": _exact_verify}[case["kind"]](s)


def _exact_layout(s):
    page, tables, free, cursor = s["page_size"], s["block_table"].tolist(), s["free_pages"].tolist(), s["cursor"].tolist()[0]
    offsets, after, slots, positions = [0], [], [], []
    for length, count, table in zip(s["lengths"].tolist(), s["counts"].tolist(), tables):
        for position in range(length, length + count):
            entry = position // page
            if entry < len(table) and table[entry] < 0:
                table[entry] = free[cursor] if cursor < len(free) else -1
                cursor += 1
            there = entry < len(table) and table[entry] >= 0
            slots.append(table[entry] * page + position % page if there else -1)
            positions.append(position)
        offsets.append(offsets[-1] + count)
        after.append(length + count)

    def whole(x, t):
        return torch.tensor(x, dtype=t)

    return (whole(offsets, torch.int32), whole(after, torch.int32), whole(slots, torch.int64), whole(positions, torch.int64),
            whole(tables, torch.int32), whole([cursor], torch.int32))


def _exact_append(s):
    got = []
    for x, cache, scale in ((s["k"], s["k_cache"], s["k_scale"]), (s["v"], s["v_cache"], s["v_scale"])):
        flat = cache.double().flatten(0, 1)
        flat[s["slots"]] = x.double() if scale is None else (x.double() / scale.double()[:, None]).clamp(-448, 448)
        got.append(flat.view(cache.shape))
    return tuple(got)


def _exact_attention(s):
    q, out = s["q"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    offsets, lengths = s["offsets"].tolist(), s["lengths"].tolist()
    page, hk, d = s["k_cache"].shape[1:]
    group = q.size(1) // hk
    for i, length in enumerate(lengths):
        a, b = offsets[i], offsets[i + 1]
        ids = s["block_table"][i, :_pages_of(length, page)].long()
        for h in range(hk):
            k, v = [c[ids][:, :, h].double().reshape(-1, d)[:length] for c in (s["k_cache"], s["v_cache"])]
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            future = torch.arange(length, device="cuda")[None] > torch.arange(length - (b - a), length, device="cuda")[:, None]
            for g in range(group):
                scores = (q[a:b, h * group + g].double() @ k.t()) * d ** -0.5
                out[a:b, h * group + g] = torch.softmax(scores.masked_fill(future, -math.inf), -1) @ v
    return out if s["gate"] is None else out / (1 + torch.exp(-s["gate"].double()))


def _exact_verify(s):
    offsets, taken, out = s["offsets"].tolist(), [], []
    tokens, u = s["tokens"].tolist(), s["uniforms"].double().tolist()
    for i, (a, b) in enumerate(zip(offsets, offsets[1:])):
        n = 0
        while True:
            x = s["logits"][a + n].double() / s["temperature"][i].double()
            p = torch.exp(x - torch.logsumexp(x, 0))
            if a + n + 1 == b:
                w = p
                break
            draft = tokens[a + n + 1]
            if s["draft_probs"] is None:
                q = torch.zeros_like(p)
                q[draft] = 1
            else:
                q = s["draft_probs"][a + n - i].double()
            if not u[a + n] * float(q[draft]) < float(p[draft]):
                w = torch.relu(p - q)
                w = w if float(w.sum()) > 0 else p
                break
            n += 1
        sums = w.cumsum(0)
        pick = int(torch.searchsorted(sums, u[b - 1] * sums[-1], right=True))
        pick = min(pick, int(w.nonzero()[-1]))
        taken.append(n)
        out += tokens[a + 1:a + 1 + n] + [pick] + [-1] * (b - a - n - 1)
    return torch.tensor(taken, dtype=torch.int32), torch.tensor(out, dtype=torch.int64)
