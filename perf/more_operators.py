"""Operators of a serving step whose cache is held in 8 bits with a scale for
each block of tokens and head, as cases to time and compare: the rotation of
heads by their positions, the append to the cache with the rotation (and the
heads' norm) on the way, and the attention over such a cache.

`run` takes the state that a server holds before the call.  With `own` it makes
fp8lin's calls; without, the same in elementary torch operations.

Head layouts are one rank's of the shipped configuration (24/4 heads of 256
over two ranks, a quarter of each head rotated, a gate per query head) and
generic ones.
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "a100-vision-infer_amd"))

own = False

RANK = {"heads": 12, "kv_heads": 2, "head_dim": 256}
QUARTER = {"rotary": 64, "pairs": "half", "theta": 10000000.0}
EPS = 1e-6


def listed():
    return [
        # one token's query heads far into a context stretched to eight times its length, the smallest call
        {"name": "rotate_1", "kind": "rotate", "tokens": 1, "heads": 24, "head_dim": 256, "axes": 1, "scaling": "yarn", "first": 1500001, **QUARTER},
        # a prompt of text and image tokens, read in place beside the gates
        {"name": "rotate_axes_3913", "kind": "rotate", "tokens": 3913, "heads": 12, "head_dim": 256, "axes": 3, "scaling": "none", "first": 0, **QUARTER},
        # a long prompt's whole heads, neighbouring dimensions as pairs
        {"name": "rotate_8191", "kind": "rotate", "tokens": 8191, "heads": 32, "head_dim": 128, "rotary": 128, "pairs": "neighbours", "theta": 500000.0,
         "axes": 1, "scaling": "linear", "first": 77},
        # one request's next token: the call itself counts
        {"name": "append_1", "kind": "append", "requests": 1, "chunks": 0, "count_max": 1, "len_max": 4001, "page": 16, "block": 16, "cache": "blocks",
         "norm": True, "mix": 1, **RANK, **QUARTER},
        # a batched decode step
        {"name": "append_61", "kind": "append", "requests": 61, "chunks": 0, "count_max": 1, "len_max": 2048, "page": 64, "block": 64, "cache": "blocks",
         "norm": True, "mix": 2, **RANK, **QUARTER},
        # a prompt in one piece
        {"name": "append_3913", "kind": "append", "requests": 1, "chunks": 1, "count_max": 3913, "len_max": 3913, "page": 64, "block": 64,
         "cache": "blocks", "norm": True, "mix": 3, **RANK, **QUARTER},
        # prompt chunks beside decoding requests into a BF16 cache, whole heads of 128 without a norm
        {"name": "append_bf16_mixed", "kind": "append", "requests": 13, "chunks": 3, "count_max": 700, "len_max": 6000, "page": 32, "block": 32,
         "cache": "bf16", "norm": False, "mix": 4, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128, "pairs": "half", "theta": 500000.0},
        # the decode loop of one request
        {"name": "decode_1", "kind": "attention", "requests": 1, "chunks": 0, "count_max": 1, "len_max": 4001, "page": 16, "block": 16, "gate": True,
         "mix": 5, **RANK},
        # a batched decode step over contexts of all lengths
        {"name": "decode_61", "kind": "attention", "requests": 61, "chunks": 0, "count_max": 1, "len_max": 20480, "page": 64, "block": 64, "gate": True,
         "mix": 6, **RANK},
        # drafted tokens of a few requests to verify, every head on one card
        {"name": "drafts_7", "kind": "attention", "requests": 7, "chunks": 0, "count_max": 4, "len_max": 12000, "page": 32, "block": 16, "gate": True,
         "mix": 7, "heads": 24, "kv_heads": 4, "head_dim": 256},
        # prompt chunks beside decoding requests, generic heads of 128 without a gate
        {"name": "mixed_13", "kind": "attention", "requests": 13, "chunks": 3, "count_max": 700, "len_max": 6000, "page": 128, "block": 32, "gate": False,
         "mix": 8, "heads": 32, "kv_heads": 8, "head_dim": 128},
        # a prompt of text and image tokens in one piece, the largest call
        {"name": "prompt_3913", "kind": "attention", "requests": 1, "chunks": 1, "count_max": 3913, "len_max": 3913, "page": 64, "block": 64,
         "gate": True, "mix": 9, **RANK},
    ]


def _log_range(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    heads, kv, dim = rng.choice([(12, 2, 256), (24, 4, 256), (32, 8, 128), (28, 4, 128), (8, 8, 64), (16, 2, 64)])
    return {"heads": heads, "kv_heads": kv, "head_dim": dim}


def _rotary(rng, dim):
    # whole heads, a part of them, and a part that is no multiple of eight pairs
    return {"rotary": rng.choice([dim, dim, dim // 2, dim // 4, 20]), "pairs": rng.choice(["half", "neighbours"]),
            "theta": rng.choice([10000.0, 500000.0, 10000000.0])}


def draw(rng):
    kind = rng.choice(["rotate", "append", "append", "attention", "attention"])
    mix = rng.randrange(1 << 30)
    if kind == "rotate":
        dim = rng.choice([64, 80, 96, 128, 256])
        return {"kind": kind, "tokens": _log_range(rng, 1, 4000), "heads": rng.randint(1, 32), "head_dim": dim, **_rotary(rng, dim),
                "axes": rng.choice([1, 1, 3]), "scaling": rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]), "first": _log_range(rng, 1, 1000000)}
    page = rng.choice([16, 32, 64, 128])
    case = {"kind": kind, "page": page, "block": rng.choice([b for b in (16, 32, 64, 128) if b <= page]), "mix": mix, **_heads(rng)}
    if kind == "append":
        case.update(cache=rng.choice(["blocks", "blocks", "heads", "bf16"]), norm=rng.random() < 0.5, **_rotary(rng, case["head_dim"]))
    else:
        case.update(gate=rng.random() < 0.5)
    form = rng.choice(["decode", "drafts", "chunk", "mixed"])
    long = 20480 if kind == "attention" else 2048
    if form == "decode":
        case.update(requests=_log_range(rng, 1, 61), chunks=0, count_max=1, len_max=_log_range(rng, 1, long))
    elif form == "drafts":
        case.update(requests=_log_range(rng, 1, 32), chunks=0, count_max=rng.randint(2, 8), len_max=_log_range(rng, 8, long // 2))
    elif form == "chunk":
        count = _log_range(rng, 9, 3000)
        case.update(requests=1, chunks=1, count_max=count, len_max=_log_range(rng, count, 4 * count + 2000))
    else:
        case.update(requests=rng.randint(2, 13), chunks=rng.randint(1, 2), count_max=_log_range(rng, 9, 500), len_max=_log_range(rng, 500, 4000))
    # no larger than the largest listed case, in bytes and operations
    while kind == "attention" and (work(case)["flops"] > 9e10 or work(case)["bytes"] > 4.5e8):
        case["len_max"] = case["len_max"] * 3 // 4
        case["count_max"] = min(case["count_max"], case["len_max"])
    return case


def _lengths(case):
    """The requests' (length before the step, new tokens): the first `chunks` requests bring up to count_max new tokens (one of
    them all), the others one to count_max (to four beside chunks), in a drawn order; the longest context is len_max."""
    rng, n, top = random.Random(case["mix"]), case["requests"], case["count_max"]
    few = min(top, 4) if case["chunks"] else top
    got = []
    for i in range(n):
        count = top if i == 0 and case["chunks"] else rng.randint(max(1, top // 4), top) if i < case["chunks"] else rng.randint(1, few)
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

    def bf16(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.bfloat16)

    def ints(self, lo, hi, *shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=self.gen, device="cuda").to(dtype)

    def perm(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _pages_of(length, page):
    return -(-length // page)


def prepare(case, seed):
    return {"case": case, **{"rotate": _rotate_inputs, "append": _append_inputs, "attention": _attention_inputs}[case["kind"]](case, _Inputs(seed))}


def _frequencies(rotary, theta, scaling):
    """Radians per position of each pair (64 bits), and what the cosines and sines are multiplied by."""
    j = torch.arange(rotary // 2, dtype=torch.float64)
    f = theta ** (-2 * j / rotary)
    if scaling == "linear":
        return f / 4, 1.0
    if scaling == "ntk":
        return (theta * 4 ** (rotary / max(rotary - 2, 1))) ** (-2 * j / rotary), 1.0
    if scaling == "yarn":
        # pairs that turn fewer than once in the original context are stretched by the factor, those that turn over 32 times are kept
        factor, original = 8.0, 32768
        low, high = [rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(low), 0), min(math.ceil(high), rotary - 1)
        ramp = ((j - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1
    if scaling == "wavelength":
        # by the turns of a pair in the original context: under one stretched, over four kept
        kept = ((8192 * f / (2 * math.pi) - 1) / (4 - 1)).clamp(0, 1)
        return f * kept + f / 8 * (1 - kept), 1.0
    return f, 1.0


def _rotation(case):
    """The plan that a program keeps: each pair's part of a turn per position (units of 2^-64 turns, the position's axis in the
    two lowest bits), and the same as frequencies and axes."""
    freq, magnitude = _frequencies(case["rotary"], case["theta"], case.get("scaling", "none"))
    half = case["rotary"] // 2
    j = torch.arange(half)
    axes = torch.zeros(half, dtype=torch.int64)
    if case.get("axes", 1) == 3:
        # height and width in the second and third of each three pairs, as far as their sections go
        section = half // 3
        axes = torch.where((j % 3 == 1) & (j < 3 * section), 1, torch.where((j % 3 == 2) & (j < 3 * section), 2, 0))
    steps = [(round(f / (2 * math.pi) * 2 ** 62) * 4 + a) % 2 ** 64 for f, a in zip(freq.tolist(), axes.tolist())]
    steps = torch.tensor([s - 2 ** 64 if s >= 2 ** 63 else s for s in steps], dtype=torch.int64)
    return {"steps": steps.cuda(), "magnitude": magnitude, "neighbours": case["pairs"] == "neighbours", "freq": freq.cuda(), "axes": axes.cuda()}


def _rotate_inputs(case, r):
    t, h, d = case["tokens"], case["heads"], case["head_dim"]
    query_gate = r.bf16(t, h, 2 * d)
    positions = case["first"] + torch.arange(t, device="cuda")
    if case["axes"] == 3:
        # an image's tokens share their first position, and have a row and a column
        positions = torch.stack([positions // 7 * 7, positions // 7 * 7 + r.ints(0, 40, t, dtype=torch.int64), positions])
    return {"x": query_gate[..., :d], "positions": positions, **_rotation(case)}


def _values(r, pages, page, block, hk, d):
    """Normal values whose size differs from block to block and head to head."""
    x = r.bf16(pages, page // block, block, hk, d)
    return x * torch.exp2(r.ints(-1, 2, pages, page // block, 1, hk, 1).float()).to(torch.bfloat16)


def _to_blocks(x):
    """[pages, blocks, block, heads, dim] as E4M3 codes and the power of two of each block and head: the least that holds its largest value."""
    mantissa, power = torch.frexp(x.float().abs().amax((2, 4)))
    power = (power - torch.where(mantissa <= 0.875, 9, 8)).clamp(-120, 120)
    codes = (x.float() * torch.exp2(-power.float())[:, :, None, :, None]).to(torch.float8_e4m3fn)
    return codes.flatten(1, 2), (power + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _tables(held, page, r, spare):
    """A table of shuffled pages for the requests' tokens after the step, and how many pages there are."""
    need = [_pages_of(b + c, page) for b, c in held]
    pages, width = sum(need) + spare, max(need)
    ids = r.perm(pages).int()
    table = torch.full((len(held), width), -1, dtype=torch.int32, device="cuda")
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    at = torch.arange(width, device="cuda")
    there = at[None] < torch.tensor(need, device="cuda")[:, None]
    table[there] = ids[(first[:, None] + at[None])[there]]
    return table, pages


def _head_scales(r, hk):
    """A scale of each head: four standard deviations at the top of the range, more or less."""
    return 4.0 / 448 * (1 + 0.5 * r.ints(0, 5, hk).float())


def _append_inputs(case, r):
    held, page, block, h, hk, d = _lengths(case), case["page"], case["block"], case["heads"], case["kv_heads"], case["head_dim"]
    table, pages = _tables(held, page, r, 5)
    positions = torch.cat([torch.arange(b, b + c) for b, c in held]).cuda()
    owner = torch.cat([torch.full((c,), i) for i, (_, c) in enumerate(held)]).cuda()
    slots = table[owner, positions // page].long() * page + positions % page
    t = positions.numel()
    projected = r.bf16(t, 2 * (h + hk) * d)
    k, v = [_values(r, pages, page, block, hk, d) for _ in range(2)]
    if case["cache"] == "blocks":
        (k, k_scale), (v, v_scale) = _to_blocks(k), _to_blocks(v)
    elif case["cache"] == "heads":
        k_scale, v_scale = _head_scales(r, hk), _head_scales(r, hk)
        k, v = [(x.flatten(1, 2) / s[:, None].to(torch.bfloat16)).clamp(-448, 448).to(torch.float8_e4m3fn) for x, s in ((k, k_scale), (v, v_scale))]
    else:
        k, v, k_scale, v_scale = k.flatten(1, 2), v.flatten(1, 2), None, None
    norms = [0.3 * r.bf16(d) for _ in range(2)] if case["norm"] else [None, None]
    # the projection's queries beside their gates, its keys and its values: read where they are
    return {"q": projected[:, :2 * h * d].unflatten(1, (h, 2 * d))[..., :d], "k": projected[:, 2 * h * d:(2 * h + hk) * d].unflatten(1, (hk, d)),
            "v": projected[:, (2 * h + hk) * d:].unflatten(1, (hk, d)), "positions": positions, "slots": slots, "k_cache": k, "v_cache": v,
            "k_scale": k_scale, "v_scale": v_scale, "q_norm": norms[0], "k_norm": norms[1], **_rotation(case)}


def _attention_inputs(case, r):
    held, page, block, hk, d = _lengths(case), case["page"], case["block"], case["kv_heads"], case["head_dim"]
    counts, lengths = [c for _, c in held], [b + c for b, c in held]
    table, pages = _tables(held, page, r, 5)
    k, k_scale = _to_blocks(_values(r, pages, page, block, hk, d))
    v, v_scale = _to_blocks(_values(r, pages, page, block, hk, d))
    offsets = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    query_gate = r.bf16(sum(counts), case["heads"], 2 * d)
    # normed heads times a learned weight: scores with a standard deviation of one to four
    return {"q": (2 * query_gate[..., :d]).contiguous(), "gate": query_gate[..., d:] if case["gate"] else None, "k_cache": k, "v_cache": v,
            "k_scale": k_scale, "v_scale": v_scale, "block_table": table, "offsets": offsets,
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "max_count": max(counts)}


# ---- one pass -------------------------------------------------------------------


def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        return _run_own(s, kind)
    return {"rotate": _rotate, "append": _append, "attention": _attention}[kind](s)


def _run_own(s, kind):
    import fp8lin
    if kind == "attention":
        return fp8lin.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["offsets"], s["lengths"],
                                      max_count=s["max_count"], gate=s["gate"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    plan = fp8lin.RotaryPlan(s["steps"], s["magnitude"], s["neighbours"])
    if kind == "rotate":
        return fp8lin.rotate(s["x"], s["positions"], plan)
    q = fp8lin.paged_rotate_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_cache"], s["v_cache"], plan, q_norm=s["q_norm"],
                                   k_norm=s["k_norm"], eps=EPS, k_scale=s["k_scale"], v_scale=s["v_scale"])
    return (q, s["k_cache"], s["v_cache"]) + ((s["k_scale"], s["v_scale"]) if s["case"]["cache"] == "blocks" else ())


def _rotated(s, x, positions):
    """x [tokens, heads, dim] in 32 bits, its first dimensions turned by position times frequency; the angle in 64 bits."""
    half = s["freq"].numel()
    at = positions[s["axes"]].t() if positions.dim() == 2 else positions[:, None]
    turns = at.double() * (s["freq"] / (2 * math.pi))
    angle = ((turns - turns.floor()) * (2 * math.pi)).float()
    c, z = s["magnitude"] * torch.cos(angle)[:, None], s["magnitude"] * torch.sin(angle)[:, None]
    if s["neighbours"]:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * z, b * c + a * z], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * c - b * z, b * c + a * z], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _rotate(s):
    return _rotated(s, s["x"].float(), s["positions"]).to(torch.bfloat16)


def _normed(x, weight):
    x = x.float()
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + weight.float())


def _append(s):
    q = _rotated(s, _normed(s["q"], s["q_norm"]), s["positions"]).to(torch.bfloat16)
    rows = _rotated(s, _normed(s["k"], s["k_norm"]), s["positions"]), s["v"].float()
    out = [q]
    for x, cache, scale in zip(rows, (s["k_cache"], s["v_cache"]), (s["k_scale"], s["v_scale"])):
        if s["case"]["cache"] == "blocks":
            _store_blocks(cache, scale, x, s["slots"], s["case"]["block"])
        else:
            x = x if scale is None else (x / scale[:, None]).clamp(-448, 448)
            _as_int(cache).flatten(0, 1)[s["slots"]] = _as_int(x.to(cache.dtype))
        out.append(cache)
    return tuple(out) + ((s["k_scale"], s["v_scale"]) if s["case"]["cache"] == "blocks" else ())


def _as_int(x):
    # one-byte types have no index_put: the same bytes as integers
    return x.view(torch.int16 if x.element_size() == 2 else torch.uint8)


def _store_blocks(cache, scale, x, slots, block):
    """The rows as codes in units of their block's power of two, which holds its largest value: a block whose first slot is among
    the rows' starts with theirs (its other slots hold nothing yet), another one's grows where it has to, and its codes with it."""
    old = scale.view(torch.uint8).flatten(0, 1).int()
    at = slots // block
    mantissa, power = torch.frexp(x.abs().amax(-1))
    need = (power - torch.where(mantissa <= 0.875, 9, 8)).clamp(-120, 120).int() + 127
    starts = torch.zeros(old.size(0), dtype=torch.int32, device=old.device).scatter_reduce(0, at, (slots % block == 0).int(), "amax") > 0
    held = torch.where(starts[:, None], 0, old)
    new = held.scatter_reduce(0, at[:, None].expand_as(need), need, "amax")
    codes = cache.unflatten(1, (-1, block)).flatten(0, 1)
    shift = torch.where((new > held) & ~starts[:, None], held - new, 0).clamp_min(-126)
    grown = (codes.float() * torch.exp2(shift.float())[:, None, :, None]).to(torch.float8_e4m3fn)
    _as_int(cache).copy_(_as_int(grown).view(cache.shape))
    _as_int(cache).flatten(0, 1)[slots] = _as_int((x * torch.exp2(127.0 - new[at])[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn))
    scale.view(torch.uint8).copy_(new.to(torch.uint8).view(scale.shape))


def _opened(cache, scale, pages):
    """The pages' values [requests, keys, heads, dim] in 32 bits."""
    blocks = scale.size(1)
    power = torch.exp2(scale.view(torch.uint8)[pages].float() - 127)
    return (cache[pages].float().unflatten(2, (blocks, -1)) * power[:, :, :, None, :, None]).flatten(1, 3)


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
    k, v = [_opened(c, x, table.clamp_min(0)).permute(0, 2, 1, 3) for c, x in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]))]
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


# ---- what a pass cannot do without ----------------------------------------------


def work(case):
    kind, h, d = case["kind"], case["heads"], case["head_dim"]
    if kind == "rotate":
        t = case["tokens"]
        return {"bytes": 4 * t * h * d + 8 * t * case["axes"], "flops": 3.0 * t * h * case["rotary"]}
    held, hk = _lengths(case), case["kv_heads"]
    tokens = sum(c for _, c in held)
    if kind == "append":
        blocks = sum(_pages_of(b + c, case["block"]) - b // case["block"] for b, c in held) if case["cache"] == "blocks" else 0
        return {"bytes": 4 * tokens * h * d + 2 * tokens * hk * d * (2 + (2 if case["cache"] == "bf16" else 1)) + 16 * tokens + 4 * blocks * hk,
                "flops": 3.0 * tokens * (h + hk) * case["rotary"] + (4.0 * tokens * (h + hk) * d if case["norm"] else 0)}
    keys = sum(b + c for b, c in held)
    pairs = sum(c * b + c * (c + 1) // 2 for b, c in held)
    return {"bytes": 2 * keys * hk * d + 2 * keys // case["block"] * hk + 2 * tokens * h * d * (3 if case["gate"] else 2), "flops": 4.0 * pairs * h * d}


# ---- the same in 64 bits ----------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "append": _exact_append, "attention": _exact_attention}[case["kind"]](s)


def _exact_turn(s, x, positions):
    """By complex numbers: each pair times magnitude e^(i angle)."""
    case = s["case"]
    freq, magnitude = _frequencies(case["rotary"], case["theta"], case.get("scaling", "none"))
    n, x = case["rotary"], x.double()
    at = positions.view(-1, x.size(0)).double()
    angle = torch.stack([at[a] * f for a, f in zip(s["axes"].tolist(), freq.tolist())], 1)
    z = torch.polar(torch.full_like(angle, magnitude), angle)[:, None]
    first, second = (x[..., :n].unflatten(-1, (-1, 2)).unbind(-1) if s["neighbours"] else x[..., :n].unflatten(-1, (2, -1)).unbind(-2))
    z = z * torch.complex(first.contiguous(), second.contiguous())
    y = x.clone()
    if s["neighbours"]:
        y[..., 0:n:2], y[..., 1:n:2] = z.real, z.imag
    else:
        y[..., :n // 2], y[..., n // 2:n] = z.real, z.imag
    return y


def _exact_rotate(s):
    return _exact_turn(s, s["x"], s["positions"])


def _exact_norm(x, weight):
    x = x.double()
    return x if weight is None else x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.size(-1) + EPS) * (weight.double() + 1)


def _exact_append(s):
    case, slots = s["case"], s["slots"].tolist()
    k = _exact_turn(s, _exact_norm(s["k"], s["k_norm"]), s["positions"])
    caches, powers = [], []
    for x, cache, scale in ((k, s["k_cache"], s["k_scale"]), (s["v"].double(), s["v_cache"], s["v_scale"])):
        flat = cache.double().flatten(0, 1)
        if case["cache"] == "blocks":
            block, power = case["block"], scale.view(torch.uint8).double().flatten(0, 1) - 127
            rows_of = {}
            for i, slot in enumerate(slots):
                rows_of.setdefault(slot // block, []).append(i)
            for at, rows in rows_of.items():
                # the least power of two that 448 times it holds the largest value
                need = torch.ceil(torch.log2(x[rows].abs().amax((0, 2)) / 448))
                new = need if any(slots[i] % block == 0 for i in rows) else torch.maximum(need, power[at])
                if not any(slots[i] % block == 0 for i in rows):
                    flat[at * block:(at + 1) * block] *= torch.exp2(power[at] - new)[:, None]
                power[at] = new
                flat[[slots[i] for i in rows]] = x[rows] / torch.exp2(new)[:, None]
            powers.append(torch.exp2(power).view(scale.shape))
        else:
            flat[slots] = x if scale is None else (x / scale.double()[:, None]).clamp(-448, 448)
        caches.append(flat.view(cache.shape))
    return (_exact_turn(s, _exact_norm(s["q"], s["q_norm"]), s["positions"]), *caches, *powers)


def _exact_attention(s):
    q, out = s["q"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    offsets, lengths = s["offsets"].tolist(), s["lengths"].tolist()
    page, hk, d = s["k_cache"].shape[1:]
    group = q.size(1) // hk
    for i, length in enumerate(lengths):
        a, b = offsets[i], offsets[i + 1]
        ids = s["block_table"][i, :_pages_of(length, page)].long()
        for h in range(hk):
            k, v = [(c[ids][:, :, h].double() * (2.0 ** (x.view(torch.uint8)[ids][:, :, h].double() - 127)).repeat_interleave(page // x.size(1), 1)
                     [..., None]).reshape(-1, d)[:length] for c, x in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]))]
            future = torch.arange(length, device="cuda")[None] > torch.arange(length - (b - a), length, device="cuda")[:, None]
            for g in range(group):
                scores = (q[a:b, h * group + g].double() @ k.t()) * d ** -0.5
                out[a:b, h * group + g] = torch.softmax(scores.masked_fill(future, -math.inf), -1) @ v
    return out if s["gate"] is None else out / (1 + torch.exp(-s["gate"].double()))
