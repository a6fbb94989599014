"""Serving over a paged cache: the layout of a step, the append to the cache,
attention of the new tokens over it, and the verification of drafted tokens.

They stand between `LinearEngine.full_attention_inputs` and the output
projection, and between the output head and the next step
(`LinearEngine.full_attention` runs the first part).  A step never waits for
the host: lengths, tables and counts stay on the device, so it can be captured
as one HIP graph.  All arithmetic runs in the HIP library (include/fp8lin.h
describes each operator); as in `ops`, work is enqueued on torch's current
stream of the tensors' device and violated preconditions raise Fp8linError.
"""
import ctypes
from collections import namedtuple

import torch

from ._lib import ERR_ARGUMENT, ERR_SHAPE, PagedCacheRecord, check, lib
from .ops import _fail, _is_dev, _stream

PagedLayout = namedtuple("PagedLayout", "offsets lengths slots positions block_table cursor")
PagedLayout.__doc__ = """What paged_layout returns: offsets int32 [requests + 1], lengths int32 [requests] after the step, slots and
positions int64 [tokens], block_table int32 [requests, width], cursor int32 [1]."""

_FP8 = (torch.float8_e4m3fn, torch.uint8)


def _vector(t, n, dtype, device, what):
    if not (_is_dev(t) and t.dtype == dtype and t.dim() == 1 and t.is_contiguous() and t.device == device and
            (n is None or t.size(0) == n)):
        _fail(ERR_ARGUMENT, what)


def _on(device, call):
    """call() with `device` current: the library launches on the current one."""
    if device.index is None or device.index == torch.cuda.current_device():
        return call()
    with torch.cuda.device(device):
        return call()


def paged_layout(lengths, counts, block_table, free_pages, tokens, page_size, cursor=None, out=None):
    """The layout of a step (fp8lin_paged_layout): request b holds lengths[b]
    tokens and gets counts[b] more (int32 [requests], on the device).
    block_table int32 [requests, width] holds page ids, negative where there is
    none; the pages that the new tokens need are taken from free_pages (int32)
    from index cursor[0] on, in the order of the requests.  tokens: rows of the
    step's token tensors, at least the sum of the counts; rows behind the last
    request get slot -1 and position 0.  Returns a PagedLayout: its block_table
    is a new tensor, or `out`, which may be block_table itself; its cursor goes
    into the next call and is above len(free_pages) when pages were short (their
    tokens have slot -1)."""
    if not (_is_dev(block_table) and block_table.dtype == torch.int32 and block_table.dim() == 2 and
            block_table.stride(1) == 1):
        _fail(ERR_ARGUMENT, "Invalid block table")
    device, (requests, width) = block_table.device, block_table.shape
    what = "Paged layout expects int32 vectors on the block table's device"
    _vector(lengths, requests, torch.int32, device, what)
    _vector(counts, requests, torch.int32, device, what)
    _vector(free_pages, None, torch.int32, device, what)
    if cursor is not None:
        _vector(cursor, 1, torch.int32, device, what)
    if out is None:
        out = torch.empty((requests, width), dtype=torch.int32, device=device)
    elif not (_is_dev(out) and out.device == device and out.dtype == torch.int32 and out.shape == block_table.shape and
              out.stride(1) == 1):
        _fail(ERR_ARGUMENT, "Invalid output block table")
    tokens = int(tokens)
    if tokens < 0:
        _fail(ERR_SHAPE, "Invalid number of tokens")
    whole = torch.empty(2 * requests + 2, dtype=torch.int32, device=device)
    rows = torch.empty((2, tokens), dtype=torch.int64, device=device)
    need = lib().fp8lin_paged_layout_workspace_bytes(requests)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=device)
    offsets, after, next_cursor = whole[:requests + 1], whole[requests + 1:2 * requests + 1], whole[2 * requests + 1:]
    _on(device, lambda: check(lib().fp8lin_paged_layout(
        lengths.data_ptr(), counts.data_ptr(), block_table.data_ptr(), block_table.stride(0), free_pages.data_ptr(),
        free_pages.numel(), cursor.data_ptr() if cursor is not None else None, requests, width, int(page_size), tokens,
        offsets.data_ptr(), after.data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(), out.data_ptr(), out.stride(0),
        next_cursor.data_ptr(), ws.data_ptr(), need, _stream(block_table))))
    return PagedLayout(offsets, after, rows[0], rows[1], out, next_cursor)


def _cache(k_cache, v_cache, k_scale, v_scale):
    """The library's record of a cache [pages, page_size, kv_heads, head_dim]
    (any strides, the last dimension contiguous), BF16 or E4M3FN codes
    (torch.float8_e4m3fn or uint8) with a float32 scale per kv head."""
    ok = (_is_dev(k_cache) and _is_dev(v_cache) and k_cache.dim() == 4 and k_cache.shape == v_cache.shape and
          k_cache.dtype == v_cache.dtype and k_cache.device == v_cache.device)
    if not ok:
        _fail(ERR_ARGUMENT, "Paged caches must be equal device tensors [pages, page_size, kv_heads, head_dim]")
    fp8 = k_cache.dtype in _FP8
    if not fp8 and k_cache.dtype != torch.bfloat16:
        _fail(ERR_ARGUMENT, "Paged caches must be BF16 or E4M3FN")
    ks, vs = k_cache.stride(), v_cache.stride()
    if ks[3] != 1 or vs[3] != 1:
        _fail(ERR_ARGUMENT, "Paged caches need a contiguous last dimension")
    pages, page_size, kv_heads, head_dim = k_cache.shape
    if fp8:
        _vector(k_scale, kv_heads, torch.float32, k_cache.device, "An 8-bit cache needs float32 k_scale [kv_heads]")
        _vector(v_scale, kv_heads, torch.float32, k_cache.device, "An 8-bit cache needs float32 v_scale [kv_heads]")
    elif k_scale is not None or v_scale is not None:
        _fail(ERR_ARGUMENT, "A BF16 cache has no scales")
    return PagedCacheRecord(k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], pages, page_size,
                            kv_heads, head_dim, int(fp8), k_scale.data_ptr() if fp8 else None,
                            v_scale.data_ptr() if fp8 else None)


def _heads(t, tokens, heads, dim, device, what):
    if not (_is_dev(t) and t.dtype == torch.bfloat16 and t.dim() == 3 and t.device == device and t.stride(2) == 1 and
            t.shape == (tokens, heads, dim)):
        _fail(ERR_ARGUMENT, what)


def paged_append(k, v, slots, k_cache, v_cache, k_scale=None, v_scale=None):
    """k and v (BF16 [tokens, kv_heads, head_dim], last dimension contiguous)
    into their slots (int64 [tokens]) of the caches, in place
    (fp8lin_paged_append); rows whose slot is outside the cache are skipped."""
    rec = _cache(k_cache, v_cache, k_scale, v_scale)
    if not (isinstance(k, torch.Tensor) and k.dim() == 3):
        _fail(ERR_ARGUMENT, "Paged append expects BF16 keys and values [tokens, kv_heads, head_dim]")
    device, tokens = k_cache.device, k.size(0)
    for t in (k, v):
        _heads(t, tokens, rec.kv_heads, rec.head_dim, device,
               "Paged append expects BF16 keys and values [tokens, kv_heads, head_dim]")
    _vector(slots, tokens, torch.int64, device, "Paged append expects int64 slots [tokens]")
    if tokens == 0:
        return
    _on(device, lambda: check(lib().fp8lin_paged_append(
        ctypes.byref(rec), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), slots.data_ptr(),
        tokens, _stream(k_cache))))


def paged_attention(q, k_cache, v_cache, block_table, offsets, lengths, max_count=None, gate=None, k_scale=None, v_scale=None,
                    scale=None, causal=True, out=None):
    """Attention of a step's new tokens over the paged cache, which holds their
    keys and values already (fp8lin_paged_attention).  q BF16 [tokens, heads,
    head_dim]; request b has rows offsets[b] .. offsets[b+1] (int32
    [requests + 1]), the last of its lengths[b] tokens (int32, new ones
    included).  out = softmax(scale q k^T) v over the keys up to each row's own
    token (all of the request's with causal=False), times sigmoid(gate) when a
    gate (as q) is given; scale defaults to head_dim ** -0.5.  max_count: the most
    rows that a request has (a hint that picks the kernel; by default the
    tokens beyond one per request).  Returns BF16 [tokens, heads, head_dim]:
    `out` if given, whose rows behind the last request stay as they were."""
    rec = _cache(k_cache, v_cache, k_scale, v_scale)
    device = k_cache.device
    if not (_is_dev(q) and q.dim() == 3 and q.dtype == torch.bfloat16 and q.stride(2) == 1 and q.device == device and
            q.size(2) == rec.head_dim):
        _fail(ERR_ARGUMENT, "Paged attention expects BF16 queries [tokens, heads, head_dim]")
    tokens, heads, dim = q.shape
    if heads == 0 or heads % rec.kv_heads:
        _fail(ERR_SHAPE, "Paged attention: heads must be a multiple of kv_heads")
    if not (_is_dev(block_table) and block_table.dtype == torch.int32 and block_table.dim() == 2 and
            block_table.device == device and block_table.stride(1) == 1):
        _fail(ERR_ARGUMENT, "Invalid block table")
    requests, width = block_table.shape
    _vector(offsets, requests + 1, torch.int32, device, "Paged attention expects int32 offsets [requests + 1]")
    _vector(lengths, requests, torch.int32, device, "Paged attention expects int32 lengths [requests]")
    if gate is not None:
        _heads(gate, tokens, heads, dim, device, "Paged attention expects a BF16 gate as the queries")
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=torch.bfloat16, device=device)
    else:
        _heads(out, tokens, heads, dim, device, "Paged attention expects a BF16 output as the queries")
    count = max(tokens - requests + 1, 1) if max_count is None else int(max_count)
    need = lib().fp8lin_paged_attention_workspace_bytes(heads, rec.kv_heads, dim, count)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=device)
    _on(device, lambda: check(lib().fp8lin_paged_attention(
        ctypes.byref(rec), q.data_ptr(), q.stride(0), q.stride(1), gate.data_ptr() if gate is not None else None,
        gate.stride(0) if gate is not None else 0, gate.stride(1) if gate is not None else 0, block_table.data_ptr(),
        block_table.stride(0), width, offsets.data_ptr(), lengths.data_ptr(), requests, tokens, heads, count, int(bool(causal)),
        float(scale) if scale is not None else dim ** -0.5, out.data_ptr(), out.stride(0), out.stride(1), ws.data_ptr(), need,
        _stream(q))))
    return out


def verify_drafts(logits, tokens, uniforms, offsets, draft_probs=None, temperature=None):
    """Verification of drafted tokens (fp8lin_verify_drafts).  Request b has
    rows offsets[b] .. offsets[b+1] (int32 [requests + 1]) of the target's
    logits (BF16 or FP32 [rows, vocab]), after its last token and after each of
    its drafts; tokens (int64 [rows]) were fed in, so its drafts are tokens but
    its first row's.  uniforms (float32 [rows], in [0, 1)): a row's number
    decides its draft, a request's last one draws its next token.
    draft_probs (float32 [rows - requests, vocab]): the draft model's
    distributions, the rows of all requests but each one's last; None: drafts
    without probabilities.  temperature (float32 [requests], 0: the most likely
    token).  Returns (accepted int32 [requests], out int64 [rows]: per request
    the drafts kept, the next token, then -1)."""
    if not (_is_dev(logits) and logits.dim() == 2 and logits.dtype in (torch.bfloat16, torch.float32) and
            logits.stride(1) == 1 and logits.size(1) > 0):
        _fail(ERR_ARGUMENT, "Verification expects BF16 or FP32 logits [rows, vocab]")
    device, (rows, vocab) = logits.device, logits.shape
    _vector(tokens, rows, torch.int64, device, "Verification expects int64 tokens [rows]")
    _vector(uniforms, rows, torch.float32, device, "Verification expects float32 uniforms [rows]")
    _vector(offsets, None, torch.int32, device, "Verification expects int32 offsets [requests + 1]")
    requests = offsets.size(0) - 1
    if requests < 1:
        _fail(ERR_SHAPE, "Verification expects offsets of at least one request")
    if draft_probs is not None and not (_is_dev(draft_probs) and draft_probs.dim() == 2 and draft_probs.device == device and
                                        draft_probs.dtype == torch.float32 and draft_probs.size(1) == vocab and
                                        draft_probs.stride(1) == 1):
        _fail(ERR_ARGUMENT, "Verification expects float32 draft probabilities [drafts, vocab]")
    if temperature is not None:
        _vector(temperature, requests, torch.float32, device, "Verification expects float32 temperatures [requests]")
    accepted = torch.empty(requests, dtype=torch.int32, device=device)
    out = torch.empty(rows, dtype=torch.int64, device=device)
    need = lib().fp8lin_verify_drafts_workspace_bytes(requests, rows, vocab)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=device)
    # an empty tensor has a null pointer: without rows it stands for "no draft is left to test"
    probs = draft_probs if draft_probs is not None and draft_probs.numel() else None
    _on(device, lambda: check(lib().fp8lin_verify_drafts(
        logits.data_ptr(), int(logits.dtype == torch.float32), logits.stride(0) if rows > 1 else vocab,
        probs.data_ptr() if probs is not None else None,
        (probs.stride(0) if probs.size(0) > 1 else vocab) if probs is not None else vocab,
        probs.size(0) if probs is not None else 0, tokens.data_ptr(), uniforms.data_ptr(), offsets.data_ptr(),
        temperature.data_ptr() if temperature is not None else None, requests, rows, vocab, accepted.data_ptr(),
        out.data_ptr(), ws.data_ptr(), need, _stream(logits))))
    return accepted, out
