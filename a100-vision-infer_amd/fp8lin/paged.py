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
from .ops import _fail, _is_dev, _ready_devices, _stream

PagedLayout = namedtuple("PagedLayout", "offsets lengths slots positions block_table cursor")
PagedLayout.__doc__ = """What paged_layout returns: offsets int32 [requests + 1], lengths int32 [requests] after the step, slots and
positions int64 [tokens], block_table int32 [requests, width], cursor int32 [1]."""

_FP8 = (torch.float8_e4m3fn, torch.uint8)


# Calls of this module take the host about as long as the GPU where batches are
# small, so their checks are one expression each and call nothing twice.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice
_byref, _i32, _i64, _f32, _bf16 = ctypes.byref, torch.int32, torch.int64, torch.float32, torch.bfloat16


def _call(name, device, *args):
    """A library call on the device's current torch stream, with that device
    current: the library launches on the current one."""
    index = device.index
    if index not in _ready_devices:
        _stream(torch.empty(0, device=device))  # prepares the device once
    if index == _current():
        rc = getattr(lib(), name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = getattr(lib(), name)(*args, _raw_stream(index))
    if rc:
        check(rc)


def _vector(t, n, dtype, device):
    """Whether t is a contiguous vector of n (None: any number) on the device."""
    return (isinstance(t, torch.Tensor) and t.dtype is dtype and t.dim() == 1 and t.device == device and t.is_contiguous() and
            (n is None or t.size(0) == n))


def paged_layout(lengths, counts, block_table, free_pages, tokens, page_size, cursor=None, out=None):
    """The layout of a step (fp8lin_paged_layout): request b holds lengths[b]
    tokens and gets counts[b] more (int32 [requests], on the device).
    block_table int32 [requests, width] holds page ids, negative where there is
    none; the pages that the new tokens need are taken from free_pages (int32)
    from index cursor[0] on, in the order of the requests.  tokens: rows of the
    step's token tensors, at least the sum of the counts; rows behind the last
    request get slot -1 and position 0.  Returns a PagedLayout: its block_table
    is a new tensor, or `out`, which may be block_table itself (and overlap no
    other input); its cursor goes into the next call and is above
    len(free_pages) when pages were short (their tokens have slot -1)."""
    if not (_is_dev(block_table) and block_table.dtype is _i32 and block_table.dim() == 2 and block_table.stride(1) == 1):
        _fail(ERR_ARGUMENT, "Invalid block table")
    device, (requests, width) = block_table.device, block_table.shape
    if not (_vector(lengths, requests, _i32, device) and _vector(counts, requests, _i32, device) and
            _vector(free_pages, None, _i32, device) and (cursor is None or _vector(cursor, 1, _i32, device))):
        _fail(ERR_ARGUMENT, "Paged layout expects int32 vectors on the block table's device")
    if out is None:
        out = lengths.new_empty((requests, width))
    elif not (_is_dev(out) and out.device == device and out.dtype is _i32 and out.shape == block_table.shape and
              out.stride(1) == 1):
        _fail(ERR_ARGUMENT, "Invalid output block table")
    tokens = int(tokens)
    if tokens < 0:
        _fail(ERR_SHAPE, "Invalid number of tokens")
    offsets, after, next_cursor = lengths.new_empty(requests + 1), lengths.new_empty(requests), lengths.new_empty(1)
    slots = torch.empty(tokens, dtype=_i64, device=device)
    positions = slots.new_empty(tokens)
    at, to = block_table.data_ptr(), out.data_ptr()
    need = lib().fp8lin_paged_layout_workspace_bytes(requests, int(at == to))
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _call("fp8lin_paged_layout", device, lengths.data_ptr(), counts.data_ptr(), at, _row_stride(block_table, width),
          free_pages.data_ptr(), free_pages.numel(), cursor.data_ptr() if cursor is not None else None, requests, width,
          int(page_size), tokens, offsets.data_ptr(), after.data_ptr(), slots.data_ptr(), positions.data_ptr(), to,
          _row_stride(out, width), next_cursor.data_ptr(), ws.data_ptr() if need else None, need)
    return PagedLayout(offsets, after, slots, positions, out, next_cursor)


def _row_stride(t, width):
    """The stride of a matrix' rows; torch leaves that of a single row open."""
    return t.stride(0) if t.size(0) > 1 else width


def _cache(k_cache, v_cache, k_scale, v_scale):
    """The library's record of a cache [pages, page_size, kv_heads, head_dim]
    (any strides, the last dimension contiguous), BF16 or E4M3FN codes
    (torch.float8_e4m3fn or uint8) with a float32 scale per kv head."""
    if not (_is_dev(k_cache) and isinstance(v_cache, torch.Tensor) and k_cache.dim() == 4 and
            k_cache.shape == v_cache.shape and k_cache.dtype is v_cache.dtype and k_cache.device == v_cache.device):
        _fail(ERR_ARGUMENT, "Paged caches must be equal device tensors [pages, page_size, kv_heads, head_dim]")
    fp8 = k_cache.dtype in _FP8
    if not fp8 and k_cache.dtype is not _bf16:
        _fail(ERR_ARGUMENT, "Paged caches must be BF16 or E4M3FN")
    ks, vs = k_cache.stride(), v_cache.stride()
    if ks[3] != 1 or vs[3] != 1:
        _fail(ERR_ARGUMENT, "Paged caches need a contiguous last dimension")
    pages, page_size, kv_heads, head_dim = k_cache.shape
    if fp8:
        if not (_vector(k_scale, kv_heads, _f32, k_cache.device) and _vector(v_scale, kv_heads, _f32, k_cache.device)):
            _fail(ERR_ARGUMENT, "An 8-bit cache needs float32 k_scale and v_scale [kv_heads]")
    elif k_scale is not None or v_scale is not None:
        _fail(ERR_ARGUMENT, "A BF16 cache has no scales")
    return PagedCacheRecord(k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], pages, page_size,
                            kv_heads, head_dim, int(fp8), k_scale.data_ptr() if fp8 else None,
                            v_scale.data_ptr() if fp8 else None)


def _heads(t, shape, device):
    """Whether t is a BF16 tensor of that shape on the device, its last dimension contiguous."""
    return (isinstance(t, torch.Tensor) and t.dtype is _bf16 and t.shape == shape and t.device == device and t.stride(2) == 1)


def paged_append(k, v, slots, k_cache, v_cache, k_scale=None, v_scale=None):
    """k and v (BF16 [tokens, kv_heads, head_dim], last dimension contiguous)
    into their slots (int64 [tokens]) of the caches, in place
    (fp8lin_paged_append); rows whose slot is outside the cache are skipped."""
    rec = _cache(k_cache, v_cache, k_scale, v_scale)
    device = k_cache.device
    tokens = k.size(0) if isinstance(k, torch.Tensor) and k.dim() == 3 else -1
    shape = (tokens, rec.kv_heads, rec.head_dim)
    if not (_heads(k, shape, device) and _heads(v, shape, device)):
        _fail(ERR_ARGUMENT, "Paged append expects BF16 keys and values [tokens, kv_heads, head_dim]")
    if not _vector(slots, tokens, _i64, device):
        _fail(ERR_ARGUMENT, "Paged append expects int64 slots [tokens]")
    if tokens == 0:
        return
    ks, vs = k.stride(), v.stride()
    _call("fp8lin_paged_append", device, _byref(rec), k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], slots.data_ptr(),
          tokens)


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
    `out` if given, which overlaps no input and whose rows behind the last
    request stay as they were."""
    rec = _cache(k_cache, v_cache, k_scale, v_scale)
    device, kv_heads, dim = k_cache.device, rec.kv_heads, rec.head_dim
    if not (isinstance(q, torch.Tensor) and q.dim() == 3 and q.dtype is _bf16 and q.stride(2) == 1 and q.device == device and
            q.size(2) == dim):
        _fail(ERR_ARGUMENT, "Paged attention expects BF16 queries [tokens, heads, head_dim]")
    shape = q.shape
    tokens, heads, _ = shape
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        _fail(ERR_SHAPE, "Paged attention: heads must be a multiple of kv_heads")
    if not (isinstance(block_table, torch.Tensor) and block_table.dtype is _i32 and block_table.dim() == 2 and
            block_table.device == device and block_table.stride(1) == 1):
        _fail(ERR_ARGUMENT, "Invalid block table")
    requests, width = block_table.shape
    if not (_vector(offsets, requests + 1, _i32, device) and _vector(lengths, requests, _i32, device)):
        _fail(ERR_ARGUMENT, "Paged attention expects int32 offsets [requests + 1] and lengths [requests]")
    if gate is not None:
        if not _heads(gate, shape, device):
            _fail(ERR_ARGUMENT, "Paged attention expects a BF16 gate as the queries")
        gs, gate_at = gate.stride(), gate.data_ptr()
    else:
        gs, gate_at = (0, 0), None
    if out is None:
        out = q.new_empty(shape)
    elif not _heads(out, shape, device):
        _fail(ERR_ARGUMENT, "Paged attention expects a BF16 output as the queries")
    count = max(tokens - requests + 1, 1) if max_count is None else int(max_count)
    need = lib().fp8lin_paged_attention_workspace_bytes(heads, kv_heads, dim, count)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    qs, os = q.stride(), out.stride()
    _call("fp8lin_paged_attention", device, _byref(rec), q.data_ptr(), qs[0], qs[1], gate_at, gs[0], gs[1],
          block_table.data_ptr(), _row_stride(block_table, width), width, offsets.data_ptr(), lengths.data_ptr(), requests,
          tokens, heads, count, int(causal), dim ** -0.5 if scale is None else float(scale), out.data_ptr(), os[0], os[1],
          ws.data_ptr(), need)
    return out


def verify_drafts(logits, tokens, uniforms, offsets, draft_probs=None, temperature=None):
    """Verification of drafted tokens (fp8lin_verify_drafts).  Request b has
    rows offsets[b] .. offsets[b+1] (int32 [requests + 1]) of the target's
    logits (BF16 or FP32 [rows, vocab]), after its last token and after each of
    its drafts; tokens (int64 [rows]) were fed in, so its drafts are tokens but
    its first row's.  uniforms (float32 [rows], in [0, 1)): a row's number
    decides its draft, a request's last one draws its next token.
    draft_probs (float32 [drafts, vocab]): the draft model's distributions, the
    rows of all requests but each one's last, in order; None (or no row): drafts
    without probabilities.  temperature (float32 [requests], 0: the most likely
    token).  Returns (accepted int32 [requests], out int64 [rows]: per request
    the drafts kept, the next token, then -1)."""
    if not (_is_dev(logits) and logits.dim() == 2 and logits.dtype in (_bf16, _f32) and logits.stride(1) == 1 and
            logits.size(1) > 0):
        _fail(ERR_ARGUMENT, "Verification expects BF16 or FP32 logits [rows, vocab]")
    device, (rows, vocab) = logits.device, logits.shape
    if not (_vector(tokens, rows, _i64, device) and _vector(uniforms, rows, _f32, device) and
            _vector(offsets, None, _i32, device)):
        _fail(ERR_ARGUMENT, "Verification expects int64 tokens [rows], float32 uniforms [rows] and int32 offsets [requests + 1]")
    requests = offsets.size(0) - 1
    if requests < 1:
        _fail(ERR_SHAPE, "Verification expects offsets of at least one request")
    probs, prob_rows, prob_ld = None, 0, vocab
    if draft_probs is not None:
        if not (_is_dev(draft_probs) and draft_probs.dim() == 2 and draft_probs.device == device and
                draft_probs.dtype is _f32 and draft_probs.size(1) == vocab and draft_probs.stride(1) == 1):
            _fail(ERR_ARGUMENT, "Verification expects float32 draft probabilities [drafts, vocab]")
        # without rows there is no draft to test, and no pointer
        if draft_probs.size(0):
            probs, prob_rows, prob_ld = draft_probs.data_ptr(), draft_probs.size(0), _row_stride(draft_probs, vocab)
    if temperature is not None and not _vector(temperature, requests, _f32, device):
        _fail(ERR_ARGUMENT, "Verification expects float32 temperatures [requests]")
    accepted, out = offsets.new_empty(requests), tokens.new_empty(rows)
    need = lib().fp8lin_verify_drafts_workspace_bytes(requests, rows, vocab)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    _call("fp8lin_verify_drafts", device, logits.data_ptr(), int(logits.dtype is _f32), _row_stride(logits, vocab), probs,
          prob_ld, prob_rows, tokens.data_ptr(), uniforms.data_ptr(), offsets.data_ptr(),
          temperature.data_ptr() if temperature is not None else None, requests, rows, vocab, accepted.data_ptr(),
          out.data_ptr(), ws.data_ptr(), need)
    return accepted, out
