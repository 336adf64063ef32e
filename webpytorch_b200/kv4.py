"""Serving several requests from a paged key/value cache held in 4 bits: block tables and slot maps
from request lengths (`plan`), the norms and rotation of queries and keys with the write into the
cache (`qk_norm_rope`), and the attention that reads it (`attention`).

The reference keeps one request's keys and values as fp32 arrays (package `webtorch`,
lm_engine.py:89-101, llm.py:1573-1616); the norm and rotation are its `_rms`, `_rope` and `_rot`
(lm_engine.py:62-74). The cache here is one tensor for each layer, shared by all requests in pages:
4.5 bits a value at group 64 instead of 32. Block layout and rounding are in include/qlinear.h.

A step of a batch:

    p = kv4.plan(lens, new, table, free, n_free, cache.page, max_tokens)     # once a step
    q, _ = kv4.qk_norm_rope(qkv, NH, NKV, HD, p.positions, cos, sin, cache=cache, slots=p.slots)
    o = kv4.attention(q, cache, table, p.seq_lens, p.cu_new)                 # each layer

Every call is asynchronous on the current stream (or `stream`), without a host read of any length,
so a step can be captured in a CUDA graph. All tensors of a call are on the current GPU (that of `stream`, where it
is given); others are refused.
"""
from collections import namedtuple

import torch

from . import _ffi
from .qlinear import _device

__all__ = ["KV4Cache", "Plan", "plan", "qk_norm_rope", "attention"]

_INT_MAX = 2 ** 31 - 1

Plan = namedtuple("Plan", "seq_lens cu_new slots positions requests n_free")


def _need(t, name, dtype, dim, dev):
    """t is a tensor of this type and number of dimensions on GPU `dev` (the current one, which the kernels are
    launched on), its last dimension contiguous."""
    if type(t) is torch.Tensor and t.dtype is dtype and t.get_device() == dev and t.dim() == dim and (
            t.is_contiguous() or t.stride(-1) == 1):
        return                                     # the calls take a few microseconds: keep this short
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != dim:
        raise TypeError("%s must be a %d-D %s tensor, got %s" % (
            name, dim, dtype, "%s %s" % (t.dtype, tuple(t.shape)) if isinstance(t, torch.Tensor) else type(t).__name__))
    _on(t, name, dev)
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError("%s must be contiguous along its last dimension" % name)


def _out(t, dtype, shape, dev):
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError("out must be a contiguous %s tensor %s" % (dtype, shape))
    _on(t, "out", dev)


def _on(t, name, dev):
    if t.get_device() != dev:
        raise ValueError("%s must be on the current GPU, cuda:%d, not on %s" % (name, dev, t.device))


class KV4Cache:
    """One layer's keys and values in 4 bits: `num_pages` pages of `page` positions for `NKV` heads of
    `HD` elements, quantised in groups of `group` elements. `data` wraps memory that the caller owns
    (uint8 [num_pages, NKV, page / 16, block bytes]); otherwise it is allocated, uninitialised."""

    def __init__(self, num_pages, NKV, HD, page=64, group=64, device=None, data=None):
        bb = int(_ffi.fn("ql_kv4_block_bytes")(int(HD), int(group)))
        if not bb or page < 16 or page > 4096 or page & (page - 1) or NKV <= 0 or num_pages <= 0:
            raise ValueError("unsupported cache: HD %s (64, 128 or 256), group %s (32, 64 or 128, at most HD), page %s "
                             "(a power of two, 16 to 4096), %s heads, %s pages" % (HD, group, page, NKV, num_pages))
        shape = (num_pages, NKV, page // 16, bb)
        if data is None:
            data = torch.empty(shape, dtype=torch.uint8, device=_device(device))
        elif not data.is_cuda or data.dtype != torch.uint8 or tuple(data.shape) != shape or not data.is_contiguous():
            raise ValueError("data must be a contiguous uint8 GPU tensor %s" % (shape,))
        self.data = data
        self.num_pages, self.NKV, self.HD, self.page, self.group = num_pages, NKV, HD, page, group
        self.device = data.device

    def nbytes(self):
        return self.data.numel()

    def read(self, slots, stream=None):
        """(k, v) fp16 [T, NKV, HD]: the values that slots int64 [T] stand for; zeros for -1."""
        if stream is not None:
            with torch.cuda.stream(stream):
                return self.read(slots)
        dev = torch.cuda.current_device()
        _on(self.data, "the cache", dev)
        _need(slots, "slots", torch.int64, 1, dev)
        T = slots.shape[0]
        k, v = slots.new_empty((2, T, self.NKV, self.HD), dtype=torch.float16).unbind(0)
        _ffi.call("ql_kv4_read", self.data.data_ptr(), self.num_pages, self.NKV, self.HD, self.page, self.group,
                  slots.data_ptr(), T, k.data_ptr(), v.data_ptr(), _ffi.stream_ptr(None, self.device))
        return k, v


_workspaces = {}     # (GPU, HD, stream): the workspace of the calls on that stream
_captured = {}       # the same: (capture, workspace) of the calls that a graph takes up there
_COUNTER_BYTES = 2048                             # QL_KV4_COUNTER_BYTES


def _attention_workspace(cache, NH):
    """The attention's workspace on the current stream, made once and shared by the layers' caches: its counters
    are zero between calls, and calls that share one may not overlap. A graph is replayed on any stream, beside
    others, so the calls that it captures have a workspace of their own in the graph's memory, whose counters the
    graph zeroes before the first of them."""
    stream = _ffi.stream_ptr(None, cache.device)
    key = (cache.device.index, cache.HD, stream)
    if torch.cuda.is_current_stream_capturing():
        capture = _ffi.fn("ql_stream_capture_id")(stream)
        held = _captured.get(key)
        if held is None or held[0] != capture:
            held = _captured[key] = (capture, _new_workspace(cache, NH))
        return held[1]
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = _new_workspace(cache, NH)
    return ws


def _new_workspace(cache, NH):
    n = int(_ffi.fn("ql_kv4_attention_workspace")(NH, cache.NKV, cache.HD))
    ws = torch.empty(n, dtype=torch.uint8, device=cache.device)
    ws[:_COUNTER_BYTES].zero_()
    return ws


def plan(prev_lens, new_lens, block_table, free_pages, n_free, page, max_tokens, stream=None):
    """Block tables and slot maps of a step from request lengths, on the GPU (ql_kv_plan).

    prev_lens, new_lens int32 [n]: tokens in the cache, tokens to append (negative: the request ends
    and its pages are free again). block_table int32 [n, width] and free_pages int32 [capacity] (a
    stack of height n_free, int32 [1]) are updated in place; lengths and the stack's height come back
    as new tensors. Requests are served first come first served, as far as max_tokens and the free
    pages go; one that is not keeps its length. Returns Plan(seq_lens, cu_new [n + 1], slots, positions,
    requests [max_tokens], n_free); entries past cu_new[n] are -1."""
    if stream is not None:
        with torch.cuda.stream(stream):              # what is allocated here belongs to it too
            return plan(prev_lens, new_lens, block_table, free_pages, n_free, page, max_tokens)
    dev = torch.cuda.current_device()
    _need(prev_lens, "prev_lens", torch.int32, 1, dev)
    _need(new_lens, "new_lens", torch.int32, 1, dev)
    _need(block_table, "block_table", torch.int32, 2, dev)
    _need(free_pages, "free_pages", torch.int32, 1, dev)
    _need(n_free, "n_free", torch.int32, 1, dev)
    n, width = block_table.shape
    if new_lens.shape[0] != n or prev_lens.shape[0] != n:
        raise ValueError("prev_lens, new_lens and block_table must have a row for each request: %d, %d, %d"
                         % (prev_lens.shape[0], new_lens.shape[0], n))
    max_tokens = int(max_tokens)
    ws_ints = int(_ffi.fn("ql_kv_plan_workspace")(n)) // 4
    lens, cu, pos, req, left, ws = torch.unsafe_split_with_sizes(
        prev_lens.new_empty(2 * n + 2 + 2 * max_tokens + ws_ints), (n, n + 1, max_tokens, max_tokens, 1, ws_ints))
    slots = prev_lens.new_empty(max_tokens, dtype=torch.int64)
    _ffi.call("ql_kv_plan", prev_lens.data_ptr(), new_lens.data_ptr(), n, block_table.data_ptr(),
              block_table.stride(0) if n > 1 else width, width, free_pages.data_ptr(), free_pages.shape[0],
              n_free.data_ptr(), page, max_tokens, lens.data_ptr(), cu.data_ptr(), slots.data_ptr(), pos.data_ptr(),
              req.data_ptr(), left.data_ptr(), ws.data_ptr() if ws_ints else None, 4 * ws_ints,
              _ffi.stream_ptr(None, prev_lens.device))
    return Plan(lens, cu, slots, pos, req, left)


def qk_norm_rope(qkv, NH, NKV, HD, positions, cos, sin, *, q_weight=None, k_weight=None, eps=1e-6, cache=None,
                 slots=None, out=None, stream=None):
    """RMS norms of the query and key heads (where a weight fp32 [HD] is given) and rotate-half position
    embedding over rows q | k | v of `qkv` [T, (NH + 2 NKV) HD] (ql_qk_norm_rope). cos, sin fp32
    [lmax, rot / 2]. With a cache, keys and values are quantised into its slots int64 [T] and (q, None)
    comes back, without one (q, k); q [T, NH, HD], k [T, NKV, HD] in qkv's dtype. A negative position is
    padding."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return qk_norm_rope(qkv, NH, NKV, HD, positions, cos, sin, q_weight=q_weight, k_weight=k_weight, eps=eps,
                                cache=cache, slots=slots, out=out)
    dev = torch.cuda.current_device()
    _need(qkv, "qkv", qkv.dtype, 2, dev)
    T, width = qkv.shape
    if width != (NH + 2 * NKV) * HD:
        raise ValueError("qkv must be [T, %d], got %s" % ((NH + 2 * NKV) * HD, tuple(qkv.shape)))
    _need(positions, "positions", torch.int32, 1, dev)
    _need(cos, "cos", torch.float32, 2, dev)
    _need(sin, "sin", torch.float32, 2, dev)
    lmax, half = cos.shape
    if positions.shape[0] != T or sin.shape != cos.shape or not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError("positions must be [T], cos and sin contiguous [lmax, rot / 2]")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _need(w, name, torch.float32, 1, dev)
            if w.shape[0] != HD:
                raise ValueError("%s must be [%d]" % (name, HD))
    if out is None:
        out = qkv.new_empty((T, NH, HD))
    else:
        _out(out, qkv.dtype, (T, NH, HD), dev)
    k = None
    if cache is None:
        k = qkv.new_empty((T, NKV, HD))
        where = (k.data_ptr(), None, 0, 0, 0, None)
    else:
        _need(slots, "slots", torch.int64, 1, dev)
        _on(cache.data, "the cache", dev)
        if cache.NKV != NKV or cache.HD != HD or slots.shape[0] != T:
            raise ValueError("the cache holds %d heads of %d, and slots must be [T]" % (cache.NKV, cache.HD))
        where = (None, cache.data.data_ptr(), cache.num_pages, cache.page, cache.group, slots.data_ptr())
    _ffi.call("ql_qk_norm_rope", qkv.data_ptr(), _ffi.dtype_code(qkv.dtype), qkv.stride(0) if T > 1 else width, T, NH, NKV,
              HD, positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), lmax, 2 * half, _ffi.ptr(q_weight),
              _ffi.ptr(k_weight), eps, out.data_ptr(), *where, _ffi.stream_ptr(None, qkv.device))
    return out, k


def attention(q, cache, block_table, seq_lens, cu_q=None, *, scale=None, window=0, out=None, workspace=None,
              stream=None):
    """softmax(q K^T scale) V over the cache for each request, causal from its end (ql_kv4_attention).

    q [T, NH, HD] fp32, fp16 or bf16 (heads contiguous; tokens may be strided): rows cu_q[b] ..
    cu_q[b + 1] - 1 are request b's last tokens (cu_q int32 [B + 1]; None: one token each). block_table
    int32 [B, width], seq_lens int32 [B] with those tokens counted. window: positions that a query sees
    (0: all). workspace: uint8 of ql_kv4_attention_workspace bytes, zeroed once and not shared by calls that
    overlap (None: one for each stream, and one for each graph that is captured there). Rows that see nothing, and rows past cu_q[B], are zero. Returns
    [T, NH, HD] in q's dtype."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return attention(q, cache, block_table, seq_lens, cu_q, scale=scale, window=window, out=out, workspace=workspace)
    dev = torch.cuda.current_device()
    _need(q, "q", q.dtype, 3, dev)
    _on(cache.data, "the cache", dev)
    T, NH, HD = q.shape
    ldq = NH * HD
    dense = q.is_contiguous()
    if not dense:
        if q.stride(2) != 1 or (NH > 1 and q.stride(1) != HD):
            raise ValueError("q must be [T, NH, HD] with contiguous heads, got %s, strides %s" % (tuple(q.shape), q.stride()))
        ldq = q.stride(0)
    _need(block_table, "block_table", torch.int32, 2, dev)
    _need(seq_lens, "seq_lens", torch.int32, 1, dev)
    B, width = block_table.shape
    if HD != cache.HD or NH % cache.NKV or seq_lens.shape[0] != B:
        raise ValueError("q has %d heads of %d, the cache %d of %d; block_table has %d rows for %d requests"
                         % (NH, HD, cache.NKV, cache.HD, B, seq_lens.shape[0]))
    if cu_q is None:
        if T < B:
            raise ValueError("%d queries for %d requests" % (T, B))
    else:
        _need(cu_q, "cu_q", torch.int32, 1, dev)
        if cu_q.shape[0] != B + 1:
            raise ValueError("cu_q must be [%d]" % (B + 1))
    if q.data_ptr() % 16 or ldq * q.element_size() % 16:      # the kernel reads 16 bytes at a time
        q, ldq, dense = torch.empty((T, NH, HD), dtype=q.dtype, device=q.device).copy_(q), NH * HD, True
    if out is None:
        out = torch.empty_like(q) if dense else q.new_empty((T, NH, HD))
    else:
        _out(out, q.dtype, (T, NH, HD), dev)
    if workspace is None:
        ws = _attention_workspace(cache, NH)
    else:
        ws = workspace
        _on(ws, "workspace", dev)
        if not ws.is_contiguous():
            raise ValueError("workspace must be contiguous")
    _ffi.call("ql_kv4_attention", q.data_ptr(), _ffi.dtype_code(q.dtype), ldq, T, NH, cache.NKV, HD, cache.data.data_ptr(),
              cache.num_pages, cache.page, cache.group, block_table.data_ptr(), block_table.stride(0) if B > 1 else width,
              width, seq_lens.data_ptr(), _ffi.ptr(cu_q), B, HD ** -0.5 if scale is None else scale, min(window, _INT_MAX),
              out.data_ptr(), ws.data_ptr(), ws.nbytes, _ffi.stream_ptr(None, q.device))
    return out
