"""Attention and cache operators over torch tensors that the caller owns (the operators of
include/yue2_cuda.h): whole packed prompts, drafted tokens over paged K/V, the pass that
norms, rotates and appends, and the page moves.

Every call runs on the current stream of its tensors' device, allocates through torch only
(outputs and workspaces) and can be captured into a CUDA graph: lengths, page tables and
lists are read on the device. Sizes, types and strides are checked at once (Yue2Error); what
only the device sees (page indexes, lengths, positions) is checked there, an entry out of
range is skipped, and `check_status` reports it.

A step over a batch of requests: `qk_rope_append` writes the new rows' K and V into the pages,
`attention_packed` attends over whole prompts, `attention_tree` checks drafted tokens against
the pages, `kv_gather` keeps the accepted ones, and `kv_copy` forks the last page of a prompt
that several takes share.
"""
import ctypes
import math
import threading

import torch

from . import _lib

PAGE = 64  # positions of a page

_DTYPES = {torch.bfloat16: 0, torch.float16: 2}
_BITS = ((1, "a page index or slot outside the pool"), (2, "a length, offset or position out of range"),
         (4, "a bounded device wait gave up"))

_status = {}  # device index -> int32 status word
_lock = threading.Lock()


def _invalid(message):
    return _lib.Yue2Error(-1, message)


def _status_of(device):
    s = _status.get(device.index)
    if s is None:
        with _lock, torch.cuda.device(device):
            if torch.cuda.is_current_stream_capturing():
                raise _invalid("call an operator (or check_status) once on this device before any capture")
            s = _status.get(device.index)
            if s is None:
                s = torch.zeros(1, dtype=torch.int32, device=device)
                torch.cuda.synchronize(device)  # cleared before any stream's kernels see it
                _status[device.index] = s
    return s


def check_status(device=None):
    """Waits for the device, then raises Yue2Error for what the operators' kernels found since
    the last check and clears it."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    s = _status_of(device)
    torch.cuda.synchronize(device)
    bits = int(s.item())
    if bits:
        s.zero_()
        torch.cuda.synchronize(device)
        text = "; ".join(t for b, t in _BITS if bits & b)
        raise _lib.Yue2Error(-7 if bits & 4 else -1, text)


class KvPool:
    """Paged K/V over `data`, a contiguous [pages, layers, 2, kv heads, 64, dim] bf16 or f16
    tensor: the layout of the engine's own caches. Position p of a sequence lives in page
    table[p // 64], place p % 64; its slot is 64 * page + place."""

    def __init__(self, data):
        if data.dim() != 6 or data.shape[2] != 2 or data.shape[4] != PAGE or not data.is_contiguous():
            raise _invalid("a KV pool is a contiguous [pages, layers, 2, kv heads, 64, dim] tensor")
        if data.dtype not in _DTYPES or not data.is_cuda:
            raise _invalid("a KV pool holds bf16 or f16 values on a GPU")
        self.data = data
        self.device, self.dtype = data.device, data.dtype
        self.pages, self.layers, _, self.kv_heads, _, self.dim = data.shape
        self._c = _lib.KvPool(data.data_ptr(), self.pages, self.layers, self.kv_heads, self.dim, _DTYPES[data.dtype])
        self._ref = ctypes.addressof(self._c)

    @classmethod
    def zeros(cls, pages, layers, kv_heads, dim, dtype=torch.bfloat16, device="cuda"):
        return cls(torch.zeros((pages, layers, 2, kv_heads, PAGE, dim), dtype=dtype, device=device))


def _int(t, dtype, device, what, shape=None):
    """The address of a contiguous device tensor of integers (or 32-bit floats)."""
    if t.dtype is not dtype or t.device != device or not t.is_contiguous() or (shape is not None and t.shape != shape):
        raise _invalid(f"{what} must be a contiguous {dtype} tensor on {device}"
                       + (f" of shape {tuple(shape)}" if shape is not None else ""))
    return t.data_ptr()


def _rows(t, device, dtype, what):
    """The address and row stride of a [rows, heads, dim] tensor with adjacent heads."""
    if t.dim() != 3 or t.dtype is not dtype or t.device != device:
        raise _invalid(f"{what} must be a [rows, heads, dim] tensor of {dtype} on {device}")
    rows, heads, dim = t.shape
    s = t.stride()
    if t.numel() and (s[2] != 1 or (heads > 1 and s[1] != dim)):
        raise _invalid(f"{what}: the heads of a row must be adjacent")
    return t.data_ptr(), s[0] if rows > 1 and t.numel() else heads * dim


def _call(device, fn, *args):
    """fn(*args, status, stream) on the device's current stream."""
    status = _status_of(device).data_ptr()
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            rc = fn(*args, status, torch.cuda.current_stream(device).cuda_stream)
    else:
        rc = fn(*args, status, torch.cuda.current_stream(device).cuda_stream)
    if rc:
        _lib.check(rc)


def qk_rope_append(qkv, q_norm, k_norm, eps, cos, sin, positions, pool, layer, slots, q_out=None, k_out=None):
    """Per-head RMSNorm of q and k, rotation, and K/V into the pages, in one pass.

    qkv [rows, heads + 2 kv, dim] (rows may be strided); gains [dim] f32 or both None; cos and
    sin [table rows, dim/2] f32, looked up at positions [rows] int32 (pairs (i, i + dim/2));
    slots [rows] int64, 64 * page + place, negative for a row whose K/V is not kept. Returns
    q [rows, heads, dim] (q_out when given); k_out [rows, kv, dim], when given, gets the rotated
    K as well. q_out and k_out may be the q and k parts of qkv."""
    dev = pool.device
    src, stride = _rows(qkv, dev, pool.dtype, "qkv")
    rows, width, dim = qkv.shape
    heads = width - 2 * pool.kv_heads
    if heads < 1 or dim != pool.dim:
        raise _invalid("qkv must be [rows, heads + 2 kv heads, dim] of the pool's kv heads and dim")
    if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != dim // 2:
        raise _invalid("cos and sin must be [table rows, dim / 2]")
    if (q_norm is None) != (k_norm is None):
        raise _invalid("q_norm and k_norm go together")
    if q_out is None:
        q_out = torch.empty((rows, heads, dim), dtype=qkv.dtype, device=dev)
    elif q_out.shape != (rows, heads, dim):
        raise _invalid("q_out must be [rows, heads, dim]")
    qp, qs = _rows(q_out, dev, pool.dtype, "q_out")
    kp, ks = 0, 0
    if k_out is not None:
        if k_out.shape != (rows, pool.kv_heads, dim):
            raise _invalid("k_out must be [rows, kv heads, dim]")
        kp, ks = _rows(k_out, dev, pool.dtype, "k_out")
    f32 = torch.float32
    _call(dev, _lib.lib().yue2_qk_rope_append, src, rows, heads, stride,
          0 if q_norm is None else _int(q_norm, f32, dev, "q_norm", (dim,)),
          0 if k_norm is None else _int(k_norm, f32, dev, "k_norm", (dim,)), eps, _int(cos, f32, dev, "cos"),
          _int(sin, f32, dev, "sin"), cos.shape[0], _int(positions, torch.int32, dev, "positions", (rows,)), pool._ref, layer,
          _int(slots, torch.int64, dev, "slots", (rows,)), qp, qs, kp if rows else 0, ks)
    return q_out


def attention_packed(q, k, v, cu, causal=True, scale=None, out=None):
    """Attention over whole packed sequences: rows cu[s] .. cu[s + 1] - 1 of q [tokens, heads,
    dim], k and v [tokens, kv, dim] are sequence s (cu int32 [seqs + 1]; at most 1,024
    sequences, empty ones allowed, and 262,144 tokens). A row sees its sequence up to itself,
    or all of it with causal=False. scale: 1 / sqrt(dim) by default. Rows outside
    [cu[0], cu[-1]) of `out` are left as they were (undefined when `out` is None). bf16 or
    f16, dim 64 or 128; strided rows are fine."""
    dev, dtype = q.device, q.dtype
    if dtype not in _DTYPES or not q.is_cuda:
        raise _invalid("attention takes bf16 or f16 tensors on a GPU")
    qp, qs = _rows(q, dev, dtype, "q")
    kp, ks = _rows(k, dev, dtype, "k")
    vp, vs = _rows(v, dev, dtype, "v")
    tokens, heads, dim = q.shape
    kv = k.shape[1]
    if k.shape != v.shape or k.shape[0] != tokens or k.shape[2] != dim:
        raise _invalid("k and v must be [tokens, kv heads, dim] of q's tokens and dim")
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=dtype, device=dev)
    elif out.shape != q.shape:
        raise _invalid("out must have q's shape")
    op, os_ = _rows(out, dev, dtype, "out")
    if cu.dim() != 1 or cu.shape[0] < 1:
        raise _invalid("cu must be [seqs + 1]")
    _call(dev, _lib.lib().yue2_attention_packed, qp, kp, vp, op, _int(cu, torch.int32, dev, "cu"), cu.shape[0] - 1, tokens,
          heads, kv, dim, qs, ks, vs, os_, _DTYPES[dtype], 1 if causal else 0, 1 / math.sqrt(dim) if scale is None else scale)
    return out


def attention_tree(q, pool, layer, table, context, cu, mask=None, scale=None, out=None):
    """Attention of drafted tokens over the pages. Sequence s holds context[s] positions (int32)
    in the pages table[s] (int32 [seqs, pages]) and after them its drafted ones, at most 64,
    whose K/V are in the pages too; rows cu[s] .. cu[s + 1] - 1 of q [rows, heads, dim] are
    theirs. Row i sees the context and the drafted positions whose bit is set in mask[row]
    (int64: a node's ancestors and itself); mask None: all up to itself, so that one row per
    sequence is an ordinary decode step. A row that sees nothing gets zeros; rows outside
    [cu[0], cu[-1]) of `out` are left as they were (undefined when `out` is None)."""
    dev = pool.device
    qp, qs = _rows(q, dev, pool.dtype, "q")
    rows, heads, dim = q.shape
    if dim != pool.dim:
        raise _invalid("q must have the pool's dim")
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=q.dtype, device=dev)
    elif out.shape != q.shape:
        raise _invalid("out must have q's shape")
    op, os_ = _rows(out, dev, pool.dtype, "out")
    if table.dim() != 2:
        raise _invalid("table must be [seqs, pages]")
    seqs, pages = table.shape
    L = _lib.lib()
    need = L.yue2_attention_tree_workspace(rows, heads, seqs, pages, pool._ref)
    work = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(dev, L.yue2_attention_tree, qp, rows, heads, qs, pool._ref, layer, _int(table, torch.int32, dev, "table"), seqs, pages,
          _int(context, torch.int32, dev, "context", (seqs,)), _int(cu, torch.int32, dev, "cu", (seqs + 1,)),
          0 if mask is None else _int(mask, torch.int64, dev, "mask", (rows,)), 1 / math.sqrt(dim) if scale is None else scale,
          op, os_, work.data_ptr() if need else 0, need)
    return out


def kv_copy(pool, src, dst, count=None):
    """Positions [0, count[i]) (all 64 when count is None) of page src[i] to page dst[i], in
    every layer; int32 [n] each. The dst pages are distinct and none of them is a src page."""
    n = src.shape[0]
    _call(pool.device, _lib.lib().yue2_kv_copy, pool._ref, _int(src, torch.int32, pool.device, "src", (n,)),
          _int(dst, torch.int32, pool.device, "dst", (n,)),
          0 if count is None else _int(count, torch.int32, pool.device, "count", (n,)), n)


def kv_gather(pool, src_table, dst_table, begin, cu, keep):
    """Position keep[cu[s] + i] of sequence s to its position begin[s] + i, in every layer.

    dst_table None: in place; keep strictly increasing and not before begin[s] (accepting a
    path of a drafted tree, dropping positions), and the pages written are the sequence's
    own. Otherwise into the pages of dst_table, none of which the call reads; keep in any
    order. Tables int32 [seqs, pages], begin int32 [seqs], cu int32 [seqs + 1], keep int32."""
    dev, i32 = pool.device, torch.int32
    if src_table.dim() != 2 or (dst_table is not None and (dst_table.dim() != 2 or dst_table.shape[0] != src_table.shape[0])):
        raise _invalid("page tables must be [seqs, pages] of the same sequences")
    seqs = src_table.shape[0]
    if keep.dim() != 1:
        raise _invalid("keep must be one list")
    _call(dev, _lib.lib().yue2_kv_gather, pool._ref, _int(src_table, i32, dev, "src_table"), src_table.shape[1],
          0 if dst_table is None else _int(dst_table, i32, dev, "dst_table"), 0 if dst_table is None else dst_table.shape[1],
          _int(begin, i32, dev, "begin", (seqs,)), _int(cu, i32, dev, "cu", (seqs + 1,)), _int(keep, i32, dev, "keep"), seqs,
          keep.shape[0])
