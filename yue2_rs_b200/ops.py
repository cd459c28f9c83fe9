"""Attention and cache operators over torch tensors that the caller owns (the operators of
include/yue2_cuda.h): whole packed prompts, drafted tokens over paged K/V, the pass that
norms, rotates and appends, and the page moves.

Every call runs on the current stream of its tensors' device, allocates through torch only
(outputs and workspaces) and can be captured into a CUDA graph: lengths, page tables and
lists are read on the device. Sizes, types and strides are checked at once (Yue2Error); what
only the device sees (page indexes, lengths, positions) is checked there, an entry out of
range is skipped, and `check_status` reports it. The operators serve: they have no gradients,
and refuse rows, gains, tables and pools that ask for one.

A step over a batch of requests: `qk_rope_append` writes the new rows' K and V into the pages,
`attention_packed` attends over whole prompts, `attention_tree` checks drafted tokens against
the pages, `kv_gather` keeps the accepted ones, and `kv_copy` forks the last page of a prompt
that several takes share.
"""
import ctypes
import threading

import torch
from torch.autograd import forward_ad as _forward  # its _current_level: -1 outside of any dual level

from . import _lib

PAGE = 64  # positions of a page

_DTYPES = {torch.bfloat16: 0, torch.float16: 2}
_BITS = ((1, "a page index or slot outside the pool"), (2, "a length, offset or position out of range"),
         (4, "a bounded device wait gave up"))

_status = {}  # device index -> (address, int32 status word)
_lock = threading.Lock()


def _invalid(message):
    return _lib.Yue2Error(-1, message)


def _status_of(index):
    """The address of the device's status word."""
    s = _status.get(index)
    if s is None:
        device = torch.device("cuda", index)
        with _lock, torch.cuda.device(device):
            if torch.cuda.is_current_stream_capturing():
                raise _invalid("call an operator (or check_status) once on this device before any capture")
            s = _status.get(index)
            if s is None:
                with torch.inference_mode(False):  # check_status clears it in either mode
                    word = torch.zeros(1, dtype=torch.int32, device=device)
                torch.cuda.synchronize(device)  # cleared before any stream's kernels see it
                s = _status[index] = (word.data_ptr(), word)
    return s[0]


def check_status(device=None):
    """Waits for the device, then raises Yue2Error for what the operators' kernels found since
    the last check and clears it. Not for use inside a capture, which no wait survives."""
    if torch.cuda.is_current_stream_capturing():
        raise _invalid("check_status waits for the device: call it outside of a capture")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    _status_of(device.index)
    s = _status[device.index][1]
    torch.cuda.synchronize(device)
    bits = int(s.item())
    if bits:
        s.bitwise_and_(~bits)  # not what other threads' calls have found since
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
        self.device, self.dtype, self.index = data.device, data.dtype, data.get_device()
        self.pages, self.layers, _, self.kv_heads, _, self.dim = data.shape
        self._c = _lib.KvPool(data.data_ptr(), self.pages, self.layers, self.kv_heads, self.dim, _DTYPES[data.dtype])
        self._ref = ctypes.addressof(self._c)
        self._sizes = {}  # bytes of the tree attention's workspace by (rows, heads, seqs, pages)

    def _workspace(self, *shape):
        need = self._sizes.get(shape)
        if need is None:
            with torch.cuda.device(self.index):
                need = _lib.lib().yue2_attention_tree_workspace(*shape, self._ref)
            if len(self._sizes) < 4096:
                self._sizes[shape] = need
        return need

    @classmethod
    def zeros(cls, pages, layers, kv_heads, dim, dtype=torch.bfloat16, device="cuda"):
        return cls(torch.zeros((pages, layers, 2, kv_heads, PAGE, dim), dtype=dtype, device=device))


# Calls of a few microseconds are the smallest cases' whole cost, so the checks below read each
# attribute once and the stream's handle without building a Stream object.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


# What the kernels write through an address counts as modified in place, so that a backward pass which
# saved it notices.
_written = torch.autograd.graph.increment_version


def _flat(t, dtype, index, what, count):
    """The address of a contiguous device tensor of `count` values."""
    if t.dtype is dtype and t.get_device() == index and t.numel() == count and t.is_contiguous():
        return t.data_ptr()
    raise _invalid(f"{what} must be a contiguous tensor of {count} {dtype} values on cuda:{index}")


def _table(t, dtype, index, what):
    """The address, rows and columns of a contiguous two-dimensional device tensor."""
    if t.dtype is dtype and t.get_device() == index and t.dim() == 2 and t.is_contiguous():
        return t.data_ptr(), *t.shape
    raise _invalid(f"{what} must be a contiguous two-dimensional tensor of {dtype} on cuda:{index}")


def _no_gradient(what):
    if torch.is_grad_enabled():
        raise _invalid(f"{what} asks for a gradient, which these operators do not have: call them under torch.no_grad()")


def _no_tangents(*tensors):
    for t in tensors:
        if t is not None and _forward.unpack_dual(t).tangent is not None:
            raise _invalid("a tensor carries a tangent, and these operators have no forward-mode gradient")


def _rows(t, index, dtype, what, shape=None):
    """The address, row stride and shape of a [rows, heads, dim] tensor with adjacent heads."""
    if t.dtype is not dtype or t.get_device() != index or t.dim() != 3 or (shape is not None and t.shape != shape):
        raise _invalid(f"{what} must be a [rows, heads, dim] tensor of {dtype} on cuda:{index}"
                       + (f" of shape {tuple(shape)}" if shape is not None else ""))
    if t.requires_grad:
        _no_gradient(what)
    rows, heads, dim = t.shape
    step, head, one = t.stride()
    if (one != 1 or (heads > 1 and head != dim)) and rows and heads and dim:
        raise _invalid(f"{what}: the heads of a row must be adjacent")
    return t.data_ptr(), step if rows > 1 else heads * dim, rows, heads, dim


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(index, name, *args):
    """The library's `name`(*args, status, stream) on the device's current stream."""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.lib(), name)
    s = _status.get(index)
    status = _status_of(index) if s is None else s[0]
    if _current_device() != index:
        with torch.cuda.device(index):
            rc = fn(*args, status, _raw_stream(index))
    else:
        rc = fn(*args, status, _raw_stream(index))
    if rc:
        _lib.check(rc)


_fns = {}


def qk_rope_append(qkv, q_norm, k_norm, eps, cos, sin, positions, pool, layer, slots, q_out=None, k_out=None):
    """Per-head RMSNorm of q and k, rotation, and K/V into the pages, in one pass.

    qkv [rows, heads + 2 kv, dim] (rows may be strided); gains [dim] f32 or both None; cos and
    sin [table rows, dim/2] f32, looked up at positions [rows] int32 (pairs (i, i + dim/2));
    slots [rows] int64, 64 * page + place, negative for a row whose K/V is not kept. Returns
    q [rows, heads, dim] (q_out when given); k_out [rows, kv, dim], when given, gets the rotated
    K as well. q_out and k_out may be the q and k parts of qkv."""
    dev, dtype, kv, f32 = pool.index, pool.dtype, pool.kv_heads, torch.float32
    src, stride, rows, width, dim = _rows(qkv, dev, dtype, "qkv")
    if pool.data.requires_grad:
        _no_gradient("the pool")
    heads = width - 2 * kv
    if heads < 1 or dim != pool.dim:
        raise _invalid("qkv must be [rows, heads + 2 kv heads, dim] of the pool's kv heads and dim")
    cp, steps, half = _table(cos, f32, dev, "cos")
    if half != dim // 2:
        raise _invalid("cos and sin must be [table rows, dim / 2]")
    if (q_norm is None) != (k_norm is None):
        raise _invalid("q_norm and k_norm go together")
    if q_norm is not None and (q_norm.requires_grad or k_norm.requires_grad):
        _no_gradient("the norm")
    if cos.requires_grad or sin.requires_grad:
        _no_gradient("the table of cos or sin")
    if _forward._current_level >= 0:
        _no_tangents(qkv, q_norm, k_norm, cos, sin, pool.data, q_out, k_out)
    if q_out is None:
        q_out = qkv.new_empty((rows, heads, dim))
        qp, qs = q_out.data_ptr(), heads * dim
    else:
        qp, qs = _rows(q_out, dev, dtype, "q_out", (rows, heads, dim))[:2]
    kp, ks = (0, 0) if k_out is None else _rows(k_out, dev, dtype, "k_out", (rows, kv, dim))[:2]
    _call(dev, "yue2_qk_rope_append", src, rows, heads, stride,
          0 if q_norm is None else _flat(q_norm, f32, dev, "q_norm", dim),
          0 if k_norm is None else _flat(k_norm, f32, dev, "k_norm", dim), eps, cp, _flat(sin, f32, dev, "sin", steps * half), steps,
          _flat(positions, torch.int32, dev, "positions", rows), pool._ref, layer, _flat(slots, torch.int64, dev, "slots", rows),
          qp, qs, kp if rows else 0, ks)
    _written((q_out, pool.data) if k_out is None else (q_out, pool.data, k_out))
    return q_out


def attention_packed(q, k, v, cu, causal=True, scale=None, out=None):
    """Attention over whole packed sequences: rows cu[s] .. cu[s + 1] - 1 of q [tokens, heads,
    dim], k and v [tokens, kv, dim] are sequence s (cu int32 [seqs + 1]; at most 1,024
    sequences, empty ones allowed, and 262,144 tokens). A row sees its sequence up to itself,
    or all of it with causal=False. scale: 1 / sqrt(dim) by default. A key whose score is -inf
    has no weight, and a row of such keys alone is zero. Rows outside [cu[0], cu[-1]) of `out`
    are left as they were (undefined when `out` is None). bf16 or f16, dim 64 or 128; strided
    rows are fine."""
    dev, dtype = q.get_device(), q.dtype
    code = _DTYPES.get(dtype)
    if code is None or dev < 0:
        raise _invalid("attention takes bf16 or f16 tensors on a GPU")
    if _forward._current_level >= 0:
        _no_tangents(q, k, v, out)
    qp, qs, tokens, heads, dim = _rows(q, dev, dtype, "q")
    kp, ks, keys, kv, kdim = _rows(k, dev, dtype, "k")
    vp, vs = _rows(v, dev, dtype, "v", (tokens, kv, dim))[:2]
    if keys != tokens or kdim != dim:
        raise _invalid("k and v must be [tokens, kv heads, dim] of q's tokens and dim")
    if out is None:
        out = q.new_empty((tokens, heads, dim))
        op, os_ = out.data_ptr(), heads * dim
    else:
        op, os_ = _rows(out, dev, dtype, "out", (tokens, heads, dim))[:2]
    if cu.dim() != 1 or cu.shape[0] < 1:
        raise _invalid("cu must be [seqs + 1]")
    seqs = cu.shape[0] - 1
    _call(dev, "yue2_attention_packed", qp, kp, vp, op, _flat(cu, torch.int32, dev, "cu", seqs + 1), seqs, tokens,
          heads, kv, dim, qs, ks, vs, os_, code, 1 if causal else 0, (dim or 1) ** -0.5 if scale is None else scale)
    _written(out)
    return out


def attention_tree(q, pool, layer, table, context, cu, mask=None, scale=None, out=None):
    """Attention of drafted tokens over the pages. Sequence s holds context[s] positions (int32)
    in the pages table[s] (int32 [seqs, pages]) and after them its drafted ones, at most 64,
    whose K/V are in the pages too; rows cu[s] .. cu[s + 1] - 1 of q [rows, heads, dim] are
    theirs. Row i sees the context and the drafted positions whose bit is set in mask[row]
    (int64: a node's ancestors and itself); mask None: all up to itself, so that one row per
    sequence is an ordinary decode step. A row that sees nothing, or scores of -inf alone, gets
    zeros; rows outside [cu[0], cu[-1]) of `out` are left as they were (undefined when `out` is
    None)."""
    dev, dtype, i32 = pool.index, pool.dtype, torch.int32
    if pool.data.requires_grad:
        _no_gradient("the pool")
    qp, qs, rows, heads, dim = _rows(q, dev, dtype, "q")
    if dim != pool.dim:
        raise _invalid("q must have the pool's dim")
    if _forward._current_level >= 0:
        _no_tangents(q, pool.data, out)
    if out is None:
        out = q.new_empty((rows, heads, dim))
        op, os_ = out.data_ptr(), heads * dim
    else:
        op, os_ = _rows(out, dev, dtype, "out", (rows, heads, dim))[:2]
    tp, seqs, pages = _table(table, i32, dev, "table")
    need = pool._workspace(rows, heads, seqs, pages)
    work = q.new_empty((need + 1) // 2) if need else None  # 16-bit values
    _call(dev, "yue2_attention_tree", qp, rows, heads, qs, pool._ref, layer, tp, seqs, pages,
          _flat(context, i32, dev, "context", seqs), _flat(cu, i32, dev, "cu", seqs + 1),
          0 if mask is None else _flat(mask, torch.int64, dev, "mask", rows), (dim or 1) ** -0.5 if scale is None else scale,
          op, os_, work.data_ptr() if need else 0, need)
    _written(out)
    return out


def kv_copy(pool, src, dst, count=None):
    """Positions [0, count[i]) (all 64 when count is None) of page src[i] to page dst[i], in
    every layer; int32 [n] each. The dst pages are distinct and none of them is a src page."""
    if src.dim() != 1:
        raise _invalid("src must be one list")
    dev, i32, n = pool.index, torch.int32, src.shape[0]
    if pool.data.requires_grad:
        _no_gradient("the pool")
    if _forward._current_level >= 0:
        _no_tangents(pool.data)
    _call(dev, "yue2_kv_copy", pool._ref, _flat(src, i32, dev, "src", n), _flat(dst, i32, dev, "dst", n),
          0 if count is None else _flat(count, i32, dev, "count", n), n)
    _written(pool.data)


def kv_gather(pool, src_table, dst_table, begin, cu, keep):
    """Position keep[cu[s] + i] of sequence s to its position begin[s] + i, in every layer.

    dst_table None: in place; keep strictly increasing and not before begin[s] (accepting a
    path of a drafted tree, dropping positions), and the pages written are the sequence's
    own. Otherwise into the pages of dst_table, none of which the call reads; keep in any
    order. Tables int32 [seqs, pages], begin int32 [seqs], cu int32 [seqs + 1], keep int32."""
    dev, i32 = pool.index, torch.int32
    if pool.data.requires_grad:
        _no_gradient("the pool")
    sp, seqs, pages = _table(src_table, i32, dev, "src_table")
    dp, dst_seqs, dst_pages = (0, seqs, 0) if dst_table is None else _table(dst_table, i32, dev, "dst_table")
    if dst_seqs != seqs:
        raise _invalid("src_table and dst_table must hold the same sequences")
    if keep.dim() != 1:
        raise _invalid("keep must be one list")
    if _forward._current_level >= 0:
        _no_tangents(pool.data)
    total = keep.shape[0]
    _call(dev, "yue2_kv_gather", pool._ref, sp, pages, dp, dst_pages, _flat(begin, i32, dev, "begin", seqs),
          _flat(cu, i32, dev, "cu", seqs + 1), _flat(keep, i32, dev, "keep", total), seqs, total)
    _written(pool.data)
