"""Single-op entry points of the C ABI (include/ivh.h) for Python callers: one operation on
device buffers the caller owns, given as integer device pointers (e.g. a torch tensor's
data_ptr()), enqueued on `stream` (a hipStream_t as an integer, None for the null stream).
The op-level counterpart of the reference's scripts/kernel_check.py driving one kernel at a
time.  Every call raises RuntimeError with the library's message on failure."""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import (AppendDesc, AttentionDesc, CacheDesc, ConvDesc, PagedAttentionDesc, RopeDesc, Rotation, _check,
               lib)

ACT_NONE, ACT_SILU, ACT_RELU, ACT_HSWISH, ACT_HSIGMOID, ACT_SIGMOID = range(6)
EW_ADD, EW_SUB, EW_MUL, EW_DIV = range(4)
POOL_MAX, POOL_RESIZE = 0, 1
F16, BF16 = 0, 1


def conv_desc(cin, cout, h, w, k=1, stride=1, pad=0, groups=1, act=ACT_NONE, has_bias=True,
              channels_last=True) -> ConvDesc:
    return ConvDesc(cin, cout, h, w, k, stride, pad, groups, act, int(bool(has_bias)), int(bool(channels_last)))


def conv_out_dims(d: ConvDesc):
    ho, wo = C.c_int(), C.c_int()
    _check(lib().ivh_conv_out_dims(C.byref(d), C.byref(ho), C.byref(wo)))
    return ho.value, wo.value


def conv_packed_bytes(d: ConvDesc) -> int:
    n = C.c_size_t()
    _check(lib().ivh_conv_packed_bytes(C.byref(d), C.byref(n)))
    return n.value


def pack_conv_weights(d: ConvDesc, w: np.ndarray, bias: np.ndarray | None, packed_dev: int) -> None:
    """w: plan-order fp16 bits [cout][cin/groups][k][k]; bias: fp16 bits [cout] or None."""
    w = np.ascontiguousarray(w, np.uint16)
    b = None if bias is None else np.ascontiguousarray(bias, np.uint16)
    _check(lib().ivh_pack_conv_weights(C.byref(d), w.ctypes.data_as(C.c_void_p),
                                       None if b is None else b.ctypes.data_as(C.c_void_p), C.c_void_p(packed_dev)))


def _vp(p):
    return None if p is None else C.c_void_p(p)


def conv2d(d: ConvDesc, x: int, packed: int, res: int | None, y: int, batch: int, stream=None) -> None:
    _check(lib().ivh_conv2d_f16(C.byref(d), _vp(x), _vp(packed), _vp(res), _vp(y), batch, _vp(stream)))


def dwconv(d: ConvDesc, x: int, packed: int, res: int | None, y: int, batch: int, stream=None) -> None:
    _check(lib().ivh_dwconv_f16(C.byref(d), _vp(x), _vp(packed), _vp(res), _vp(y), batch, _vp(stream)))


def gemv(d: ConvDesc, x: int, packed: int, y: int, batch: int, stream=None) -> None:
    _check(lib().ivh_gemv_f16(C.byref(d), _vp(x), _vp(packed), _vp(y), batch, _vp(stream)))


def eltwise(op: int, a: int, b: int | None, y: int, n: int, batch: int, b_scalar=False, stream=None) -> None:
    _check(lib().ivh_eltwise_f16(op, _vp(a), _vp(b), int(b_scalar), _vp(y), n, batch, _vp(stream)))


def pool(kind: int, x: int, y: int, c: int, h: int, w: int, k: int, s: int, p: int, batch: int, stream=None) -> None:
    _check(lib().ivh_pool_f16(kind, _vp(x), _vp(y), c, h, w, k, s, p, batch, _vp(stream)))


def softmax(x: int, y: int, outer: int, axis: int, inner: int, batch: int, stream=None) -> None:
    _check(lib().ivh_softmax_f16(_vp(x), _vp(y), outer, axis, inner, batch, _vp(stream)))


def bmm(a: int, b: int, y: int, bb: int, m: int, k: int, n: int, batch: int, stream=None) -> None:
    _check(lib().ivh_bmm_f16(_vp(a), _vp(b), _vp(y), bb, m, k, n, batch, _vp(stream)))


# ---- sequence operators (include/ivh.h).  Strides are (token, head) in elements; positions, lengths, page
# tables and row offsets are int32 device arrays.  Descriptors may be kept and reused.

def rotation(sections=(), rot=None, adjacent=False, dealt=False) -> Rotation:
    """sections: frequencies of each axis; rot defaults to twice their sum."""
    sections = tuple(sections)
    if len(sections) > 4:
        raise RuntimeError("rotation: 1 to 4 axes")
    return Rotation(2 * sum(sections) if rot is None else rot, int(bool(adjacent)), len(sections),
                    (C.c_int * 4)(*sections), int(bool(dealt)))


def rope_desc(type, heads, dim, sections, rot=None, adjacent=False, dealt=False, x=None, y=None, pos_axis=0) -> RopeDesc:
    """x, y: strides, dense rows by default; pos_axis: elements between two axes' positions."""
    dense = (heads * dim, dim)
    x, y = x or dense, y or dense
    return RopeDesc(type, heads, dim, rotation(sections, rot, adjacent, dealt), x[0], x[1], y[0], y[1], pos_axis)


def rope(d: RopeDesc, x: int, pos: int, freq: int, y: int, tokens: int, stream=None) -> None:
    _check(lib().ivh_rope(d, x, pos, freq, y, tokens, stream))


def cache_desc(type, bits, heads, dim, page, pages, table_width) -> CacheDesc:
    return CacheDesc(type, bits, heads, dim, page, pages, table_width)


def cache_bytes(d: CacheDesc):
    """(bytes of each page buffer, bytes of each scale buffer)."""
    a, b = C.c_size_t(), C.c_size_t()
    _check(lib().ivh_cache_bytes(d, C.byref(a), C.byref(b)))
    return a.value, b.value


def append_desc(cache: CacheDesc, sections=(), rot=None, adjacent=False, dealt=False, k=None, v=None, pos_axis=0) -> AppendDesc:
    """No sections: keys are not rotated."""
    dense = (cache.heads * cache.dim, cache.dim)
    k, v = k or dense, v or dense
    return AppendDesc(cache, rotation(sections, rot, adjacent, dealt), k[0], k[1], v[0], v[1], pos_axis)


def kv_append(d: AppendDesc, k, v, pos, freq, cu, lens, table, kc, vc, ks, vs, batch: int, tokens: int, stream=None) -> None:
    _check(lib().ivh_kv_append(d, k, v, pos, freq, cu, lens, table, kc, vc, ks, vs, batch, tokens, stream))


def paged_attention_desc(cache: CacheDesc, heads, scale, window=0, sinks=0, q=None, o=None, max_new=0,
                         max_len=0) -> PagedAttentionDesc:
    dense = (heads * cache.dim, cache.dim)
    q, o = q or dense, o or dense
    return PagedAttentionDesc(cache, heads, scale, window, sinks, q[0], q[1], o[0], o[1], max_new, max_len)


def paged_attention_workspace(d: PagedAttentionDesc, batch: int, tokens: int) -> int:
    n = C.c_size_t()
    _check(lib().ivh_paged_attention_workspace(d, batch, tokens, C.byref(n)))
    return n.value


def paged_attention(d: PagedAttentionDesc, q, kc, vc, ks, vs, cu, lens, table, o, batch: int, tokens: int, workspace=None,
                    workspace_bytes=0, stream=None) -> None:
    _check(lib().ivh_paged_attention(d, q, kc, vc, ks, vs, cu, lens, table, o, batch, tokens, workspace, workspace_bytes, stream))


def attention_desc(type, heads, kv_heads, dim, scale, causal=True, window=0, sinks=0, q=None, k=None, v=None, o=None,
                   max_q=0) -> AttentionDesc:
    dq, dk = (heads * dim, dim), (kv_heads * dim, dim)
    q, k, v, o = q or dq, k or dk, v or dk, o or dq
    return AttentionDesc(type, heads, kv_heads, dim, scale, int(bool(causal)), window, sinks, q[0], q[1], k[0], k[1], v[0], v[1],
                         o[0], o[1], max_q)


def attention(d: AttentionDesc, q, k, v, cu_q, cu_k, o, batch: int, tokens_q: int, tokens_k: int, stream=None) -> None:
    _check(lib().ivh_attention(d, q, k, v, cu_q, cu_k, o, batch, tokens_q, tokens_k, stream))
