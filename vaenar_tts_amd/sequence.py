"""Operators on packed sequences and on a paged key / value cache (include/vaenar_hip.h, section of that name).

Ragged batches without their padding: the rows of all sequences lie one behind the other in ``[rows, heads, head_dim]`` arrays and ``cu``
(int32 ``[batch + 1]``) holds the sequences' first rows.  Arrays are ``DeviceArray``s of one engine: float32, float16, or uint16 for
bfloat16 (NumPy has no such type: the array holds its bits; ``to_bf16`` / ``from_bf16`` convert on the host).  Row strides (``ldq=`` ...,
in elements) let q, k and v be column blocks of one projection: pass a view of the first row and the stride.

The prompt of a batch goes through ``packed_attention`` and ``PagedCache.append``; every later chunk of rows -- one row a sequence in a
decoding step -- through ``append`` and ``attend``.  ``packed_attention_grad`` is the backward pass of ``packed_attention``.

Every call runs once (``Engine.call_once``): one that follows calls of the model waits until their results are known to hold, and none is
issued again when the range word is raised later.  Context, table and starts may therefore be rewritten in place between calls.
"""
import ctypes as C

import numpy as np

from ._lib import (VnrError, vnr_kv_append_desc, vnr_kv_cache, vnr_packed_attention_desc, vnr_packed_attention_grad,
                   vnr_paged_attention_desc)

_I32, _F32 = np.dtype(np.int32), np.dtype(np.float32)
_CODES = {np.dtype(np.float32): 0, np.dtype(np.float16): 1, np.dtype(np.uint16): 2}


def to_bf16(x):
    """float array -> bfloat16 bits (uint16), rounded to nearest even; NaN stays NaN."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32)
    r = ((u + (0x7FFF + ((u >> 16) & 1))) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(x):
    """bfloat16 bits (uint16) -> float32"""
    return (np.ascontiguousarray(x, np.uint16).astype(np.uint32) << 16).view(np.float32)


def _code(who, first, *others):
    kind = first.dtype
    code = _CODES.get(kind)
    if code is None:
        raise VnrError("%s: float32, float16 or uint16 (bfloat16 bits) arrays, not %s" % (who, first.dtype))
    for a in others:
        if a is not None and a.dtype is not kind and a.dtype != kind:
            raise VnrError("%s: arrays of one type: %s and %s" % (who, first.dtype, a.dtype))
    return code


def _ints(who, name, a, shape):
    if (a.dtype is not _I32 and a.dtype != _I32) or a.shape != shape:
        raise VnrError("%s: %s must be int32 %s, not %s %s" % (who, name, shape, a.dtype, a.shape))


def _shape(who, name, a, shape):
    if a.shape != shape:
        raise VnrError("%s: %s must be %s, not %s" % (who, name, shape, a.shape))


def _floats(who, name, a, shape):
    if (a.dtype is not _F32 and a.dtype != _F32) or a.shape != shape:
        raise VnrError("%s: %s must be float32 %s, not %s %s" % (who, name, shape, a.dtype, a.shape))


def _packed_desc(who, q, k, v, cu_q, cu_k, causal, scale, out, lse, ldq, ldk, ldv, ldo):
    if len(q.shape) != 3 or len(k.shape) != 3:
        raise VnrError("%s: q and k must be [rows, heads, head_dim]" % who)
    (rows_q, heads, dim), (rows_k, kv_heads, _) = q.shape, k.shape
    _shape(who, "k", k, (rows_k, kv_heads, dim))
    _shape(who, "v", v, k.shape)
    _shape(who, "out", out, q.shape)
    batch = cu_q.shape[0] - 1
    _ints(who, "cu_q", cu_q, (batch + 1,))
    _ints(who, "cu_k", cu_k, (batch + 1,))
    if lse is not None:
        _floats(who, "lse", lse, (heads, rows_q))
    return vnr_packed_attention_desc(
        _code(who, q, k, v, out), batch, heads, kv_heads, dim, 1 if causal else 0, dim ** -0.5 if scale is None else scale, rows_q, rows_k,
        cu_q.ptr, cu_k.ptr, q.ptr, k.ptr, v.ptr, ldq or heads * dim, ldk or kv_heads * dim, ldv or kv_heads * dim, out.ptr, ldo or heads * dim,
        None if lse is None else lse.ptr)


def packed_attention(engine, q, k, v, cu_q, cu_k=None, causal=True, scale=None, out=None, lse=None, ldq=None, ldk=None, ldv=None, ldo=None):
    """softmax(scale q k' + mask) v of every sequence: (out [rows_q, heads, head_dim], lse [heads, rows_q]).

    q [rows_q, heads, head_dim], k and v [rows_k, kv_heads, head_dim]; query head h reads head h // (heads // kv_heads).  ``cu_k`` defaults
    to ``cu_q``; ``scale`` to head_dim ** -0.5.  causal: row i of nq sees keys 0 .. i + nk - nq.  A row that sees no key: zeros, lse -inf."""
    if out is None:
        out = engine.empty(q.shape, q.dtype)
    if lse is None:
        lse = engine.empty((q.shape[1], q.shape[0]))
    d = _packed_desc("packed_attention", q, k, v, cu_q, cu_q if cu_k is None else cu_k, causal, scale, out, lse, ldq, ldk, ldv, ldo)
    engine.call_once("vnr_op_packed_attention", C.byref(d))
    return out, lse


def packed_attention_grad(engine, dout, q, k, v, out, lse, cu_q, cu_k=None, causal=True, scale=None, dq=None, dk=None, dv=None,
                          lddout=None, ldq=None, ldk=None, ldv=None, ldo=None, lddq=None, lddk=None, lddv=None):
    """(dq, dk, dv) of ``packed_attention`` from the gradient ``dout`` of its ``out`` and what it returned (``out``, ``lse``)."""
    who = "packed_attention_grad"
    dq = engine.empty(q.shape, q.dtype) if dq is None else dq
    dk = engine.empty(k.shape, k.dtype) if dk is None else dk
    dv = engine.empty(v.shape, v.dtype) if dv is None else dv
    d = _packed_desc(who, q, k, v, cu_q, cu_q if cu_k is None else cu_k, causal, scale, out, lse, ldq, ldk, ldv, ldo)
    _code(who, q, dout, dq, dk, dv)
    for name, a, like in (("dout", dout, q), ("dq", dq, q), ("dk", dk, k), ("dv", dv, k)):
        _shape(who, name, a, like.shape)
    wq, wk = d.heads * d.head_dim, d.kv_heads * d.head_dim
    g = vnr_packed_attention_grad(dout.ptr, lddout or wq, dq.ptr, dk.ptr, dv.ptr, lddq or wq, lddk or wk, lddv or wk)
    engine.call_once("vnr_op_packed_attention_grad", C.byref(d), C.byref(g))
    return dq, dk, dv


def rotation_table(engine, positions, rot_dim, base=10000.0):
    """float32 [positions, rot_dim]: cosines, then sines, of position / base ** (2 c / rot_dim)."""
    t = engine.empty((int(positions), int(rot_dim)))
    engine.call_once("vnr_op_rotation_table", int(positions), int(rot_dim), float(base), t.ptr)
    return t


class PagedCache:
    """Keys and values of many sequences in a pool of pages, ``[pages, kv_heads, page_size, head_dim]`` each; ``table`` (int32
    ``[batch, table_width]``) names a sequence's pages in order and belongs to the caller, like the sequences' lengths."""

    def __init__(self, engine, k, v):
        who = "PagedCache"
        if len(k.shape) != 4:
            raise VnrError("%s: the pools must be [pages, kv_heads, page_size, head_dim]" % who)
        _shape(who, "v", v, k.shape)
        self.engine, self.k, self.v = engine, k, v
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self._kind, self._row = k.dtype, (self.kv_heads, self.head_dim)
        self._desc = vnr_kv_cache(_code(who, k, v), self.kv_heads, self.head_dim, self.pages, self.page_size, k.ptr, v.ptr)
        self._ref = C.byref(self._desc)

    @classmethod
    def empty(cls, engine, pages, kv_heads, page_size, head_dim, dtype=np.uint16):
        shape = (int(pages), int(kv_heads), int(page_size), int(head_dim))
        return cls(engine, engine.zeros(shape, dtype), engine.zeros(shape, dtype))

    def _batch(self, who, cu, context, table):
        batch = cu.shape[0] - 1
        # (one look where all is well: a decoding step is a few microseconds long)
        if not (cu.dtype is _I32 and context.dtype is _I32 and table.dtype is _I32 and context.shape == (batch,) and len(cu.shape) == 1
                and len(table.shape) == 2 and table.shape[0] == batch):
            _ints(who, "cu", cu, (batch + 1,))
            _ints(who, "context", context, (batch,))
            if len(table.shape) != 2:
                raise VnrError("%s: table must be [batch, table_width]" % who)
            _ints(who, "table", table, (batch, table.shape[1]))
        return batch

    def append(self, k, v, cu, context, table, rotation=None, q=None, q_out=None, interleaved=False, ldk=None, ldv=None, ldq=None, ldqo=None):
        """k, v [rows, kv_heads, head_dim] into the cache: row cu[b] + i to position context[b] + i of sequence b.  ``rotation``
        (``rotation_table``) turns the keys' first rot_dim channels on the way, and ``q`` [rows, heads, head_dim] into ``q_out``,
        which is returned.  Positions behind the table's end and pages outside the pool are dropped."""
        who = "PagedCache.append"
        batch = self._batch(who, cu, context, table)
        rows = k.shape[0]
        if not (k.shape == v.shape and k.shape[1:] == self._row):
            _shape(who, "k", k, (rows,) + self._row)
            _shape(who, "v", v, k.shape)
        heads = 0
        if q is not None:
            heads = q.shape[1]
            _shape(who, "q", q, (rows, heads, self.head_dim))
            if q_out is None:
                q_out = self.engine.empty(q.shape, q.dtype)
            _shape(who, "q_out", q_out, q.shape)
        elif q_out is not None:
            raise VnrError("%s: q_out without q" % who)
        if not (k.dtype is v.dtype is self._kind and (q is None or q.dtype is q_out.dtype is self._kind)):
            _code(who, self.k, k, v, q, q_out)
        if rotation is not None and (rotation.dtype != _F32 or len(rotation.shape) != 2):
            raise VnrError("%s: rotation must be float32 [positions, rot_dim]" % who)
        rot = (None, 0, 0) if rotation is None else (rotation.ptr,) + rotation.shape
        wk, wq = self.kv_heads * self.head_dim, heads * self.head_dim
        d = vnr_kv_append_desc(batch, heads, rows, cu.ptr, context.ptr, table.ptr, table.shape[1], k.ptr, v.ptr, ldk or wk, ldv or wk,
                               None if q is None else q.ptr, None if q is None else q_out.ptr, ldq or wq, ldqo or wq, rot[0], rot[1], rot[2],
                               1 if interleaved else 0)
        self.engine.call_once("vnr_op_kv_append", self._ref, C.byref(d))
        return q_out

    def attend(self, q, cu, context, table, max_new, max_context, scale=None, out=None, lse=None, ldq=None, ldo=None):
        """q [rows, heads, head_dim] over everything the cache holds of their sequences: row cu[b] + i sees positions 0 .. context[b] + i
        (append the rows' own keys first).  ``max_new`` / ``max_context``: the host's bounds for the new rows and for context + new rows
        of any sequence.  Returns ``out``; ``lse`` (float32 [heads, rows]) is filled where it is given."""
        who = "PagedCache.attend"
        batch = self._batch(who, cu, context, table)
        if len(q.shape) != 3 or q.shape[2] != self.head_dim:
            raise VnrError("%s: q must be [rows, heads, %d], not %s" % (who, self.head_dim, q.shape))
        rows, heads, _ = q.shape
        if out is None:
            out = self.engine.empty(q.shape, q.dtype)
        _shape(who, "out", out, q.shape)
        if not q.dtype is out.dtype is self._kind:
            _code(who, self.k, q, out)
        if lse is not None:
            _floats(who, "lse", lse, (heads, rows))
        wq = heads * self.head_dim
        d = vnr_paged_attention_desc(batch, heads, rows, cu.ptr, context.ptr, table.ptr, table.shape[1], int(max_new), int(max_context),
                                     self.head_dim ** -0.5 if scale is None else scale, q.ptr, ldq or wq, out.ptr, ldo or wq,
                                     None if lse is None else lse.ptr)
        self.engine.call_once("vnr_op_paged_attention", self._ref, C.byref(d))
        return out
