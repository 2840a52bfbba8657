"""Packed documents over several axes on the MI355X backend (include/svl_hip.h):

* ``PositionPlan`` / ``axis_positions`` — (time, height, width) positions of
  documents made of text runs and image or video grids
* ``rope_axes`` — queries and keys rotated by them, one axis per pair of columns
* ``AttentionPlan`` / ``masked_attention`` — attention over packed documents
  with causal, window and prefix masks, a score cap and a distance bias

A plan is made once per batch and shared by its layers. Tensors are torch
tensors on the plan's device, float32 or bfloat16, with any strides but a
contiguous last axis. The calls enqueue on the device's current stream and
return; they can be captured into graphs. There is no CPU fallback.

The reference has no counterpart: its rotation takes one axis
(src/tensor/kernels.rs:1014-1035), its attention one row with a symmetric
window (kernels.rs:1037-1135).
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np
import torch

import svl_amd
from svl_amd import SvlError, _check, lib

TEXT, GRID = 0, 1
ROPE_LAYOUTS = {"half": 0, "adjacent": 1, "axial": 2}


class _Segment(ctypes.Structure):
    _fields_ = [("document", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in
                                                 ("kind", "frames", "rows", "cols", "step")]


# svl_rope_rows of queries and of keys, and svl_attention_args, as bytes.
_ROPE_ROWS = struct.Struct("=2Q5q")
_ATTENTION_ARGS = struct.Struct("=5Q8q2fQ")


class _Shape(ctypes.Structure):
    _fields_ = [("num_heads", ctypes.c_int64), ("num_kv_heads", ctypes.c_int64),
                ("head_dim", ctypes.c_int64), ("dtype", ctypes.c_int32),
                ("causal", ctypes.c_int32), ("window", ctypes.c_int64)]


_library = None


def _load():
    global _library
    if _library is None:
        L = lib()
        vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
        L.svl_position_plan_create.argtypes = [vp, vp, i64, ctypes.POINTER(vp)]
        L.svl_position_plan_destroy.argtypes = [vp]
        L.svl_position_plan_tokens.restype = i64
        L.svl_position_plan_tokens.argtypes = [vp]
        L.svl_axis_positions.argtypes = [vp, vp, vp]
        L.svl_rope_axes.argtypes = [vp, i32, i32, vp, i64, i32, i64, vp, vp, i64, i32, vp]
        L.svl_attention_plan_create.argtypes = [vp, ctypes.POINTER(_Shape), vp, vp, vp, i32,
                                                ctypes.POINTER(vp)]
        L.svl_attention_plan_destroy.argtypes = [vp]
        L.svl_attention_plan_workspace.restype = i64
        L.svl_attention_plan_workspace.argtypes = [vp]
        L.svl_masked_attention.argtypes = [vp, vp, vp, ctypes.c_size_t, vp]
        _library = L
    return _library


def _usage(msg):
    return SvlError(2, msg)


def _dtype(t):
    if t == torch.float32:
        return 0
    if t == torch.bfloat16:
        return 1
    raise SvlError(6, f"type {t}: float32 and bfloat16 are supported")


# The calls below are a few microseconds of Python each, beside kernels of as
# many: shapes and strides are read once, and nothing is converted that is
# already in its form.

def _on(device, name, t):
    """The tensor lies on the device."""
    if t.get_device() != device:
        raise _usage(f"{name} is on {t.device}, not on cuda:{device}")


def _rows(name, t, device, dtype, tokens, heads, head_dim):
    """[tokens, heads, head dim], at least `tokens` of them, with a contiguous
    last axis: (data, token stride, head stride). The strides of a single token
    or head are not used."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim or shape[0] < tokens:
        raise _usage(f"{name} of shape {tuple(shape)}: expected [{tokens}, {heads}, {head_dim}]")
    if t.dtype is not dtype or t.get_device() != device:
        raise _usage(f"{name} is {t.dtype} on {t.device}, not {dtype} on cuda:{device}")
    token, head, last = t.stride()
    if last != 1 and head_dim > 1 and t.numel():
        raise _usage(f"{name}: the last axis is not contiguous")
    return (t.data_ptr(), token if shape[0] > 1 else head_dim, head if heads > 1 else head_dim)


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device)


def _host(values, dtype):
    return np.ascontiguousarray(values, dtype)


def _array(a):
    return ctypes.c_void_p(a.ctypes.data)


class PositionPlan:
    """Positions of packed documents. `segments`: (document, kind, frames,
    rows, cols, step) each, kind TEXT (a run of `frames` tokens) or GRID."""

    def __init__(self, segments, device: svl_amd.Device | None = None):
        self.device = device or svl_amd.Device.get(0)
        rows = np.asarray(segments, np.int64).reshape(-1, 6)
        if rows.size and (rows[:, 1:].max() > 2**31 - 1 or rows[:, 1:].min() < -2**31):
            raise _usage("a segment's size does not fit 32 bits")
        table = np.zeros(len(rows), np.dtype([(n, np.int64 if n == "document" else np.int32)
                                              for n, _ in _Segment._fields_], align=True))
        for i, (name, _) in enumerate(_Segment._fields_):
            table[name] = rows[:, i]
        h = ctypes.c_void_p()
        _check(_load().svl_position_plan_create(self.device.handle, _array(table), len(rows),
                                                ctypes.byref(h)))
        self.handle = h
        self.tokens = int(_load().svl_position_plan_tokens(h))

    def __del__(self):
        if getattr(self, "handle", None) and _library is not None:
            _library.svl_position_plan_destroy(self.handle)
            self.handle = None


def axis_positions(plan: PositionPlan, out):
    """Positions of the plan's tokens into `out` [tokens, 3] (int32)."""
    device = plan.device.ordinal
    _on(device, "out", out)
    if out.dtype != torch.int32 or out.shape != (plan.tokens, 3) or not out.is_contiguous():
        raise _usage(f"positions of {plan.tokens} tokens take a contiguous int32 [tokens, 3]")
    _check(_load().svl_axis_positions(plan.handle, out.data_ptr(), _stream(device)))


def rope_axes(q, k, positions, inv_freq, pair_axis, layout, out_q, out_k):
    """Rotates q [tokens, heads, head dim] and k (may be None) by positions
    [tokens, axes] (int32): pair j by positions[:, pair_axis[j]] *
    inv_freq[j], its columns by `layout` (ROPE_LAYOUTS). out_q and out_k may
    be q and k."""
    if layout not in ROPE_LAYOUTS:
        raise _usage(f"rotation layout {layout!r} is not one of {sorted(ROPE_LAYOUTS)}")
    if q.dim() != 3 or not q.is_cuda:
        raise _usage("q must be [tokens, heads, head dim] on a GPU")
    device, dtype = q.get_device(), q.dtype
    _on(device, "positions", positions)
    if positions.dim() != 2 or positions.dtype != torch.int32 or not positions.is_contiguous():
        raise _usage("positions must be a contiguous int32 [tokens, axes]")
    tokens, axes = positions.shape
    freq, axis = _host(inv_freq, np.float32), _host(pair_axis, np.uint8)
    if freq.ndim != 1 or freq.shape != axis.shape:
        raise _usage("one frequency and one axis per pair are required")
    if (k is None) != (out_k is None):
        raise _usage("keys and their output come together")
    code, hd = _dtype(dtype), q.shape[2]
    rows, n = b"", 0
    for x, y in ((q, out_q), (k, out_k)):
        if x is None:
            continue
        shape = x.shape
        if shape != y.shape or shape[0] != tokens or len(shape) != 3:
            raise _usage(f"rows of shape {tuple(shape)} into {tuple(y.shape)}: positions are of "
                         f"{tokens} tokens")
        heads = shape[1]
        data, *strides = _rows("q or k", x, device, dtype, tokens, heads, hd)
        out, *out_strides = _rows("their output", y, device, dtype, tokens, heads, hd)
        rows += _ROPE_ROWS.pack(data, out, heads, *strides, *out_strides)
        n += 1
    # bytes pass as pointers that live as long as the call
    call = (rows, n, code, positions.data_ptr(), tokens, axes, hd, freq.tobytes(), axis.tobytes(),
            freq.size, ROPE_LAYOUTS[layout], _stream(device))
    if torch.cuda.current_device() == device:
        status = _load().svl_rope_axes(*call)
    else:
        with torch.cuda.device(device):
            status = _load().svl_rope_axes(*call)
    _check(status)


class AttentionPlan:
    """Lengths and masks of a packed batch: document d has query rows
    q_offsets[d]:q_offsets[d + 1] and key rows kv_offsets[d]:kv_offsets[d + 1]
    (None: the same), its last query at its last key. A key is visible to a
    query of its document if it is one of the first prefix[d], or if it is
    neither after it (causal) nor further than `window` from it."""

    def __init__(self, q_offsets, kv_offsets=None, *, num_heads, num_kv_heads, head_dim, dtype,
                 causal=False, window=None, prefix=None, device: svl_amd.Device | None = None):
        self.device = device or svl_amd.Device.get(0)
        q = _host(q_offsets, np.int64)
        k = None if kv_offsets is None else _host(kv_offsets, np.int64)
        p = None if prefix is None else _host(prefix, np.int64)
        if q.ndim != 1 or q.size < 1 or (k is not None and k.shape != q.shape) or \
                (p is not None and p.shape != (q.size - 1,)):
            raise _usage("offsets are [documents + 1], prefixes [documents]")
        if window is not None and window < 0:
            raise _usage("a window is None or not negative")
        self.dtype, self.num_heads, self.num_kv_heads = dtype, int(num_heads), int(num_kv_heads)
        self.head_dim = int(head_dim)
        shape = _Shape(self.num_heads, self.num_kv_heads, self.head_dim, _dtype(dtype),
                       1 if causal else 0, -1 if window is None else int(window))
        h = ctypes.c_void_p()
        _check(_load().svl_attention_plan_create(
            self.device.handle, ctypes.byref(shape), _array(q), None if k is None else _array(k),
            None if p is None else _array(p), q.size - 1, ctypes.byref(h)))
        self.handle = h
        self.q_rows, self.kv_rows = int(q[-1]), int((q if k is None else k)[-1])
        self.workspace_bytes = int(_load().svl_attention_plan_workspace(h))

    def __del__(self):
        if getattr(self, "handle", None) and _library is not None:
            _library.svl_attention_plan_destroy(self.handle)
            self.handle = None


def masked_attention(plan: AttentionPlan, q, k, v, out, scale, soft_cap=0.0, slopes=None,
                     lse=None, workspace=None):
    """Attention of q [query rows, heads, head dim] over k and v [key rows, kv
    heads, head dim] into `out`: scores scale * q . k, then cap * tanh(score /
    cap) (0: no cap), then minus slopes[head] * |position - key|. lse [query
    rows, heads] float32 receives the log of each row's sum. Rows outside
    every document are left as they were. workspace: at least
    plan.workspace_bytes of uint8, or None to allocate it for the call."""
    device, dtype = plan.device.ordinal, plan.dtype
    nh, kv, hd = plan.num_heads, plan.num_kv_heads, plan.head_dim
    rows = [_rows("q", q, device, dtype, plan.q_rows, nh, hd),
            _rows("k", k, device, dtype, plan.kv_rows, kv, hd),
            _rows("v", v, device, dtype, plan.kv_rows, kv, hd),
            _rows("out", out, device, dtype, plan.q_rows, nh, hd)]
    lse_ptr = slope_ptr = 0
    work_ptr, size = None, 0
    if slopes is not None:
        _on(device, "slopes", slopes)
        if slopes.dtype != torch.float32 or slopes.shape != (nh,) or not slopes.is_contiguous():
            raise _usage(f"slopes must be a contiguous float32 [{nh}]")
        slope_ptr = slopes.data_ptr()
    if lse is not None:
        _on(device, "lse", lse)
        if lse.dtype != torch.float32 or lse.dim() != 2 or lse.shape[0] < plan.q_rows or \
                lse.shape[1] != nh or not lse.is_contiguous():
            raise _usage(f"lse must be a contiguous float32 [query rows, {nh}]")
        lse_ptr = lse.data_ptr()
    if workspace is None and plan.workspace_bytes:
        workspace = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=q.device)
    if workspace is not None:
        _on(device, "workspace", workspace)
        if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise _usage("the workspace must be a contiguous uint8 tensor")
        work_ptr, size = workspace.data_ptr(), workspace.numel()
    (qp, *qs), (kp, *ks), (vp, *vs), (op, *os) = rows
    try:
        args = _ATTENTION_ARGS.pack(qp, kp, vp, op, lse_ptr, *qs, *ks, *vs, *os, scale, soft_cap,
                                    slope_ptr)
    except (OverflowError, struct.error):
        raise _usage(f"scale {scale} or cap {soft_cap} is no 32-bit number") from None
    _check(_load().svl_masked_attention(plan.handle, args, work_ptr, size, _stream(device)))
