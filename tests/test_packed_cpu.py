"""Host checks of the operators on packed documents (include/svl_hip.h): every
refusal comes before anything touches a device."""
import ctypes

import numpy as np
import pytest

import svl_amd
import svl_packed as P

U, LIM, UNS = "Usage", "LimitExceeded", "Unsupported"


def _status(call):
    with pytest.raises(svl_amd.SvlError) as e:
        svl_amd._check(call())
    return e.value.kind


def _ctx():
    return ctypes.byref(ctypes.c_int(0))   # a context is its device's ordinal


def _segments(rows):
    return (P._Segment * max(len(rows), 1))(*[P._Segment(*r) for r in rows])


@pytest.mark.parametrize("rows,kind", [
    ([(1, 0, 3, 0, 0, 0), (0, 0, 3, 0, 0, 0)], U),              # documents out of order
    ([(0, 2, 3, 1, 1, 1)], U),                                  # unknown kind
    ([(0, 0, -1, 1, 1, 1)], U), ([(0, 1, 2, -1, 1, 1)], U), ([(0, 1, 2, 1, -3, 1)], U),
    ([(0, 1, 2, 2, 2, 0)], U),                                  # a step that stands still
    ([(0, 1, 2**20, 2**10, 2, 1)], LIM),                        # 2^31 tokens in one grid
    ([(0, 0, 2**30, 1, 1, 1), (1, 0, 2**30, 1, 1, 1)], LIM),    # and in two segments
    ([(0, 1, 3, 1, 1, 2**30)], LIM)])                           # a position of 2^31
def test_position_plans_refuse(rows, kind):
    L = P._load()
    h = ctypes.c_void_p()
    assert _status(lambda: L.svl_position_plan_create(_ctx(), _segments(rows), len(rows),
                                                      ctypes.byref(h))) == kind
    assert not h


def test_position_plans_refuse_null_arguments():
    L = P._load()
    h = ctypes.c_void_p()
    seg = _segments([(0, 0, 1, 0, 0, 0)])
    assert _status(lambda: L.svl_position_plan_create(None, seg, 1, ctypes.byref(h))) == U
    assert _status(lambda: L.svl_position_plan_create(_ctx(), None, 1, ctypes.byref(h))) == U
    assert _status(lambda: L.svl_position_plan_create(_ctx(), seg, -1, ctypes.byref(h))) == U
    assert _status(lambda: L.svl_position_plan_create(_ctx(), seg, 1, None)) == U
    assert _status(lambda: L.svl_axis_positions(None, None, None)) == U
    assert L.svl_position_plan_destroy(None) == 0
    assert L.svl_position_plan_tokens(None) == 0


def _rope(tokens=4, axes=2, hd=8, pairs=4, layout=0, dtype=0, n=1, freq=None, axis=None,
          positions=256, **row):
    L = P._load()
    r = dict(inp=1024, out=4096, heads=2, in_token=16, in_head=8, out_token=16, out_head=8)
    r.update(row)
    rows = P._ROPE_ROWS.pack(*[r[k] or 0 for k in ("inp", "out", "heads", "in_token", "in_head",
                                                   "out_token", "out_head")])
    freq = np.ones(max(pairs, 1), np.float32) if freq is None else freq
    axis = np.zeros(max(pairs, 1), np.uint8) if axis is None else axis
    return L.svl_rope_axes(rows, n, dtype, positions, tokens, axes, hd, P._array(freq),
                           P._array(axis), pairs, layout, None)


@pytest.mark.parametrize("change,kind", [
    (dict(n=0), U), (dict(n=3), U), (dict(dtype=2), UNS), (dict(axes=0), U), (dict(axes=5), U),
    (dict(layout=3), U), (dict(hd=0, pairs=0), UNS), (dict(hd=1025), UNS), (dict(pairs=5), U),
    (dict(pairs=-1), U), (dict(hd=1024, pairs=300, in_token=2048, in_head=1024, out_token=2048,
                               out_head=1024), UNS),
    (dict(tokens=-1), U), (dict(tokens=2**31), LIM),
    (dict(axis=np.array([0, 1, 2, 0], np.uint8)), U),
    (dict(freq=np.array([1, np.inf, 1, 1], np.float32)), U),
    (dict(freq=np.array([1, np.nan, 1, 1], np.float32)), U),
    (dict(heads=-1), U), (dict(heads=32768), LIM), (dict(positions=258), U), (dict(inp=None), U), (dict(out=None), U),
    (dict(positions=None), U), (dict(in_token=-1), U), (dict(in_token=2**22 + 1), LIM),
    (dict(out_head=2**40 + 1), LIM), (dict(out_head=7), U), (dict(out_token=12), U),
    (dict(out_token=8, out_head=8), U),                       # heads and tokens share rows
    (dict(out=1024, in_token=32), U),                         # in place, with another stride
    (dict(inp=1022), U), (dict(out=4098), U), (dict(dtype=1, inp=1023), U)])
def test_rotation_refuses(change, kind):
    assert _status(lambda: _rope(**change)) == kind


@pytest.mark.parametrize("change", [dict(tokens=0), dict(heads=0), dict(pairs=0, out=1024)])
def test_rotation_of_nothing_is_no_launch(change):
    assert _rope(**change) == 0


def _plan(q=(0, 4), k=None, prefix=None, documents=None, **shape):
    L = P._load()
    s = dict(num_heads=4, num_kv_heads=2, head_dim=64, dtype=1, causal=0, window=-1)
    s.update(shape)
    h = ctypes.c_void_p()
    arr = [None if a is None else np.asarray(a, np.int64) for a in (q, k, prefix)]
    st = L.svl_attention_plan_create(
        _ctx(), ctypes.byref(P._Shape(**s)), *[None if a is None else P._array(a) for a in arr],
        len(q) - 1 if documents is None else documents, ctypes.byref(h))
    assert st == 0 or not h
    return st


@pytest.mark.parametrize("change,kind", [
    (dict(documents=-1), U), (dict(dtype=2), UNS), (dict(num_heads=3), U), (dict(num_heads=0), U),
    (dict(num_kv_heads=0), U), (dict(num_heads=65538), LIM), (dict(head_dim=0), UNS),
    (dict(head_dim=1025), UNS), (dict(q=(-1, 4)), U), (dict(q=(0, 4, 3)), U),
    (dict(q=(0, 4), k=(2, 1)), U), (dict(q=(0, 2**31)), LIM), (dict(q=(0, 4), k=(0, 2**31)), LIM),
    (dict(q=(0, 2**30 + 1), num_heads=4, num_kv_heads=2), LIM), (dict(prefix=(-1,)), U),
    (dict(q=(0, 2**31 - 4095), num_heads=1, num_kv_heads=1), LIM),
    (dict(q=(0, 2**29), num_heads=8, num_kv_heads=8), LIM)])      # groups past a launch
def test_attention_plans_refuse(change, kind):
    assert _status(lambda: _plan(**change)) == kind


def test_attention_plans_refuse_null_arguments():
    L = P._load()
    h = ctypes.c_void_p()
    off = np.array([0, 4], np.int64)
    shape = P._Shape(4, 2, 64, 1, 0, -1)
    create = L.svl_attention_plan_create
    o = P._array(off)
    assert _status(lambda: create(None, ctypes.byref(shape), o, None, None, 1, ctypes.byref(h))) == U
    assert _status(lambda: create(_ctx(), None, o, None, None, 1, ctypes.byref(h))) == U
    assert _status(lambda: create(_ctx(), ctypes.byref(shape), None, None, None, 1, ctypes.byref(h))) == U
    assert _status(lambda: create(_ctx(), ctypes.byref(shape), o, None, None, 1, None)) == U
    assert _status(lambda: L.svl_masked_attention(None, None, None, 0, None)) == U
    assert L.svl_attention_plan_destroy(None) == 0
    assert L.svl_attention_plan_workspace(None) == 0
