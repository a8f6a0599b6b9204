"""What the rotation's and the windowed entry points refuse, without a GPU: every check precedes device work."""
import ctypes

import pytest
import torch  # noqa: F401  (before bgtq, so that one HIP runtime, torch's, serves both)

from bgtq import _lib
from test_paged_host import A, BAD_PAGES, _decode, _pages, _prompt
from test_paged_host import _rows as _paged_rows


def _rotation(**kw):
    r = _lib.RotationDesc()
    for name, value in {**dict(table=A, table_rows=100, q_norm=A, k_norm=None, eps=1e-6), **kw}.items():
        setattr(r, name, value)
    return r


def _heads(**kw):
    h = _lib.HeadRows()
    base = dict(src=A, dst=2 * A, heads=3, dtype=_lib.DTYPE_F16, src_row_stride=192, src_head_stride=64, dst_row_stride=192,
                dst_head_stride=64)
    for name, value in {**base, **kw}.items():
        setattr(h, name, value)
    return h


def _rotate(r=None, dim=64, rows=5, positions=A, q=None, k=None):
    ref = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
    return _lib.lib().bgtq_rotate(None, ref(r), dim, rows, positions, ref(q), ref(k))


def _append(r, positions=A, q=None, pages=None, rows=None):
    return _lib.lib().bgtq_paged_append(None, ctypes.byref(pages or _pages()), ctypes.byref(rows or _paged_rows()), ctypes.byref(r),
                                        positions, None if q is None else ctypes.byref(q))


BAD_ROTATIONS = [dict(table=None), dict(table_rows=0), dict(table_rows=-4), dict(table=A + 4), dict(q_norm=A + 2), dict(k_norm=A + 1),
                 dict(eps=-1e-9), dict(eps=float("nan")), dict(eps=float("inf"))]


@pytest.mark.parametrize("bad", BAD_ROTATIONS, ids=str)
def test_bad_rotations(bad):
    assert _rotate(_rotation(**bad), q=_heads()) == _append(_rotation(**bad)) == _lib.ERR_RANGE
    assert b"context" not in _lib.lib().bgtq_last_error()


BAD_HEADS = [dict(src=None), dict(dst=None), dict(heads=0), dict(heads=65536), dict(dtype=_lib.DTYPE_Q8), dict(dtype=-1),
             dict(src_row_stride=-64), dict(dst_head_stride=-64), dict(src=A + 1), dict(dst=2 * A + 1), dict(dst_row_stride=64),
             dict(dst_head_stride=63), dict(dst=A, dst_row_stride=256), dict(dtype=_lib.DTYPE_F32, src=A + 2)]


@pytest.mark.parametrize("bad", BAD_HEADS, ids=str)
def test_bad_rows(bad):
    good, h = _rotation(), _heads(**bad)
    assert _rotate(good, q=h) == _rotate(good, k=h) == _rotate(good, q=_heads(), k=h) == _append(good, q=h) == _lib.ERR_RANGE
    assert b"context" not in _lib.lib().bgtq_last_error()


def test_other_refusals():
    L, good = _lib.lib(), _rotation()
    assert _rotate(good, dim=96, q=_heads()) == _lib.ERR_UNSUPPORTED
    for kw in (dict(rows=-1), dict(rows=1 << 31), dict(positions=None), dict(positions=A + 4)):
        assert _rotate(good, q=_heads(), **kw) == _lib.ERR_RANGE
        assert b"context" not in L.bgtq_last_error()
    assert _rotate(good) == _rotate(None, q=_heads()) == _lib.ERR_RANGE
    for bad in BAD_PAGES[:12]:
        assert _append(good, pages=_pages(**bad)) in (_lib.ERR_RANGE, _lib.ERR_UNSUPPORTED)
    assert _append(good, rows=_paged_rows(k=None)) == _append(good, positions=None) == _lib.ERR_RANGE
    # what is left once everything else holds: no context
    assert _rotate(good, q=_heads(), k=_heads()) == _append(good, q=_heads()) == _lib.ERR_RANGE
    assert b"context" in L.bgtq_last_error()


def test_q_and_k_that_overlap():
    """One's rows are written where the other's are read or written."""
    for q, k in ((_heads(), _heads()), (_heads(), _heads(src=8 * A)), (_heads(dst=8 * A), _heads(src=8 * A, dst=16 * A)),
                 (_heads(src=16 * A, dst=8 * A), _heads(src=4 * A, dst=16 * A))):
        assert _rotate(_rotation(), q=q, k=k) == _lib.ERR_RANGE
        assert b"overlap" in _lib.lib().bgtq_last_error()
    _rotate(_rotation(), q=_heads(), k=_heads(src=4 * A, dst=4 * A))
    assert b"context" in _lib.lib().bgtq_last_error()


@pytest.mark.parametrize("bad", [None, dict(window=0), dict(window=-1), dict(sinks=-1), dict(sinks=(1 << 30) + 1)], ids=str)
def test_bad_windows(bad):
    L, n = _lib.lib(), ctypes.c_size_t()
    w = None if bad is None else ctypes.byref(_lib.Window(**{**dict(window=5, sinks=1), **bad}))
    assert L.bgtq_prompt_attention_window(None, ctypes.byref(_prompt()), w) == _lib.ERR_RANGE
    assert L.bgtq_paged_decode_window(None, ctypes.byref(_pages()), ctypes.byref(_decode()), w) == _lib.ERR_RANGE
    assert L.bgtq_paged_decode_window_workspace_size(ctypes.byref(_pages()), ctypes.byref(_decode()), w, ctypes.byref(n)) == _lib.ERR_RANGE
    assert b"context" not in L.bgtq_last_error()


def test_windowed_workspace():
    """What a window streams sizes the workspace; the other checks are those without one."""
    L, sizes = _lib.lib(), []
    d = _decode(max_length=1 << 20, page_table_stride=1 << 15)
    for window in (1, 1 << 12, 1 << 20, (1 << 31) - 1):
        n = ctypes.c_size_t()
        assert L.bgtq_paged_decode_window_workspace_size(ctypes.byref(_pages()), ctypes.byref(d), ctypes.byref(_lib.Window(window, 1 << 30 if window > 1 << 20 else 0)),
                                                         ctypes.byref(n)) == _lib.OK
        sizes.append(n.value)
    n = ctypes.c_size_t()
    assert L.bgtq_paged_decode_workspace_size(ctypes.byref(_pages()), ctypes.byref(d), ctypes.byref(n)) == _lib.OK
    assert sizes == sorted(sizes) and sizes[-1] == n.value
    good = ctypes.byref(_lib.Window(5, 1))
    assert L.bgtq_prompt_attention_window(None, ctypes.byref(_prompt(dim=96)), good) == _lib.ERR_UNSUPPORTED
    assert L.bgtq_paged_decode_window(None, ctypes.byref(_pages()), ctypes.byref(_decode(max_length=0)), good) == _lib.ERR_RANGE
