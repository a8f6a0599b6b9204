"""What the chunk attention's entry points refuse, without a GPU: every check precedes device work."""
import ctypes

import pytest
import torch  # noqa: F401  (before bgtq, so that one HIP runtime, torch's, serves both)

from bgtq import _lib
from test_paged_host import A, BAD_PAGES, _pages


def _desc(**kw):
    d = _lib.PagedPrefillDesc()
    base = dict(q_heads=6, dtype=_lib.DTYPE_BF16, sequences=3, tokens=100, offsets=A, lengths=A, page_table=A, page_table_stride=4,
                max_length=256, q=A, q_row_stride=384, q_head_stride=64, out=2 * A, out_row_stride=384, out_head_stride=64, workspace=A,
                workspace_bytes=1 << 40)
    for name, value in {**base, **kw}.items():
        setattr(d, name, value)
    return d


def _status(pages=None, **kw):
    return _lib.lib().bgtq_paged_prefill(None, ctypes.byref(pages or _pages()), ctypes.byref(_desc(**kw)))


@pytest.mark.parametrize("bad", BAD_PAGES, ids=str)
def test_bad_pages(bad):
    assert _status(_pages(**bad)) in (_lib.ERR_RANGE, _lib.ERR_UNSUPPORTED)
    assert b"context" not in _lib.lib().bgtq_last_error()


BAD = [dict(q_heads=0), dict(q_heads=5), dict(q_heads=34), dict(dtype=_lib.DTYPE_F32), dict(dtype=_lib.DTYPE_Q8), dict(sequences=-1),
       dict(sequences=65536), dict(tokens=-1), dict(tokens=1 << 31), dict(max_length=0), dict(max_length=(1 << 24) + 1), dict(scale=-1.0),
       dict(scale=float("nan")), dict(scale=3e38), dict(window=-1), dict(sinks=1), dict(window=4, sinks=-1), dict(window=4, sinks=(1 << 30) + 1),
       dict(page_table_stride=3), dict(page_table_stride=-4), dict(offsets=None), dict(lengths=None), dict(page_table=None), dict(q=None),
       dict(out=None), dict(offsets=A + 2), dict(lengths=A + 1), dict(page_table=A + 2), dict(q=A + 8), dict(out=A + 2), dict(q_row_stride=-8),
       dict(q_head_stride=4), dict(out_row_stride=380), dict(out_row_stride=320), dict(out_head_stride=56), dict(out=A), dict(workspace=None),
       dict(workspace=A + 8), dict(workspace_bytes=1000)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_bad_descriptors(bad):
    assert _status(**bad) == _lib.ERR_RANGE
    assert b"context" not in _lib.lib().bgtq_last_error()


def test_limits_and_workspace():
    L, n = _lib.lib(), ctypes.c_size_t()
    size = lambda **kw: (L.bgtq_paged_prefill_workspace_size(ctypes.byref(_pages()), ctypes.byref(_desc(**kw)), ctypes.byref(n)), n.value)  # noqa: E731
    # no history long enough to be split and few query columns: the counters alone
    assert size(tokens=10) == (_lib.OK, _lib.PAGED_PREFILL_COUNTER_BYTES)
    # partials, and in larger calls the rebuilt rows of sequences that may have more than 32 columns: 1 GiB of those at most
    long = dict(max_length=1 << 20, page_table_stride=1 << 15)
    few, few_more = size(**long, tokens=3), size(**long, tokens=40)
    assert few == few_more and few[1] > _lib.PAGED_PREFILL_COUNTER_BYTES
    more = size(**long, tokens=700)
    assert more[0] == _lib.OK and more[1] > few[1] + (1 << 28)
    most = size(**long, tokens=5000, sequences=60000)
    assert most[0] == _lib.OK and more[1] <= most[1] < (1 << 30) + (200 << 20)
    assert _status(tokens=(1 << 31) - 1) == _lib.ERR_UNSUPPORTED  # times the heads of a group
    assert L.bgtq_paged_prefill_workspace_size(ctypes.byref(_pages()), ctypes.byref(_desc()), None) == _lib.ERR_RANGE
    assert L.bgtq_paged_prefill(None, None, None) == L.bgtq_paged_prefill(None, ctypes.byref(_pages()), None) == _lib.ERR_RANGE
    # no rows need no pointers; what is left is the context
    assert _status(tokens=0, offsets=None, lengths=None, page_table=None, q=None, out=None) == _status() == _lib.ERR_RANGE
    assert b"context" in L.bgtq_last_error()


def test_workspace_of_rebuilt_rows():
    """4 dim heads bytes a token, of as many sequences at max_length as fit 1 GiB, and of one at least."""
    L, n, heads, dim = _lib.lib(), ctypes.c_size_t(), 8, 128
    pages = _pages(kv_heads=heads, dim=dim, k_page_stride=heads * 64 * dim, k_head_stride=64 * dim, v_page_stride=heads * 64 * dim,
                   v_head_stride=64 * dim, v_scales_page_stride=heads * 64, v_scales_head_stride=64)

    def size(max_length, sequences, tokens):
        d = _desc(q_heads=16, q_row_stride=16 * dim, q_head_stride=dim, out_row_stride=16 * dim, out_head_stride=dim, max_length=max_length,
                  page_table_stride=1 << 18, sequences=sequences, tokens=tokens)
        assert L.bgtq_paged_prefill_workspace_size(ctypes.byref(pages), ctypes.byref(d), ctypes.byref(n)) == _lib.OK
        return n.value
    few = size(64, 1, 10)  # no rebuilt rows, no partials
    assert few == _lib.PAGED_PREFILL_COUNTER_BYTES
    for max_length, sequences in ((1000, 1), (1 << 17, 1), (1 << 17, 2), (1 << 17, 3), (1 << 18, 50), (1 << 19, 1), (1 << 19, 50), (1 << 20, 1),
                                  (1 << 24, 7)):
        rows = (max_length + 63) // 64 * 64
        one = rows * heads * dim * 4
        held = max(1, min(sequences, (1 << 30) // one))
        partials = size(max_length, sequences, 3)  # (a small call's: fewer than a large one's)
        assert held * one + few <= size(max_length, sequences, 5000) <= held * one + partials + (200 << 20)
