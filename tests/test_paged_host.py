"""What the paged cache's and the prompt attention's entry points refuse, without a GPU: every check precedes device work."""
import ctypes

import pytest
import torch  # (before bgtq, so that one HIP runtime, torch's, serves both)

import bgtq
from bgtq import _lib

A = 1 << 20  # an aligned address that no call reaches


def _pages(**kw):
    g = _lib.Pages()
    base = dict(kv_heads=2, dim=64, key_format=_lib.KEYS_FP16, v_format=_lib.DTYPE_Q8, page_tokens=64, pages=10, k_f16=A,
                k_page_stride=2 * 64 * 64, k_head_stride=64 * 64, v=A, v_page_stride=2 * 64 * 64, v_head_stride=64 * 64, v_scales=A,
                v_scales_page_stride=128, v_scales_head_stride=64)
    for name, value in {**base, **kw}.items():
        setattr(g, name, value)
    return g


def _rows(**kw):
    r = _lib.PagedRows()
    base = dict(rows=5, slots=A, k=A, k_dtype=_lib.DTYPE_BF16, k_row_stride=128, k_head_stride=64, v=A, v_dtype=_lib.DTYPE_F32,
                v_row_stride=128, v_head_stride=64)
    for name, value in {**base, **kw}.items():
        setattr(r, name, value)
    return r


def _decode(**kw):
    d = _lib.PagedDecodeDesc()
    base = dict(batch=3, q_heads=6, q=A, out=A, lengths=A, page_table=A, page_table_stride=4, max_length=256)
    for name, value in {**base, **kw}.items():
        setattr(d, name, value)
    return d


def _prompt(**kw):
    d = _lib.PromptDesc()
    base = dict(q_heads=6, kv_heads=2, dim=64, dtype=_lib.DTYPE_BF16, sequences=3, tokens=100, offsets=A, q=A, q_row_stride=640,
                q_head_stride=64, k=A, k_row_stride=640, k_head_stride=64, v=A, v_row_stride=640, v_head_stride=64, out=A,
                out_row_stride=384, out_head_stride=64)
    for name, value in {**base, **kw}.items():
        setattr(d, name, value)
    return d


BAD_PAGES = [dict(kv_heads=0), dict(kv_heads=17), dict(dim=96), dict(page_tokens=16), dict(page_tokens=48), dict(page_tokens=8192),
             dict(page_tokens=-64), dict(pages=0), dict(pages=1 << 31), dict(key_format=2), dict(v_format=_lib.DTYPE_F32), dict(k_f16=None),
             dict(v=None), dict(v_scales=None), dict(k_f16=A + 8), dict(v=A + 4), dict(v_scales=A + 2), dict(k_page_stride=-8),
             dict(k_page_stride=2 * 64 * 64 + 4), dict(v_head_stride=64 * 64 - 16), dict(v_scales_page_stride=63), dict(k_head_stride=0),
             dict(key_format=_lib.KEYS_PACKED),
             dict(k_page_stride=64 * 64), dict(v_page_stride=64 * 64, v_head_stride=9 * 64 * 64),
             dict(v_scales_page_stride=1 << 62, v_scales_head_stride=1 << 61, kv_heads=16, pages=1 << 30)]


@pytest.mark.parametrize("bad", BAD_PAGES, ids=str)
def test_bad_pages(bad):
    L, g, n = _lib.lib(), _pages(**bad), ctypes.c_size_t()
    status = {L.bgtq_paged_write(None, ctypes.byref(g), ctypes.byref(_rows())),
              L.bgtq_paged_read(None, ctypes.byref(g), ctypes.byref(_rows())),
              L.bgtq_paged_decode(None, ctypes.byref(g), ctypes.byref(_decode())),
              L.bgtq_paged_decode_workspace_size(ctypes.byref(g), ctypes.byref(_decode()), ctypes.byref(n))}
    assert len(status) == 1 and status <= {_lib.ERR_RANGE, _lib.ERR_UNSUPPORTED}
    assert b"context" not in L.bgtq_last_error()


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(rows=1 << 31), dict(slots=None), dict(slots=A + 4), dict(k_dtype=_lib.DTYPE_Q8),
                                 dict(v_dtype=7), dict(k_row_stride=-1), dict(v_head_stride=-64), dict(k=A + 1), dict(v=A + 2)], ids=str)
def test_bad_rows(bad):
    L = _lib.lib()
    for call in (L.bgtq_paged_write, L.bgtq_paged_read):
        assert call(None, ctypes.byref(_pages()), ctypes.byref(_rows(**bad))) == _lib.ERR_RANGE
        assert b"context" not in L.bgtq_last_error()


def test_overlaps():
    """Rows that are written lie apart, pages or rows outermost or heads; rows that are only read may not."""
    L, S = _lib.lib(), 64 * 64
    for page, head, good in ((2 * S, S, True), (S, 10 * S, True), (S, 9 * S, False), (S, S, False), (2 * S - 64, S, False)):
        g = _pages(k_page_stride=page, k_head_stride=head)
        assert L.bgtq_paged_read(None, ctypes.byref(g), ctypes.byref(_rows())) == _lib.ERR_RANGE
        assert (L.bgtq_last_error() == b"null context") == good, (page, head)
    for row, head, good in ((128, 64, True), (64, 320, True), (64, 256, False), (0, 0, False), (64, 64, False), (120, 64, False)):
        r = _rows(k_row_stride=row, k_head_stride=head)
        assert L.bgtq_paged_read(None, ctypes.byref(_pages()), ctypes.byref(r)) == _lib.ERR_RANGE
        assert (L.bgtq_last_error() == b"null context") == good, (row, head)
        assert L.bgtq_paged_write(None, ctypes.byref(_pages()), ctypes.byref(r)) == _lib.ERR_RANGE
        assert L.bgtq_last_error() == b"null context"
    for row, head, good in ((384, 64, True), (64, 6400, True), (64, 6392, False), (376, 64, False), (64, 64, False)):
        d = _prompt(out_row_stride=row, out_head_stride=head)
        assert L.bgtq_prompt_attention(None, ctypes.byref(d)) == _lib.ERR_RANGE
        assert (L.bgtq_last_error() == b"null context") == good, (row, head)


def test_most_prompt_rows():
    """A launch holds 2^32 work-items, 256 per 128 rows of a head and sequence."""
    L = _lib.lib()
    for tokens, sequences, heads, good in (((1 << 24) * 128 // 16 - 256, 1, 16, True), ((1 << 24) * 128 // 16, 1, 16, False),
                                           ((1 << 31) - 1, 1, 2, False), ((1 << 31) - 256, 1, 1, True)):
        d = _prompt(tokens=tokens, sequences=sequences, q_heads=heads, kv_heads=1, out_row_stride=64 * heads)
        assert L.bgtq_prompt_attention(None, ctypes.byref(d)) in (_lib.ERR_RANGE, _lib.ERR_UNSUPPORTED)
        assert (L.bgtq_last_error() == b"null context") == good, (tokens, heads)


def test_rows_that_are_missing():
    L = _lib.lib()
    for r, write, read in ((_rows(k=None), b"null K or V rows", b"null context"), (_rows(k=None, v=None), b"null K or V rows", b"null K or V rows")):
        assert L.bgtq_paged_write(None, ctypes.byref(_pages()), ctypes.byref(r)) == _lib.ERR_RANGE
        assert L.bgtq_last_error() == write
        assert L.bgtq_paged_read(None, ctypes.byref(_pages()), ctypes.byref(r)) == _lib.ERR_RANGE
        assert L.bgtq_last_error() == read
    for call in (L.bgtq_paged_write, L.bgtq_paged_read):
        assert call(None, None, ctypes.byref(_rows())) == _lib.ERR_RANGE
        assert call(None, ctypes.byref(_pages()), None) == _lib.ERR_RANGE
        assert call(None, ctypes.byref(_pages()), ctypes.byref(_rows())) == _lib.ERR_RANGE  # all good but for the context
        assert L.bgtq_last_error() == b"null context"


@pytest.mark.parametrize("bad", [dict(batch=0), dict(batch=65536), dict(q_heads=5), dict(q_heads=34), dict(q_heads=0), dict(max_length=0),
                                 dict(max_length=257), dict(max_length=(1 << 24) + 1, page_table_stride=1 << 20), dict(q=None), dict(out=None),
                                 dict(lengths=None), dict(page_table=None), dict(q=A + 4), dict(out=A + 8), dict(page_table=A + 2),
                                 dict(page_table_stride=3), dict(page_table_stride=-4), dict(q_rotated=2), dict(q_rotated=1)], ids=str)
def test_bad_decodes(bad):
    L, n = _lib.lib(), ctypes.c_size_t()
    for status in (L.bgtq_paged_decode_workspace_size(ctypes.byref(_pages()), ctypes.byref(_decode(**bad)), ctypes.byref(n)),
                   L.bgtq_paged_decode(None, ctypes.byref(_pages()), ctypes.byref(_decode(**bad)))):
        assert status in (_lib.ERR_RANGE, _lib.ERR_UNSUPPORTED)
        assert b"workspace" not in L.bgtq_last_error() and b"context" not in L.bgtq_last_error()


def test_decode_workspace():
    L, n = _lib.lib(), ctypes.c_size_t()
    assert L.bgtq_paged_decode_workspace_size(ctypes.byref(_pages()), ctypes.byref(_decode()), ctypes.byref(n)) == _lib.OK
    for ws, size in ((None, 1 << 30), (A, n.value - 1), (A + 8, n.value)):
        assert L.bgtq_paged_decode(None, ctypes.byref(_pages()), ctypes.byref(_decode(workspace=ws, workspace_bytes=size))) == _lib.ERR_RANGE
        assert b"workspace" in L.bgtq_last_error()
    assert L.bgtq_paged_decode(None, ctypes.byref(_pages()), ctypes.byref(_decode(workspace=A, workspace_bytes=n.value))) == _lib.ERR_RANGE
    assert L.bgtq_last_error() == b"null context"


@pytest.mark.parametrize("bad", [dict(q_heads=5), dict(kv_heads=0), dict(q_heads=0), dict(q_heads=65536), dict(dim=80), dict(dtype=_lib.DTYPE_F32),
                                 dict(sequences=-1), dict(sequences=65536), dict(tokens=-1), dict(tokens=1 << 31), dict(scale=-0.1),
                                 dict(scale=float("nan")), dict(scale=float("inf")), dict(offsets=None), dict(q=None), dict(k=None), dict(v=None),
                                 dict(out=None), dict(offsets=A + 2), dict(q=A + 8), dict(k_row_stride=644), dict(v_head_stride=-64),
                                 dict(out_row_stride=56), dict(k_row_stride=(1 << 22) + 8), dict(q_heads=65534, tokens=(1 << 31) - 1)], ids=str)
def test_bad_prompts(bad):
    L = _lib.lib()
    assert L.bgtq_prompt_attention(None, ctypes.byref(_prompt(**bad))) in (_lib.ERR_RANGE, _lib.ERR_UNSUPPORTED)
    assert b"context" not in L.bgtq_last_error()
    assert L.bgtq_prompt_attention(None, ctypes.byref(_prompt())) == _lib.ERR_RANGE
    assert L.bgtq_last_error() == b"null context"


def test_wrappers_want_gpu_tensors():
    from bgtq import batched
    x = torch.zeros((4, 2, 32, 64), dtype=torch.float16)
    with pytest.raises(bgtq.RangeError):
        batched.pages(page_tokens=32, v=x, k_f16=x)


def test_prompt_scales():
    """Every accepted scale times log2(e) is finite in FP32."""
    L = _lib.lib()
    for scale, good in ((0.0, True), (1e-45, True), (2.0e38, True), (2.5e38, False), (3.0e38, False), (3.4e38, False)):
        assert L.bgtq_prompt_attention(None, ctypes.byref(_prompt(scale=scale))) == _lib.ERR_RANGE
        assert (L.bgtq_last_error() == b"null context") == good, scale
