"""Rows that a call writes where it reads others, in the rotation, the append and the chunks: refused without a GPU, by the
bytes of the rows themselves, so that slices of one buffer that do not meet are taken."""
import ctypes
import random

import pytest
import torch  # noqa: F401  (before bgtq, so that one HIP runtime, torch's, serves both)

from bgtq import _lib
from test_chunk_host import _status
from test_paged_host import A
from test_paged_host import _rows as _paged_rows
from test_rotate_host import _append, _heads, _rotate, _rotation

SIZE = {_lib.DTYPE_F32: 4, _lib.DTYPE_F16: 2, _lib.DTYPE_BF16: 2}


def _refused(status):
    """Whether for an overlap; what is left otherwise is the context."""
    assert status == _lib.ERR_RANGE
    message = _lib.lib().bgtq_last_error()
    assert b"overlap" in message or b"context" in message, message
    return b"overlap" in message


def _bytes(at, rows, row, heads, head, size, dim=64):
    return {b for i in range(rows) for h in range(heads) for b in range(at + (i * row + h * head) * size, at + (i * row + h * head + dim) * size)}


def _src(h, rows):
    return _bytes(h.src, rows, h.src_row_stride, h.heads, h.src_head_stride, SIZE[h.dtype])


def _dst(h, rows):
    return _bytes(h.dst, rows, h.dst_row_stride, h.heads, h.dst_head_stride, SIZE[h.dtype])


def _row(count, dtype, at, row, head=64, to=None, to_row=None):
    return _heads(src=at, dst=at if to is None else to, heads=count, dtype=dtype, src_row_stride=row, src_head_stride=head,
                  dst_row_stride=row if to_row is None else to_row, dst_head_stride=head)


def test_slices_of_one_projection():
    """Nine heads of q, three of k and three of v in rows of 960 values: in place each by itself, not one over another."""
    wide, at = 15 * 64, lambda head: A + 2 * 64 * head
    q, k = _row(9, _lib.DTYPE_BF16, at(0), wide), _row(3, _lib.DTYPE_BF16, at(9), wide)
    rows = _paged_rows(k=at(9), v=at(12), k_row_stride=wide, v_row_stride=wide, v_dtype=_lib.DTYPE_BF16)
    assert not _refused(_rotate(_rotation(), q=q, k=k)) and not _refused(_append(_rotation(), q=q, rows=rows))
    # the queries, rotated, over the keys' heads, over the values', over both's first rows, or one value into the keys
    for to, to_row in ((at(9), wide), (at(3), wide), (at(12), wide), (at(0) + 2 * 64 * 9 - 9 * 64 * 2, 9 * 64), (at(0) + 2, wide)):
        over = _row(9, _lib.DTYPE_BF16, A - (1 << 19), wide, to=to, to_row=to_row)
        met = _dst(over, 5) & (_bytes(at(9), 5, wide, 2, 64, 2) | _bytes(at(12), 5, wide, 2, 64, 2))
        assert met and _refused(_append(_rotation(), q=over, rows=rows))
    assert _refused(_append(_rotation(), q=_row(1, _lib.DTYPE_F32, 4 * A, 64, to=at(9)), rows=rows))
    # one FP32 head: its five dense rows are 1280 bytes, ten heads of the projection; from head 60 (row 4) they end on the
    # first key of row 4, head 69; from its last row's end on they meet nothing
    assert _refused(_append(_rotation(), q=_row(1, _lib.DTYPE_F32, 4 * A, 64, to=at(60)), rows=rows))
    assert not _refused(_append(_rotation(), q=_row(1, _lib.DTYPE_F32, 4 * A, 64, to=at(75)), rows=rows))


def test_rows_rotated_onto_their_neighbours():
    """A destination that is not the source and meets it: a row, a head or one value on."""
    for by in (192, 64, 1, -192, 4 * 192):
        h = _heads(dst=A + 2 * by)
        for got in (_rotate(_rotation(), q=h), _rotate(_rotation(), k=h), _append(_rotation(), q=h, rows=_paged_rows(k=8 * A, v=8 * A))):
            assert _refused(got)
    assert not _refused(_rotate(_rotation(), q=_heads(dst=A + 2 * 5 * 192)))
    assert not _refused(_rotate(_rotation(), rows=0, q=_heads(dst=A + 2)))


def test_chunks_into_their_queries():
    """out as a view of q's buffer: a row, a head or eight values on; other heads of the same rows are apart."""
    for by in (384, 64, 8, -384, 99 * 384):
        assert _refused(_status(out=A + 2 * by))
    assert not _refused(_status(out=A + 2 * 100 * 384))
    wide = dict(q_row_stride=768, out_row_stride=768)
    assert not _refused(_status(out=A + 2 * 384, **wide)) and _refused(_status(out=A + 2 * 376, **wide))
    assert not _refused(_status(out=A + 2 * 64, q_head_stride=128, out_head_stride=128, **wide))
    assert _refused(_status(out=A + 2 * 72, q_head_stride=128, out_head_stride=128, **wide))
    # heads outermost
    heads = dict(q_row_stride=64, q_head_stride=12800, out_row_stride=64, out_head_stride=12800)
    assert not _refused(_status(out=A + 2 * 6400, **heads)) and _refused(_status(out=A + 2 * 6336, **heads))


@pytest.mark.parametrize("seed", range(40))
def test_any_layouts(seed):
    """Refused exactly where a byte is in two sets of rows, one of them written: against the bytes themselves."""
    rng, met = random.Random(seed), 0
    for _ in range(60):
        rows, unit, hs = rng.randint(1, 5), rng.choice([8, 16, 64]), []
        for _h in range(2):
            heads, dtype = rng.randint(1, 4), rng.choice(list(SIZE))

            def strides():
                head = 64 + unit * rng.randint(0, 6)
                row = (heads - 1) * head + 64 + unit * rng.randint(0, 12)
                if rng.random() < 0.3:  # heads outermost
                    row = 64 + unit * rng.randint(0, 4)
                    head = (rows - 1) * row + 64 + unit * rng.randint(0, 8)
                return row, head
            (r0, h0), (r1, h1) = strides(), strides()
            if rng.random() < 0.2:
                r1, h1 = r0, h0
            src, dst = (A + 4 * unit * rng.randint(0, 400) for _x in range(2))
            if rng.random() < 0.4:
                dst, r1, h1 = src, r0, h0
            hs.append(_heads(src=src, dst=dst, heads=heads, dtype=dtype, src_row_stride=r0, src_head_stride=h0, dst_row_stride=r1, dst_head_stride=h1))
        q, k = hs
        own = any(h.src != h.dst and _src(h, rows) & _dst(h, rows) for h in hs)
        cross = _dst(q, rows) & _src(k, rows) or _dst(q, rows) & _dst(k, rows) or _src(q, rows) & _dst(k, rows)
        if any(h.src == h.dst and (h.src_row_stride, h.src_head_stride) != (h.dst_row_stride, h.dst_head_stride) for h in hs):
            continue  # refused for its strides
        want = bool(own or cross)
        met += want
        assert _refused(_rotate(_rotation(), rows=rows, q=q, k=k)) == want, (rows, [(getattr(h, n), n) for h in hs for n, _t in h._fields_])
    assert met


def test_sizes_at_the_limits():
    """Strides and rows whose products pass 64 bits: no wrap, and no time."""
    far = _heads(src=A, dst=1 << 60, src_row_stride=1 << 61, dst_row_stride=1 << 61)
    assert not _refused(_rotate(_rotation(), rows=(1 << 31) - 1, q=far))
    # more pairs of pieces than are compared: left to the caller, as the header says
    many = _heads(src=A, dst=A + 2 * 64, heads=65535, src_head_stride=128, dst_head_stride=130, src_row_stride=65535 * 128, dst_row_stride=65535 * 130)
    _refused(_rotate(_rotation(), rows=1 << 20, q=many))
    assert ctypes.sizeof(_lib.HeadRows) == 56
