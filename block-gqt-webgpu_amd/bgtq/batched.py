"""Batched model-geometry entry points over caller-owned device memory.

Thin wrappers over bgtq_encode_batched / bgtq_decode (include/bgtq.h) that
take torch tensors resident on the GPU (torch supplies device memory and the
stream; all arithmetic runs in libbgtq.so). Used for layers x sequences x KV
heads workloads: the model dispatch sites encode_k / compressed_dot / softmax /
weighted of src/model/decoder.ts:46-56.
"""
from __future__ import annotations

import ctypes

from . import _lib
from ._lib import RangeError, check, lib


def _addr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def bind_torch_stream(device):
    """Order the context's work on torch's current stream."""
    import torch
    device.set_stream(torch.cuda.current_stream().cuda_stream)


def encode(device, jobs, src_dtype="f16"):
    """jobs: iterable of dicts {tables, src, src_row_stride, rows, packed, norms, dst_row0}."""
    jobs = list(jobs)
    arr = (_lib.EncodeJob * max(1, len(jobs)))()
    for i, j in enumerate(jobs):
        arr[i] = _lib.EncodeJob(j["tables"].handle, _addr(j["src"]), int(j["src_row_stride"]), int(j["rows"]),
                                _addr(j["packed"]), _addr(j["norms"]), int(j.get("dst_row0", 0)))
    code = {"f16": _lib.DTYPE_F16, "f32": _lib.DTYPE_F32}[src_dtype]
    check(lib().bgtq_encode_batched(device.handle, code, arr, len(jobs)))


def decode_desc(*, batch, q_heads, kv_heads, dim, q, out, lengths, max_length, v, v_dtype="f16",
                v_seq_stride, v_head_stride, tables=None, packed=None, packed_seq_stride=0,
                packed_head_stride=0, norms=None, norms_seq_stride=0, norms_head_stride=0, k_f16=None,
                k_seq_stride=0, k_head_stride=0, splits=0, workspace=None, q_rotated=False):
    """bgtq_decode_desc over device tensors. q_rotated: q is already R q[perm] per its KV head's
    tables (from a projection baked with calibrate.bake_qproj)."""
    d = _lib.DecodeDesc()
    d.q_rotated = int(bool(q_rotated))
    d.batch, d.q_heads, d.kv_heads, d.dim = batch, q_heads, kv_heads, dim
    d.key_format = _lib.KEYS_PACKED if packed is not None else _lib.KEYS_FP16
    for i, t in enumerate(tables or []):
        d.tables[i] = t.handle.value if hasattr(t.handle, "value") else t.handle
    d.packed, d.packed_seq_stride, d.packed_head_stride = _addr(packed), packed_seq_stride, packed_head_stride
    d.norms, d.norms_seq_stride, d.norms_head_stride = _addr(norms), norms_seq_stride, norms_head_stride
    d.k_f16, d.k_seq_stride, d.k_head_stride = _addr(k_f16), k_seq_stride, k_head_stride
    d.v, d.v_dtype = _addr(v), {"f32": _lib.DTYPE_F32, "f16": _lib.DTYPE_F16}[v_dtype]
    d.v_seq_stride, d.v_head_stride = v_seq_stride, v_head_stride
    d.q, d.out, d.lengths = _addr(q), _addr(out), _addr(lengths)
    d.max_length, d.splits = int(max_length), int(splits)
    if workspace is not None:
        d.workspace, d.workspace_bytes = _addr(workspace), workspace.numel() * workspace.element_size()
    return d


def workspace_bytes(desc) -> int:
    n = ctypes.c_size_t(0)
    check(lib().bgtq_decode_workspace_size(ctypes.byref(desc), ctypes.byref(n)))
    return n.value


def decode(device, desc) -> None:
    check(lib().bgtq_decode(device.handle, ctypes.byref(desc)))


def decode_noalloc(device, desc) -> None:
    """bgtq_decode_noalloc: the decode with the library's own device scratch (the descriptor's
    workspace is ignored); nothing is allocated."""
    check(lib().bgtq_decode_noalloc(device.handle, ctypes.byref(desc)))


def append_desc(*, k_new, v_new):
    """bgtq_append_desc over device tensors [B, Hkv, dim] (FP32 or FP16, any strides in elements)."""
    a = _lib.AppendDesc()
    dt = {"torch.float32": _lib.DTYPE_F32, "torch.float16": _lib.DTYPE_F16}
    a.k_new, a.k_new_dtype = _addr(k_new), dt[str(k_new.dtype)]
    a.k_new_seq_stride, a.k_new_head_stride = k_new.stride(0), k_new.stride(1)
    a.v_new, a.v_new_dtype = _addr(v_new), dt[str(v_new.dtype)]
    a.v_new_seq_stride, a.v_new_head_stride = v_new.stride(0), v_new.stride(1)
    return a


def decode_append(device, desc, append) -> None:
    """The decode step with its new token (bgtq_decode_append): row lengths[b] - 1 of the caches."""
    check(lib().bgtq_decode_append(device.handle, ctypes.byref(desc), ctypes.byref(append)))


def prefill_desc(*, batch, rows, q_heads, kv_heads, dim, q, out, starts, max_length, v, v_seq_stride,
                 v_head_stride, tables=None, packed=None, packed_seq_stride=0, packed_head_stride=0, norms=None,
                 norms_seq_stride=0, norms_head_stride=0, k_f16=None, k_seq_stride=0, k_head_stride=0,
                 split_tokens=0, workspace=None, q_rotated=False):
    """bgtq_prefill_desc over device tensors: q/out [B, rows, Hq, dim] FP32, v FP16, starts uint32 [B];
    q_rotated as for decode_desc."""
    d = _lib.PrefillDesc()
    d.q_rotated = int(bool(q_rotated))
    d.batch, d.rows, d.q_heads, d.kv_heads, d.dim = batch, rows, q_heads, kv_heads, dim
    d.key_format = _lib.KEYS_PACKED if packed is not None else _lib.KEYS_FP16
    for i, t in enumerate(tables or []):
        d.tables[i] = t.handle.value if hasattr(t.handle, "value") else t.handle
    d.packed, d.packed_seq_stride, d.packed_head_stride = _addr(packed), packed_seq_stride, packed_head_stride
    d.norms, d.norms_seq_stride, d.norms_head_stride = _addr(norms), norms_seq_stride, norms_head_stride
    d.k_f16, d.k_seq_stride, d.k_head_stride = _addr(k_f16), k_seq_stride, k_head_stride
    d.v, d.v_seq_stride, d.v_head_stride = _addr(v), v_seq_stride, v_head_stride
    d.q, d.out, d.starts = _addr(q), _addr(out), _addr(starts)
    d.max_length, d.split_tokens = int(max_length), int(split_tokens)
    if workspace is not None:
        d.workspace, d.workspace_bytes = _addr(workspace), workspace.numel() * workspace.element_size()
    return d


def prefill_workspace_bytes(desc) -> int:
    n = ctypes.c_size_t(0)
    check(lib().bgtq_prefill_workspace_size(ctypes.byref(desc), ctypes.byref(n)))
    return n.value


def prefill_append_desc(*, k_new, v_new):
    """bgtq_prefill_append_desc over device tensors [B, rows, Hkv, dim] (FP32 or FP16, any strides in
    elements)."""
    a = _lib.PrefillAppendDesc()
    dt = {"torch.float32": _lib.DTYPE_F32, "torch.float16": _lib.DTYPE_F16}
    a.k_new, a.k_new_dtype = _addr(k_new), dt[str(k_new.dtype)]
    a.k_new_seq_stride, a.k_new_row_stride, a.k_new_head_stride = k_new.stride(0), k_new.stride(1), k_new.stride(2)
    a.v_new, a.v_new_dtype = _addr(v_new), dt[str(v_new.dtype)]
    a.v_new_seq_stride, a.v_new_row_stride, a.v_new_head_stride = v_new.stride(0), v_new.stride(1), v_new.stride(2)
    return a


def prefill_append(device, desc, append) -> None:
    """A prefill chunk with its own rows encoded and appended in the same launch (bgtq_prefill_append)."""
    check(lib().bgtq_prefill_append(device.handle, ctypes.byref(desc), ctypes.byref(append)))


def prefill(device, desc) -> None:
    check(lib().bgtq_prefill(device.handle, ctypes.byref(desc)))


# ---- paged cache and packed prompts
#
# These wrappers check what the library cannot see (device, dtype, shape) and
# cost a call of a few microseconds: one read of each tensor property, one
# structure built at once.

_CODES: dict = {}  # torch dtype -> BGTQ_DTYPE_* of rows outside a pool


def _codes():
    if not _CODES:
        import torch
        _CODES.update({torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16})
    return _CODES


def _need(ok, message):
    if not ok:
        raise RangeError(message)


def _dense(index, name, t, dtype, dims):
    """t's strides, checked: a tensor on GPU `index` of the dtype (its name) with `dims` dimensions, the last one dense."""
    if t.get_device() != index or str(t.dtype) != "torch." + dtype or t.dim() != dims:
        raise RangeError(f"{name} must be a {dtype} tensor of {dims} dimensions on the context's device")
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] > 1:
        raise RangeError(f"{name}'s last dimension must be dense")
    return st


def _strides2(t, st):
    """The strides of t's first two dimensions, 0 for one of a single entry."""
    n = t.shape
    return (st[0] if n[0] > 1 else 0, st[1] if n[1] > 1 else 0)


class Pages:
    """A pool of pages (bgtq_pages) over device tensors; holds them."""

    def __init__(self, struct, device_index, held):
        self.struct, self.device_index, self.held = struct, device_index, held
        self.kv_heads, self.dim = struct.kv_heads, struct.dim
        self.ref = ctypes.byref(struct)


def pages(*, page_tokens, v, v_scales=None, tables=None, packed=None, norms=None, k_f16=None) -> Pages:
    """A pool of pages over tensors whose first two dimensions are (page, KV head): v [.., .., page_tokens, dim]
    float16, or int8 with v_scales [.., .., page_tokens] float16; K either k_f16 [.., .., page_tokens, dim]
    float16, or packed [.., .., bytes] uint8 and norms [.., .., scales] float16 (at least page_tokens rows of
    each head's row bytes and norm stride) with the heads' tables."""
    _need((packed is None) == (norms is None) and (packed is None) != (k_f16 is None), "K pages are packed and norms, or k_f16")
    index = v.get_device()
    _need(index >= 0, "pages must lie on a GPU")
    q8 = v_scales is not None
    g = _lib.Pages()

    def put(name, t, dtype, dims):
        st = _dense(index, name, t, dtype, dims)
        _need(t.shape[:2] == v.shape[:2], f"{name} must have the pool's pages and heads")
        if dims == 4:
            _need(t.shape == v.shape and (t.shape[2] == 1 or st[2] == t.shape[3]), f"{name} must hold page_tokens adjacent rows per page and head")
        two = _strides2(t, st)
        field = name if name != "k_f16" else "k"
        setattr(g, name, t.data_ptr())
        setattr(g, field + "_page_stride", two[0])
        setattr(g, field + "_head_stride", two[1])
    put("v", v, "int8" if q8 else "float16", 4)
    n, heads, rows, dim = v.shape
    _need(rows == page_tokens, "v must hold page_tokens rows per page and head")
    g.kv_heads, g.dim, g.page_tokens, g.pages = heads, dim, page_tokens, n
    g.v_format = _lib.DTYPE_Q8 if q8 else _lib.DTYPE_F16
    if q8:
        put("v_scales", v_scales, "float16", 3)
        _need(v_scales.shape[2] == rows, "v_scales must hold a scale per row")
    if k_f16 is not None:
        g.key_format = _lib.KEYS_FP16
        put("k_f16", k_f16, "float16", 4)
    else:
        _need(tables and len(tables) == heads, "packed K pages need the tables of every KV head")
        g.key_format = _lib.KEYS_PACKED
        put("packed", packed, "uint8", 3)
        put("norms", norms, "float16", 3)
        for i, t in enumerate(tables):
            g.tables[i] = t.handle.value if hasattr(t.handle, "value") else t.handle
        _need(packed.shape[2] >= rows * max(t.info["row_bytes"] for t in tables)
              and norms.shape[2] >= rows * max(t.info["norm_stride"] for t in tables),
              "packed and norms must hold page_tokens rows of every head")
    return Pages(g, index, (v, v_scales, tables, packed, norms, k_f16))


def _row_fields(index, name, t, shape):
    """(address, dtype, row stride, head stride) of K or V rows; zeros for none."""
    if t is None:
        return (None, 0, 0, 0)
    code = _codes().get(t.dtype)
    if code is None or t.get_device() != index or t.shape != shape:
        raise RangeError(f"{name} must be a [rows, KV heads, dim] tensor of float32, float16 or bfloat16 on the context's device")
    s = t.stride()
    if s[2] != 1:
        raise RangeError(f"{name}'s last dimension must be dense")
    return (t.data_ptr(), code, s[0] if shape[0] > 1 else 0, s[1] if shape[1] > 1 else 0)


def _paged_rows(device, pool, slots, k, v):
    index = device.index
    if pool.device_index != index:
        raise RangeError("the pool must lie on the context's device")
    _dense(index, "slots", slots, "int64", 1)
    n = slots.shape[0]
    shape = (n, pool.kv_heads, pool.dim)
    return _lib.PagedRows(n, slots.data_ptr(), *_row_fields(index, "k", k, shape), *_row_fields(index, "v", v, shape))


def paged_write(device, pool, slots, k, v) -> None:
    """bgtq_paged_write: rows k, v [n, Hkv, dim] (FP32, FP16 or BF16, any strides of the first two dimensions) into
    the slots [n] int64; slots outside the pool are skipped."""
    r = _paged_rows(device, pool, slots, k, v)
    if r.rows:
        check(lib().bgtq_paged_write(device.handle, pool.ref, ctypes.byref(r)))


def paged_read(device, pool, slots, k=None, v=None) -> None:
    """bgtq_paged_read: the slots' rows into k and / or v [n, Hkv, dim] (FP32, FP16 or BF16); rows of slots outside
    the pool stay as they are."""
    _need(k is not None or v is not None, "paged_read needs k or v")
    r = _paged_rows(device, pool, slots, k, v)
    if r.rows:
        check(lib().bgtq_paged_read(device.handle, pool.ref, ctypes.byref(r)))


# ---- head norms and position rotation

def rope_table(positions: int, dim: int, base: float, device="cuda"):
    """The rotation table [positions, dim] float32 of angles p base^(-2 i / dim) (src/model/kernels.wgsl's rope), from
    angles in 64 bits: a row's dim / 2 cosines, then as many sines."""
    import torch
    freq = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


class Rope:
    """A rotation (bgtq_rotation) over device tensors; holds them."""

    def __init__(self, struct, dim, device_index, held):
        self.struct, self.dim, self.device_index, self.held = struct, dim, device_index, held
        self.ref = ctypes.byref(struct)


def rope(*, table, q_norm=None, k_norm=None, eps=1e-6) -> Rope:
    """A rotation: table [positions, dim] float32 (see rope_table), and float32 [dim] weights of the norms of each head
    of the queries and of the keys (None: no norm)."""
    index = table.get_device()
    _need(index >= 0, "the table must lie on a GPU")
    _dense(index, "table", table, "float32", 2)
    _need(table.is_contiguous(), "the table must be contiguous")
    dim = table.shape[1]
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None:
            _dense(index, name, w, "float32", 1)
            _need(w.shape[0] == dim, f"{name} must hold a weight per dimension")
    return Rope(_lib.RotationDesc(_addr(table), table.shape[0], _addr(q_norm), _addr(k_norm), float(eps)), dim, index,
                (table, q_norm, k_norm))


def _head_rows(index, name, t, out, rows, dim):
    """bgtq_head_rows of t [rows, heads, dim] and where it goes (None: in place)."""
    shape, code = t.shape, _codes().get(t.dtype)
    if code is None or len(shape) != 3 or shape[0] != rows or shape[2] != dim or t.get_device() != index:
        raise RangeError(f"{name} must be a [rows, heads, dim] tensor of float32, float16 or bfloat16 on the context's device")
    s, src = t.stride(), t.data_ptr()
    o, dst = s, src
    if out is not None:
        if out.dtype != t.dtype or out.shape != shape or out.get_device() != index:
            raise RangeError(f"{name} and its output must agree in shape, dtype and device")
        o, dst = out.stride(), out.data_ptr()
    if s[2] != 1 or o[2] != 1:
        raise RangeError(f"{name}'s last dimension must be dense")
    heads = shape[1]
    rs, ro = (s[0], o[0]) if rows > 1 else (0, 0)
    hs, ho = (s[1], o[1]) if heads > 1 else (0, 0)
    return _lib.HeadRows(src, dst, heads, code, rs, hs, ro, ho)


def _positions(index, rope, positions):
    """The number of rows, checked."""
    if rope.device_index != index:
        raise RangeError("the rotation must lie on the context's device")
    _dense(index, "positions", positions, "int64", 1)
    return positions.shape[0]


def rotate(device, rope, positions, q=None, k=None, q_out=None, k_out=None) -> None:
    """bgtq_rotate: rows q [n, Hq, dim] and k [n, Hkv, dim] (FP32, FP16 or BF16, any strides of the first two
    dimensions) at positions [n] int64 normed and rotated into q_out and k_out (None: in place); rows whose position
    is none of the table's are left out."""
    index, dim = device.index, rope.dim
    n = _positions(index, rope, positions)
    _need(q is not None or k is not None, "rotate needs q or k")
    qr = None if q is None else ctypes.byref(_head_rows(index, "q", q, q_out, n, dim))
    kr = None if k is None else ctypes.byref(_head_rows(index, "k", k, k_out, n, dim))
    if n:
        check(lib().bgtq_rotate(device.handle, rope.ref, dim, n, positions.data_ptr(), qr, kr))


def paged_append(device, pool, slots, rope, positions, k, v, q=None, q_out=None) -> None:
    """bgtq_paged_append: rows k, v [n, Hkv, dim] of a step into the slots [n] int64, k normed and rotated to positions
    [n] int64 on the way, and the step's queries q [n, Hq, dim] (None: none) into q_out (None: in place). Rows of
    slots outside the pool, or of positions outside the table, are not written."""
    n = _positions(device.index, rope, positions)
    _need(pool.dim == rope.dim, "the pool's heads and the rotation must agree in dim")
    _need(k is not None and v is not None, "paged_append needs k and v")
    r = _paged_rows(device, pool, slots, k, v)
    _need(r.rows == n, "slots and positions must have an entry per row")
    queries = None if q is None else ctypes.byref(_head_rows(device.index, "q", q, q_out, n, rope.dim))
    if n:
        check(lib().bgtq_paged_append(device.handle, pool.ref, ctypes.byref(r), rope.ref, positions.data_ptr(), queries))


def _window(window, sinks):
    """bgtq_window of a window's tokens and sinks; None for no window (None or 0)."""
    if not window:
        _need(not sinks, "sinks need a window")
        return None
    _need(0 < window < 1 << 31 and 0 <= sinks <= 1 << 30, "window must be in 1..2^31 - 1, sinks in 0..2^30")
    return _lib.Window(int(window), int(sinks))


class PagedDecode:
    """A paged decode's descriptor with its pool and window; holds the tensors."""

    def __init__(self, pool, struct, held, window=None):
        self.pool, self.struct, self.held, self.ref = pool, struct, held, ctypes.byref(struct)
        self.window = None if window is None else ctypes.byref(window)


def paged_decode_desc(*, pages, q, out, lengths, page_table, max_length=None, splits=0, workspace=None,
                      q_rotated=False, window=None, sinks=0) -> PagedDecode:
    """bgtq_paged_decode_desc over device tensors: q, out [B, Hq, dim] FP32 contiguous, lengths [B] and
    page_table [B, pages per sequence] int32; max_length defaults to what the page table's rows hold. window (None
    or 0: none): the query sees its sequence's last `window` tokens and the first `sinks`."""
    index = pages.device_index
    for name, t in (("q", q), ("out", out)):
        _dense(index, name, t, "float32", 3)
        _need(t.is_contiguous() and t.shape == q.shape and t.shape[2] == pages.dim, "q and out must be contiguous [B, Hq, dim]")
    batch, heads = q.shape[:2]
    _dense(index, "lengths", lengths, "uint32" if str(lengths.dtype) == "torch.uint32" else "int32", 1)
    st = _dense(index, "page_table", page_table, "int32", 2)
    _need(lengths.shape[0] == batch and page_table.shape[0] == batch, "lengths and page_table must have a row per sequence")
    held_tokens = page_table.shape[1] * pages.struct.page_tokens
    tokens = held_tokens if max_length is None else int(max_length)
    _need(tokens <= held_tokens, "page_table rows hold fewer tokens than max_length")
    _need(workspace is None or (workspace.get_device() == index and workspace.is_contiguous()), "workspace must be contiguous on the pool's device")
    d = _lib.PagedDecodeDesc(batch, heads, q.data_ptr(), out.data_ptr(), lengths.data_ptr(), page_table.data_ptr(),
                             st[0] if batch > 1 else page_table.shape[1], tokens, int(splits),
                             None if workspace is None else workspace.data_ptr(),
                             0 if workspace is None else workspace.numel() * workspace.element_size(), int(bool(q_rotated)))
    return PagedDecode(pages, d, (q, out, lengths, page_table, workspace), _window(window, sinks))


def paged_decode_workspace_bytes(desc) -> int:
    n = ctypes.c_size_t(0)
    if desc.window is None:
        check(lib().bgtq_paged_decode_workspace_size(desc.pool.ref, desc.ref, ctypes.byref(n)))
    else:
        check(lib().bgtq_paged_decode_window_workspace_size(desc.pool.ref, desc.ref, desc.window, ctypes.byref(n)))
    return n.value


def paged_decode(device, desc) -> None:
    """bgtq_paged_decode, or with a window bgtq_paged_decode_window: decode attention over the descriptor's pages."""
    _need(desc.pool.device_index == device.index, "the pool must lie on the context's device")
    if desc.window is None:
        check(lib().bgtq_paged_decode(device.handle, desc.pool.ref, desc.ref))
    else:
        check(lib().bgtq_paged_decode_window(device.handle, desc.pool.ref, desc.ref, desc.window))


class PagedPrefill:
    """A chunk call's descriptor with its pool; holds the tensors."""

    def __init__(self, pool, struct, held):
        self.pool, self.struct, self.held, self.ref = pool, struct, held, ctypes.byref(struct)


def paged_prefill_desc(*, pages, q, out, offsets, lengths, page_table, max_length=None, scale=None, window=None, sinks=0,
                       workspace=None) -> PagedPrefill:
    """bgtq_paged_prefill_desc over device tensors: q, out [tokens, Hq, dim] FP16 or BF16 (any strides of the first two
    dimensions that are multiples of 8), the new rows of the sequences packed one after another at offsets
    [sequences + 1] int32; lengths [sequences] int32: the tokens of each with its new ones; page_table [sequences, pages
    per sequence] int32; max_length defaults to what its rows hold; scale to 1 / sqrt(dim); window (None or 0: none) and
    sinks as paged_decode_desc's."""
    index, dtype = pages.device_index, q.dtype
    code = _codes().get(dtype, _lib.DTYPE_F32)
    _need(code != _lib.DTYPE_F32 and q.dim() == 3 and q.shape[2] == pages.dim and offsets.shape[0] > 0,
          "q and out must be [tokens, Hq, dim] tensors of float16 or bfloat16; offsets has an entry more than sequences")
    fields = []
    for name, t in (("q", q), ("out", out)):
        if t.dtype != dtype or t.get_device() != index or t.shape != q.shape:
            raise RangeError("q and out must agree in shape, dtype and the pool's device")
        s = t.stride()
        _need(s[2] == 1, f"{name}'s last dimension must be dense")
        fields += (t.data_ptr() or None, s[0] if q.shape[0] > 1 else 0, s[1] if q.shape[1] > 1 else 0)
    _dense(index, "offsets", offsets, "int32", 1)
    _dense(index, "lengths", lengths, "uint32" if str(lengths.dtype) == "torch.uint32" else "int32", 1)
    st = _dense(index, "page_table", page_table, "int32", 2)
    sequences = offsets.shape[0] - 1
    _need(lengths.shape[0] == sequences and page_table.shape[0] == sequences, "lengths and page_table must have a row per sequence")
    held_tokens = page_table.shape[1] * pages.struct.page_tokens
    most = held_tokens if max_length is None else int(max_length)
    _need(most <= held_tokens, "page_table rows hold fewer tokens than max_length")
    _need(workspace is None or (workspace.get_device() == index and workspace.is_contiguous()), "workspace must be contiguous on the pool's device")
    _need(scale is None or ctypes.c_float(scale).value > 0, "scale must be positive in FP32")  # (0 stands for the default)
    w = _window(window, sinks)
    d = _lib.PagedPrefillDesc(q.shape[1], code, sequences, q.shape[0], offsets.data_ptr(), lengths.data_ptr(),
                              page_table.data_ptr(), st[0] if sequences > 1 else page_table.shape[1], most, *fields, scale or 0.0,
                              0 if w is None else w.window, 0 if w is None else w.sinks,
                              None if workspace is None else workspace.data_ptr(),
                              0 if workspace is None else workspace.numel() * workspace.element_size())
    return PagedPrefill(pages, d, (q, out, offsets, lengths, page_table, workspace))


def paged_prefill_workspace_bytes(desc) -> int:
    n = ctypes.c_size_t(0)
    check(lib().bgtq_paged_prefill_workspace_size(desc.pool.ref, desc.ref, ctypes.byref(n)))
    return n.value


def paged_prefill(device, desc) -> None:
    """bgtq_paged_prefill: attention of the descriptor's chunks of new tokens over its pages."""
    _need(desc.pool.device_index == device.index, "the pool must lie on the context's device")
    check(lib().bgtq_paged_prefill(device.handle, desc.pool.ref, desc.ref))


def prompt_attention(device, q, k, v, offsets, out, scale=None, window=None, sinks=0) -> None:
    """bgtq_prompt_attention: causal attention within each of the sequences packed in q, out [tokens, Hq, dim] and
    k, v [tokens, Hkv, dim] (FP16 or BF16, any strides of the first two dimensions that are multiples of 8);
    offsets [sequences + 1] int32; scale defaults to 1 / sqrt(dim). window (None or 0: none): a position sees the last
    `window` ones, its own among them, and its sequence's first `sinks` (bgtq_prompt_attention_window)."""
    index, dtype = device.index, q.dtype
    code = _codes().get(dtype, _lib.DTYPE_F32)
    _dense(index, "offsets", offsets, "int32", 1)
    _need(code != _lib.DTYPE_F32 and q.dim() == 3 and k.dim() == 3 and offsets.shape[0] > 0,
          "q, k, v and out must be 3-dimensional float16 or bfloat16 tensors; offsets has an entry more than sequences")
    tokens, heads, dim = shape = q.shape
    kv_shape = (tokens, k.shape[1], dim)
    fields = []
    for t, want in ((q, shape), (k, kv_shape), (v, kv_shape), (out, shape)):
        if t.dtype != dtype or t.get_device() != index or t.shape != want:
            raise RangeError("q and out, k and v must agree in shape, all in tokens, dim, dtype and device")
        s = t.stride()
        if s[2] != 1 and dim > 1:
            raise RangeError("the last dimension of q, k, v and out must be dense")
        fields += (t.data_ptr() or None, s[0] if tokens > 1 else 0, s[1] if want[1] > 1 else 0)
    _need(scale is None or ctypes.c_float(scale).value > 0, "scale must be positive in FP32")  # (0 stands for the default)
    d = _lib.PromptDesc(heads, kv_shape[1], dim, code, offsets.shape[0] - 1, tokens, offsets.data_ptr(), *fields, scale or 0.0)
    w = _window(window, sinks)
    if w is None:
        check(lib().bgtq_prompt_attention(device.handle, ctypes.byref(d)))
    else:
        check(lib().bgtq_prompt_attention_window(device.handle, ctypes.byref(d), ctypes.byref(w)))
