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


class PagedDecode:
    """A paged decode's descriptor with its pool; holds the tensors."""

    def __init__(self, pool, struct, held):
        self.pool, self.struct, self.held, self.ref = pool, struct, held, ctypes.byref(struct)


def paged_decode_desc(*, pages, q, out, lengths, page_table, max_length=None, splits=0, workspace=None,
                      q_rotated=False) -> PagedDecode:
    """bgtq_paged_decode_desc over device tensors: q, out [B, Hq, dim] FP32 contiguous, lengths [B] and
    page_table [B, pages per sequence] int32; max_length defaults to what the page table's rows hold."""
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
    return PagedDecode(pages, d, (q, out, lengths, page_table, workspace))


def paged_decode_workspace_bytes(desc) -> int:
    n = ctypes.c_size_t(0)
    check(lib().bgtq_paged_decode_workspace_size(desc.pool.ref, desc.ref, ctypes.byref(n)))
    return n.value


def paged_decode(device, desc) -> None:
    """bgtq_paged_decode: decode attention over the descriptor's pages."""
    _need(desc.pool.device_index == device.index, "the pool must lie on the context's device")
    check(lib().bgtq_paged_decode(device.handle, desc.pool.ref, desc.ref))


def prompt_attention(device, q, k, v, offsets, out, scale=None) -> None:
    """bgtq_prompt_attention: causal attention within each of the sequences packed in q, out [tokens, Hq, dim] and
    k, v [tokens, Hkv, dim] (FP16 or BF16, any strides of the first two dimensions that are multiples of 8);
    offsets [sequences + 1] int32; scale defaults to 1 / sqrt(dim)."""
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
    check(lib().bgtq_prompt_attention(device.handle, ctypes.byref(d)))
