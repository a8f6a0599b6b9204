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

def _strides2(t):
    """The strides of t's first two dimensions, 0 for those of one entry."""
    return [t.stride(i) if t.shape[i] > 1 else 0 for i in (0, 1)]


def _on(device, name, t, dtypes, dims):
    """t checked: a tensor on the device's GPU of one of the dtypes and `dims` dimensions, its last one dense."""
    if not t.is_cuda or (device is not None and t.device.index != device.index):
        raise RangeError(f"{name} must lie on the context's device")
    if str(t.dtype)[6:] not in dtypes:
        raise RangeError(f"{name} must be of {' or '.join(dtypes)}")
    if t.dim() != dims or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise RangeError(f"{name} must have {dims} dimensions, the last one dense")
    return t


_ROWS = {"float32": _lib.DTYPE_F32, "float16": _lib.DTYPE_F16, "bfloat16": _lib.DTYPE_BF16}


class Pages:
    """A pool of pages (bgtq_pages) over device tensors; holds them."""

    def __init__(self, struct, device_index, held):
        self.struct, self.device_index, self.held = struct, device_index, held
        self.kv_heads, self.dim = struct.kv_heads, struct.dim


def pages(*, page_tokens, v, v_scales=None, tables=None, packed=None, norms=None, k_f16=None) -> Pages:
    """A pool of pages over tensors whose first two dimensions are (page, KV head): v [.., .., page_tokens, dim]
    float16, or int8 with v_scales [.., .., page_tokens] float16; K either k_f16 [.., .., page_tokens, dim]
    float16, or packed [.., .., bytes] uint8 and norms [.., .., scales] float16 (at least page_tokens rows of
    each head's row bytes and norm stride) with the heads' tables."""
    g = _lib.Pages()
    _on(None, "v", v, ("float16", "int8"), 4)
    n, heads, rows, dim = v.shape
    if rows != page_tokens or (rows > 1 and v.stride(2) != dim):
        raise RangeError("v must hold page_tokens adjacent rows per page and head")
    if (packed is None) == (k_f16 is None):
        raise RangeError("K pages are either packed or FP16")
    if (v.dtype.itemsize == 1) != (v_scales is not None):
        raise RangeError("8-bit V pages have scales, FP16 V pages have none")
    g.kv_heads, g.dim, g.page_tokens, g.pages = heads, dim, page_tokens, n
    g.v_format = _lib.DTYPE_F16 if v_scales is None else _lib.DTYPE_Q8
    g.v, g.v_page_stride, g.v_head_stride = v.data_ptr(), *_strides2(v)
    held = [v, v_scales, tables, packed, norms, k_f16]
    arrays = [("v", v, v.shape)]
    if v_scales is not None:
        _on(None, "v_scales", v_scales, ("float16",), 3)
        g.v_scales, g.v_scales_page_stride, g.v_scales_head_stride = v_scales.data_ptr(), *_strides2(v_scales)
        arrays.append(("v_scales", v_scales, (n, heads, rows)))
    if k_f16 is not None:
        _on(None, "k_f16", k_f16, ("float16",), 4)
        if k_f16.stride(2) != dim and rows > 1:
            raise RangeError("k_f16 must hold page_tokens adjacent rows per page and head")
        g.key_format = _lib.KEYS_FP16
        g.k_f16, g.k_page_stride, g.k_head_stride = k_f16.data_ptr(), *_strides2(k_f16)
        arrays.append(("k_f16", k_f16, v.shape))
    else:
        _on(None, "packed", packed, ("uint8",), 3)
        _on(None, "norms", norms, ("float16",), 3)
        if not tables or len(tables) != heads:
            raise RangeError("packed K pages need the tables of every KV head")
        for i, t in enumerate(tables):
            g.tables[i] = t.handle.value if hasattr(t.handle, "value") else t.handle
        if (packed.shape[2] < rows * max(t.info["row_bytes"] for t in tables)
                or norms.shape[2] < rows * max(t.info["norm_stride"] for t in tables)):
            raise RangeError("packed and norms must hold page_tokens rows of every head")
        g.key_format = _lib.KEYS_PACKED
        g.packed, g.packed_page_stride, g.packed_head_stride = packed.data_ptr(), *_strides2(packed)
        g.norms, g.norms_page_stride, g.norms_head_stride = norms.data_ptr(), *_strides2(norms)
        arrays += [("packed", packed, (n, heads, packed.shape[2])), ("norms", norms, (n, heads, norms.shape[2]))]
    for name, t, shape in arrays:
        if tuple(t.shape) != tuple(shape) or t.device != v.device:
            raise RangeError(f"{name} must have the pool's pages, heads and device")
    return Pages(g, v.device.index, held)


def _paged_rows(device, pool, slots, k, v):
    if pool.device_index != device.index:
        raise RangeError("the pool must lie on the context's device")
    _on(device, "slots", slots, ("int64",), 1)
    r = _lib.PagedRows()
    r.rows, r.slots = slots.shape[0], slots.data_ptr()
    for name, t in (("k", k), ("v", v)):
        if t is None:
            continue
        _on(device, name, t, tuple(_ROWS), 3)
        if tuple(t.shape) != (slots.shape[0], pool.kv_heads, pool.dim):
            raise RangeError(f"{name} must be [rows, KV heads, dim]")
        setattr(r, name, t.data_ptr() or None)
        setattr(r, name + "_dtype", _ROWS[str(t.dtype)[6:]])
        setattr(r, name + "_row_stride", t.stride(0) if t.shape[0] > 1 else 0)
        setattr(r, name + "_head_stride", t.stride(1) if t.shape[1] > 1 else 0)
    return r


def paged_write(device, pool, slots, k, v) -> None:
    """bgtq_paged_write: rows k, v [n, Hkv, dim] (FP32, FP16 or BF16, any strides of the first two dimensions) into
    the slots [n] int64; slots outside the pool are skipped."""
    r = _paged_rows(device, pool, slots, k, v)
    if r.rows:
        check(lib().bgtq_paged_write(device.handle, ctypes.byref(pool.struct), ctypes.byref(r)))


def paged_read(device, pool, slots, k=None, v=None) -> None:
    """bgtq_paged_read: the slots' rows into k and / or v [n, Hkv, dim] (FP32, FP16 or BF16); rows of slots outside
    the pool stay as they are."""
    if k is None and v is None:
        raise RangeError("paged_read needs k or v")
    r = _paged_rows(device, pool, slots, k, v)
    if r.rows:
        check(lib().bgtq_paged_read(device.handle, ctypes.byref(pool.struct), ctypes.byref(r)))


class PagedDecode:
    """A paged decode's descriptor with its pool; holds the tensors."""

    def __init__(self, pool, struct, held):
        self.pool, self.struct, self.held = pool, struct, held


def paged_decode_desc(*, pages, q, out, lengths, page_table, max_length=None, splits=0, workspace=None,
                      q_rotated=False) -> PagedDecode:
    """bgtq_paged_decode_desc over device tensors: q, out [B, Hq, dim] FP32 contiguous, lengths [B] and
    page_table [B, pages per sequence] int32; max_length defaults to what the page table's rows hold."""
    d = _lib.PagedDecodeDesc()
    for name, t, types, dims in (("q", q, ("float32",), 3), ("out", out, ("float32",), 3),
                                 ("lengths", lengths, ("int32", "uint32"), 1), ("page_table", page_table, ("int32",), 2)):
        _on(None, name, t, types, dims)
        if t.device.index != pages.device_index:
            raise RangeError(f"{name} must lie on the pool's device")
    batch, heads, dim = q.shape
    if not q.is_contiguous() or not out.is_contiguous() or out.shape != q.shape or dim != pages.dim:
        raise RangeError("q and out must be contiguous [B, Hq, dim]")
    if lengths.shape[0] != batch or page_table.shape[0] != batch:
        raise RangeError("lengths and page_table must have a row per sequence")
    d.batch, d.q_heads, d.q, d.out = batch, heads, q.data_ptr(), out.data_ptr()
    d.lengths, d.page_table = lengths.data_ptr(), page_table.data_ptr()
    # (a row past the tensor's columns is none of the table's)
    d.page_table_stride = page_table.stride(0) if batch > 1 else page_table.shape[1]
    held_tokens = page_table.shape[1] * pages.struct.page_tokens
    if max_length is not None and max_length > held_tokens:
        raise RangeError("page_table rows hold fewer tokens than max_length")
    d.max_length, d.splits, d.q_rotated = int(held_tokens if max_length is None else max_length), int(splits), int(bool(q_rotated))
    if workspace is not None:
        if not workspace.is_cuda or workspace.device.index != pages.device_index or not workspace.is_contiguous():
            raise RangeError("workspace must be contiguous on the pool's device")
        d.workspace, d.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return PagedDecode(pages, d, [q, out, lengths, page_table, workspace])


def paged_decode_workspace_bytes(desc) -> int:
    n = ctypes.c_size_t(0)
    check(lib().bgtq_paged_decode_workspace_size(ctypes.byref(desc.pool.struct), ctypes.byref(desc.struct), ctypes.byref(n)))
    return n.value


def paged_decode(device, desc) -> None:
    """bgtq_paged_decode: decode attention over the descriptor's pages."""
    if desc.pool.device_index != device.index:
        raise RangeError("the pool must lie on the context's device")
    check(lib().bgtq_paged_decode(device.handle, ctypes.byref(desc.pool.struct), ctypes.byref(desc.struct)))


def prompt_attention(device, q, k, v, offsets, out, scale=None) -> None:
    """bgtq_prompt_attention: causal attention within each of the sequences packed in q, out [tokens, Hq, dim] and
    k, v [tokens, Hkv, dim] (FP16 or BF16, any strides of the first two dimensions that are multiples of 8);
    offsets [sequences + 1] int32; scale defaults to 1 / sqrt(dim)."""
    d = _lib.PromptDesc()
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out)):
        _on(device, name, t, ("float16", "bfloat16"), 3)
        if t.dtype != q.dtype or t.shape[0] != q.shape[0] or t.shape[2] != q.shape[2]:
            raise RangeError("q, k, v and out must agree in dtype, tokens and dim")
        setattr(d, name, t.data_ptr() or None)
        setattr(d, name + "_row_stride", t.stride(0) if t.shape[0] > 1 else 0)
        setattr(d, name + "_head_stride", t.stride(1) if t.shape[1] > 1 else 0)
    _on(device, "offsets", offsets, ("int32",), 1)
    if k.shape[1] != v.shape[1] or out.shape[1] != q.shape[1] or offsets.shape[0] < 1:
        raise RangeError("k and v, and q and out, must agree in heads; offsets has an entry more than sequences")
    d.q_heads, d.kv_heads, d.dim, d.dtype = q.shape[1], k.shape[1], q.shape[2], _ROWS[str(q.dtype)[6:]]
    d.sequences, d.tokens, d.offsets = offsets.shape[0] - 1, q.shape[0], offsets.data_ptr()
    if scale is not None:
        if not scale > 0:
            raise RangeError("scale must be positive")
        d.scale = scale
    check(lib().bgtq_prompt_attention(device.handle, ctypes.byref(d)))
