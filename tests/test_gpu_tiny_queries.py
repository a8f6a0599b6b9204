"""Queries down to the smallest FP32 numbers, on every contiguous attention path.

Their logits are nothing to a softmax: every output is the mean of the V rows that its
query sees, and none is a NaN. (The rotation and QK run on FP16 parts of the queries times
a power of two, which FP32 has to hold.)
"""
import numpy as np
import pytest

from conftest import REF
from test_gpu_prefill import Cache, _check
from test_gpu_prefill_append import _append, _chunk_rows

pytestmark = pytest.mark.gpu

SIZES = (0.0, 1e-45, 1e-39, 1e-36, 1e-30, 1e-20)


def _cache(device, layout, dim, batch, cap):
    from bgtq import BlockGTQParameters, calibrate, calibration
    if layout == "S":
        blobs = calibration.read(REF / "model")[2]
        params = [BlockGTQParameters.from_serialized(blobs[7 + h].config, blobs[7 + h].table) for h in range(2)]
        rb, ns = max(p.rowBytes for p in params), max(p.normStride for p in params)
        for p in params:
            p.rowBytes, p.normStride = rb, ns
    else:
        params = None if layout == "f16" else [{"A": calibrate.layout_a, "B": calibrate.layout_b}[layout](dim)] * 2
    return Cache(device, params=params, batch=batch, hkv=2, dim=dim, cap=cap, pad16=True, seed=3,
                 key_format="fp16" if layout == "f16" else "packed")


def _queries(size, *shape):
    import torch
    return torch.randn(shape, generator=torch.Generator().manual_seed(5)) * size


@pytest.mark.parametrize("layout,dim", [("A", 64), ("B", 64), ("B", 128), ("S", 64), ("f16", 64), ("f16", 128)])
@pytest.mark.parametrize("mode", ["decode", "append", "fp32 values", "rotated"])
def test_decode(device, layout, dim, mode):
    import torch
    from bgtq import batched
    if layout == "f16" and mode == "rotated":
        return
    lengths, G = [70, 900], 3
    cache = _cache(device, layout, dim, 2, 900)
    vd = cache.vd.float() if mode == "fp32 values" else cache.vd
    for size in SIZES:
        print(layout, dim, mode, size, flush=True)
        q, out = _queries(size, 2, 2 * G, dim).cuda(), torch.full((2, 2 * G, dim), float("nan"), device="cuda")
        kw = dict(batch=2, q_heads=2 * G, kv_heads=2, dim=dim, q=q, out=out, max_length=900, v=vd, v_seq_stride=vd.stride(0),
                  v_head_stride=vd.stride(1), lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                  v_dtype="f32" if mode == "fp32 values" else "f16", q_rotated=mode == "rotated", **cache.kw)
        ws = torch.zeros(batched.workspace_bytes(batched.decode_desc(**kw)), dtype=torch.uint8, device="cuda")
        desc = batched.decode_desc(workspace=ws, **kw)
        if mode == "append":  # the last token's rows, which the cache holds already
            last = [n - 1 for n in lengths]
            batched.decode_append(device, desc, batched.append_desc(k_new=cache.k[[0, 1], :, last].contiguous().cuda(),
                                                                    v_new=cache.v[[0, 1], :, last].contiguous().cuda()))
        else:
            batched.decode(device, desc)
        torch.cuda.synchronize()
        for b, n in enumerate(lengths):
            mean = cache.v[b, :, :n].double().mean(1).repeat_interleave(G, 0).numpy()
            _check(out[b].cpu().numpy(), mean, f"{layout} {dim} {mode} {size} T={n}")
    cache.destroy()


@pytest.mark.parametrize("layout,dim", [("A", 64), ("B", 64), ("B", 128), ("S", 64), ("f16", 64), ("f16", 128)])
@pytest.mark.parametrize("rows,append", [(5, False), (32, False), (300, False), (13, True)])
def test_prefill(device, layout, dim, rows, append):
    """Few rows (row-wise units), many (tiles), and the rows appended in the launch."""
    if layout == "f16" and append:
        return
    starts, cap, G = [0, 600], 900, 3
    cache = _cache(device, layout, dim, 2, cap)
    for size in SIZES:
        print(layout, dim, rows, append, size, flush=True)
        q = _queries(size, 2, rows, 2 * G, dim)
        got = (_append(device, cache, q, starts, cap, _chunk_rows(cache.k, starts, rows), _chunk_rows(cache.v, starts, rows))
               if append else cache.prefill(device, q, starts, cap))
        for b, s in enumerate(starts):
            v = cache.v[b, :, :s + rows].double().numpy()
            mean = (np.cumsum(v, 1) / np.arange(1, s + rows + 1)[:, None])[:, s:].transpose(1, 0, 2).repeat(G, 1)
            _check(got[b], mean, f"{layout} {dim} rows {rows} {size} start {s}")
    cache.destroy()
