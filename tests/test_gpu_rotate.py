"""Head norms and position rotation, by themselves and on the way into pages.

A rotated value is two FP32 roundings (half a step, 2^-24, of the second product and
of the result), a normed input three more (its factor, and two products) and one of
the weight's product: together below 6 2^-24 of |x1| + |x2|, plus the half step of the
rows' type. Pages: the pool after an append equals, bit for bit, the one after rotating
into FP32 rows and writing those.
"""
import numpy as np
import pytest

from test_gpu_paged import CASES, HALF_STEP, Pool, _rows, _same_bits

pytestmark = pytest.mark.gpu


def _rope(dim, norm, positions=5000, seed=0):
    import torch
    from bgtq import batched
    g = torch.Generator().manual_seed(seed)
    w = [(1 + 0.3 * torch.randn(dim, generator=g)).cuda() if norm else None for _ in range(2)]
    return batched.rope(table=batched.rope_table(positions, dim, 1e5), q_norm=w[0], k_norm=w[1], eps=1e-5), w


def _reference(x, weight, table, positions, eps=1e-5):
    """(rotated rows, |x1| + |x2| of their pairs after the norm) in 64 bits."""
    x, half = x.double().cpu().numpy(), x.shape[-1] // 2
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.double().cpu().numpy()
    cs = table.double().cpu().numpy()[positions.cpu().numpy()][:, None]
    c, s, a, b = cs[..., :half], cs[..., half:], x[..., :half], x[..., half:]
    size = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.concatenate([size, size], -1)


def _check(got, x, weight, rope, positions, what=""):
    ref, size = _reference(x, weight, rope.held[0], positions)
    tiny = {"float32": 2.0 ** -149, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}[str(got.dtype)[6:]]
    lim = 6 * 2.0 ** -24 * size + HALF_STEP[str(got.dtype)[6:]] * np.abs(ref) * 1.001 + tiny
    err = np.abs(got.double().cpu().numpy() - ref)
    assert np.all(err <= lim), f"{what}: worst {np.nanmax(err / lim):.2f} of the limit"


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows,hq,hkv,norm", [(1, 9, 3, False), (1, 1, 1, True), (2, 14, 2, True), (37, 5, 8, False), (1001, 16, 4, True)])
def test_rotate(device, dtype, dim, rows, hq, hkv, norm):
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    rope, w = _rope(dim, norm)
    x = _rows(rows, hq + hkv, dim, dtype, 1).cuda()
    q, k = x[:, :hq], x[:, hq:]  # slices of one projection
    positions = torch.randint(0, 5000, (rows,), generator=torch.Generator().manual_seed(rows)).cuda()
    q_out, k_out = torch.empty((rows, hq, dim), dtype=x.dtype, device="cuda"), torch.empty((rows, hkv, dim), dtype=x.dtype, device="cuda")
    batched.rotate(device, rope, positions, q, k, q_out, k_out)
    torch.cuda.synchronize()
    _check(q_out, q, w[0], rope, positions, "q")
    _check(k_out, k, w[1], rope, positions, "k")
    # one of the two alone, and in place: the same bits
    alone = torch.empty_like(k_out)
    batched.rotate(device, rope, positions, k=k, k_out=alone)
    batched.rotate(device, rope, positions, q=q, k=k)
    torch.cuda.synchronize()
    assert torch.equal(alone, k_out) and torch.equal(q, q_out) and torch.equal(k, k_out)


def test_unaligned_strided_and_left_out(device):
    """Rows at odd strides and addresses; rows of positions outside the table, left as they were."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    for dtype in ("float32", "float16", "bfloat16"):
        for dim in (64, 128):
            rope, w = _rope(dim, True, positions=100)
            n, heads = 53, 3
            flat = _rows(1, 1, 2 * n * (heads * (dim + 3) + 5) + 7, dtype, 2).cuda().view(-1)
            step = heads * (dim + 3) + 5
            view = flat[1:1 + n * step].view(n, step)[:, :heads * (dim + 3)].unflatten(1, (heads, dim + 3))[..., 1:dim + 1]
            dst = flat[n * step + 3:n * step + 3 + n * step].view(n, step)[:, 2:2 + heads * (dim + 3)].unflatten(1, (heads, dim + 3))[..., :dim]
            positions = torch.randint(0, 100, (n,), generator=torch.Generator().manual_seed(3)).cuda()
            positions[::7] = torch.tensor([-1, 100, 1 << 40, -(1 << 62), 99, 0, 101, -5], device="cuda")
            before = flat.clone()
            batched.rotate(device, rope, positions, q=view, q_out=dst)
            torch.cuda.synchronize()
            ok = (positions >= 0) & (positions < 100)
            _check(dst[ok], view[ok], w[0], rope, positions[ok], dtype)
            flat_rows = dst.clone()
            dst[ok] = before[n * step + 3:n * step + 3 + n * step].view(n, step)[:, 2:2 + heads * (dim + 3)].unflatten(1, (heads, dim + 3))[..., :dim][ok]
            assert torch.equal(flat, before), "nothing else is written"
            assert flat_rows.shape == dst.shape


def test_many_heads(device):
    """More items in a few rows than a workgroup's run of 65536 holds."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    rope, w = _rope(64, True)
    for rows, heads in ((3, 5000), (2, 40000), (70, 1500)):
        x = _rows(rows, heads, 64, "bfloat16", 5).cuda()
        positions, out = torch.arange(rows, device="cuda") * 70, torch.empty_like(x)
        batched.rotate(device, rope, positions, q=x, q_out=out)
        torch.cuda.synchronize()
        _check(out, x, w[0], rope, positions, f"{rows} rows of {heads} heads")


def test_append_of_mixed_types(device):
    """K, V and queries each of a type of its own."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    rope, w = _rope(64, True)
    for layout, rows in (("B", 5), ("B", 9000), ("f16", 300)):
        one, two = (Pool(device, layout, "q8", 64, 2, rows // 4096 + 2, 4096) for _ in range(2))
        k, v, q = _rows(rows, 2, 64, "float32", 1).cuda(), _rows(rows, 2, 64, "float16", 2).cuda(), _rows(rows, 6, 64, "bfloat16", 3).cuda()
        slots, positions = torch.arange(rows, device="cuda") + 7, torch.arange(rows, device="cuda") % 5000
        q_out, k32 = torch.empty_like(q), torch.empty_like(k)
        batched.paged_append(device, one.handle, slots, rope, positions, k, v, q, q_out)
        batched.rotate(device, rope, positions, k=k, k_out=k32)
        batched.paged_write(device, two.handle, slots, k32, v)
        torch.cuda.synchronize()
        _check(q_out, q, w[0], rope, positions, "q")
        for a, b in zip(one.snapshot(), two.snapshot()):
            assert a is None or _same_bits(a, b)
        one.destroy()
        two.destroy()


def test_infinities_and_zero_rows(device):
    """A row of zeros stays zero under a norm; an infinity reaches its pair, NaN only where arithmetic makes one."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    rope, _ = _rope(64, True)
    x = torch.zeros((3, 1, 64), device="cuda")
    x[1, 0, 5] = float("inf")
    x[2, 0, 5], x[2, 0, 9] = 65504.0, 1e-30
    positions = torch.tensor([7, 8, 9], device="cuda")
    plain = batched.rope(table=rope.held[0])
    out, normed = torch.empty_like(x), torch.empty_like(x)
    batched.rotate(device, plain, positions, q=x, q_out=out)
    batched.rotate(device, rope, positions, q=x, q_out=normed)
    torch.cuda.synchronize()
    assert out[1, 0, [5, 37]].isinf().all() and out[1].isfinite().sum() == 62
    assert torch.equal(normed[0], torch.zeros_like(normed[0])) and normed[2].isfinite().all()


@pytest.mark.parametrize("layout,v,dim,heads,page", CASES)
@pytest.mark.parametrize("rows,dtype,norm", [(1, "float32", False), (2, "bfloat16", True), (301, "float16", True), (5000, "float32", True),
                                             (9001, "bfloat16", False), (8999, "float16", True)])
def test_append_equals_rotate_then_write(device, layout, v, dim, heads, page, rows, dtype, norm):
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    print(layout, v, dim, heads, page, rows, dtype, norm, flush=True)
    hq, pages = 2 * heads, -(-rows // page) + 2
    rope, w = _rope(dim, norm)
    x = _rows(rows, hq + 2 * heads, dim, dtype, rows, scale=2.0).cuda()
    q, k, vv = x[:, :hq], x[:, hq:hq + heads], x[:, hq + heads:]
    g = torch.Generator().manual_seed(rows)
    slots = torch.arange(page + 1, page + 1 + rows) if rows % 2 else torch.randperm(pages * page, generator=g)[:rows]
    positions = torch.randint(0, 5000, (rows,), generator=g)
    if rows > 8:
        slots[3], positions[5], positions[6], slots[6] = -1, -1, 5000, pages * page
    slots, positions = slots.cuda(), positions.cuda()
    one, two = (Pool(device, layout, v, dim, heads, pages, page, gap=16) for _ in range(2))
    q_out = torch.full((rows, hq, dim), 7.0, dtype=x.dtype, device="cuda")
    batched.paged_append(device, one.handle, slots, rope, positions, k, vv, q, q_out)
    want_q, k32 = torch.full_like(q_out, 7.0), k.float().clone()
    batched.rotate(device, rope, positions, q, k32, want_q)
    outside = (positions < 0) | (positions >= 5000)
    batched.paged_write(device, two.handle, torch.where(outside, -1, slots), k32, vv)
    torch.cuda.synchronize()
    assert torch.equal(q_out, want_q)
    for name, a, b in zip(("v", "v_scales", "packed", "norms", "k"), one.snapshot(), two.snapshot()):
        assert a is None or _same_bits(a, b), name
    # without queries
    three = Pool(device, layout, v, dim, heads, pages, page, gap=16)
    batched.paged_append(device, three.handle, slots, rope, positions, k, vv)
    torch.cuda.synchronize()
    for a, b in zip(three.snapshot(), two.snapshot()):
        assert a is None or _same_bits(a, b)
    for p in (one, two, three):
        p.destroy()


@pytest.mark.parametrize("rows,bad", [(40, "inf"), (8200, "nan"), (8200, "-inf")])
@pytest.mark.parametrize("layout,dim", [("S", 64), ("B", 128)])
def test_append_of_non_finite_rows(device, rows, bad, layout, dim):
    """Rows with infinities or NaNs (which reach a norm's whole row) enter as rotated FP32 rows do."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    heads = 2
    for norm in (False, True):
        rope, _ = _rope(dim, norm)
        x = _rows(rows, 2 * heads, dim, "float32", 5).cuda()
        x[::9, 0, 3] = float(bad)
        x[1::50] = 0.0
        positions = torch.arange(rows, device="cuda") % 5000
        slots, pages = torch.arange(rows, device="cuda"), -(-rows // 64)
        one, two = (Pool(device, layout, "q8", dim, heads, pages, 64) for _ in range(2))
        batched.paged_append(device, one.handle, slots, rope, positions, x[:, :heads], x[:, heads:])
        k32 = x[:, :heads].clone()
        batched.rotate(device, rope, positions, k=k32)
        batched.paged_write(device, two.handle, slots, k32, x[:, heads:])
        torch.cuda.synchronize()
        for name, a, b in zip(("v", "v_scales", "packed", "norms", "k"), one.snapshot(), two.snapshot()):
            assert a is None or _same_bits(a, b), name
        one.destroy()
        two.destroy()


def test_append_captured_and_on_another_stream(device):
    """A captured append replays over new rows, slots and positions, with eager calls on another stream between."""
    import torch
    import bgtq
    from bgtq import batched
    n, heads, dim = 70, 3, 64
    rope, w = _rope(dim, True)
    pool, other = (Pool(device, "S", "q8", dim, heads, 8, 64) for _ in range(2))
    x, slots = _rows(n, 4 * heads, dim, "bfloat16", 1).cuda(), torch.arange(n, device="cuda")
    positions, q_out = torch.arange(n, device="cuda"), torch.empty((n, 2 * heads, dim), dtype=torch.bfloat16, device="cuda")
    call = lambda p, out: batched.paged_append(device, p.handle, slots, rope, positions, x[:, 2 * heads:3 * heads], x[:, 3 * heads:],  # noqa: E731
                                               x[:, :2 * heads], out)
    call(pool, q_out)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        device.set_stream(torch.cuda.current_stream().cuda_stream)
        call(pool, q_out)
    batched.bind_torch_stream(device)
    eager = bgtq.Device(0)
    for seed in (2, 3, 4):
        x.copy_(_rows(n, 4 * heads, dim, "bfloat16", seed))
        positions.copy_(torch.randperm(5000, generator=torch.Generator().manual_seed(seed))[:n])
        slots.copy_(torch.randperm(8 * 64, generator=torch.Generator().manual_seed(seed))[:n])
        for t, u in zip(pool.snapshot(), (other.v, other.v_scales, other.packed, other.norms)):
            u.copy_(t)
        want = torch.empty_like(q_out)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            batched.bind_torch_stream(eager)
            batched.paged_append(eager, other.handle, slots, rope, positions, x[:, 2 * heads:3 * heads], x[:, 3 * heads:], x[:, :2 * heads], want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q_out, want)
        for a, b in zip(pool.snapshot(), other.snapshot()):
            assert a is None or _same_bits(a, b)
    for p in (pool, other):
        p.destroy()
    eager.destroy()


def test_wrapper_refusals(device):
    import torch
    import bgtq
    from bgtq import batched
    batched.bind_torch_stream(device)
    table = batched.rope_table(10, 64, 1e4)
    rope = batched.rope(table=table)
    q, pos = torch.zeros((2, 3, 64), device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for bad in (dict(table=table.cpu()), dict(table=table.half()), dict(table=table[:, :63]), dict(table=table.T),
                dict(table=table, q_norm=torch.ones(63, device="cuda")), dict(table=table, k_norm=torch.ones(64, dtype=torch.float16, device="cuda"))):
        with pytest.raises(bgtq.RangeError):
            batched.rope(**bad)
    for args, kw in (((pos,), {}), ((pos.int(), q), {}), ((pos[:1], q), {}), ((pos, q[..., :32]), {}), ((pos, q.double()), {}),
                     ((pos, q.cpu()), {}), ((pos, q, None, q.half()), {}), ((pos, q.transpose(1, 2)), {}), ((pos, q[0]), {}),
                     ((pos, None, q), dict(k_out=q[:, :2]))):
        with pytest.raises(bgtq.RangeError):
            batched.rotate(device, rope, *args, **kw)
    with pytest.raises(bgtq.RangeError, match="eps"):
        batched.rotate(device, batched.rope(table=table, eps=-1.0), pos, q)
    batched.rotate(device, rope, pos[:0], q[:0])  # no rows: nothing to do
    pool = Pool(device, "f16", "f16", 64, 3, 2, 32)
    slots = torch.arange(2, device="cuda")
    for args in ((slots[:1], rope, pos, q, q), (slots, rope, pos[:1], q, q), (slots, rope, pos, q, None), (slots, rope, pos, q, q, q[:1]),
                 (slots, batched.rope(table=batched.rope_table(10, 128, 1e4)), pos, q, q)):
        with pytest.raises(bgtq.RangeError):
            batched.paged_append(device, pool.handle, *args)
