"""Causal attention over packed prompts against 64 bits.

An output may be off by the rounding of the probabilities (half a step u of the rows'
type, relative to each: u sum p |v|), its own rounding (u |ref|) and the FP32 logits
and sums (2^-14 of sum p |v| covers d 2^-24 times logits below 60).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _inputs(total, hq, hkv, dim, dtype, seed, scale=1.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((total, hq + 2 * hkv, dim), generator=g) * scale
    return x.to(getattr(torch, dtype))


def _offsets(lens, first=0):
    import torch
    return torch.tensor(np.concatenate([[first], first + np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _reference(q, k, v, scale):
    """(outputs, sum of p |v|) of one sequence [n, heads, d] in 64 bits."""
    n, hq, d = q.shape
    out, size = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    for h in range(hq if n else 0):
        kv = h // (hq // k.shape[1])
        s = np.where(np.tri(n, dtype=bool), q[:, h] @ k[:, kv].T * scale, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[:, h], size[:, h] = p @ v[:, kv], p @ np.abs(v[:, kv])
    return out, size


def _check(out, x, lens, hq, hkv, dtype, scale, first=0, what=""):
    x, got, at = x.double().numpy(), out.double().cpu().numpy(), first
    for i, n in enumerate(lens):
        q, k, v = x[at:at + n, :hq], x[at:at + n, hq:hq + hkv], x[at:at + n, hq + hkv:]
        ref, size = _reference(q, k, v, scale)
        err, lim = np.abs(got[at:at + n] - ref), U[dtype] * (size + np.abs(ref)) * 1.001 + 2.0 ** -14 * size + 1e-6
        assert np.all(err <= lim), f"{what} sequence {i} of {n}: worst {np.nanmax(err / lim):.2f} of the limit, {np.isnan(err).sum()} NaN"
        at += n


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hq,hkv,lens", [(1, 1, [1]), (3, 1, [2, 0, 31, 1]), (9, 3, [32, 33, 63, 64, 65, 0]), (4, 4, [127, 128, 129]),
                                         (14, 2, [300, 1, 257]), (2, 1, [0, 0, 1000, 0]), (2, 2, [5] * 70)])
def test_packed_prompts(device, dtype, dim, hq, hkv, lens):
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    print(dtype, dim, hq, hkv, lens, flush=True)
    x = _inputs(sum(lens), hq, hkv, dim, dtype, len(lens) + hq)
    xd = x.cuda()
    out = torch.full((sum(lens), hq, dim), float("nan"), dtype=x.dtype, device="cuda")
    batched.prompt_attention(device, xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], _offsets(lens), out)
    torch.cuda.synchronize()
    _check(out, x, lens, hq, hkv, dtype, 1 / np.sqrt(dim))


@pytest.mark.parametrize("dtype,dim", [("bfloat16", 64), ("float16", 128)])
def test_large_logits_and_scale(device, dtype, dim):
    """Logits of a few hundred (one key takes nearly all), a given scale, and equal logits."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    lens, hq, hkv = [200, 77], 4, 2
    for mult, scale in ((3.0, 0.25), (1.0, 1e-4), (0.0, None)):
        x = _inputs(sum(lens), hq, hkv, dim, dtype, 3)
        x[:, :hq] *= mult
        xd, out = x.cuda(), torch.empty((sum(lens), hq, dim), dtype=x.dtype, device="cuda")
        batched.prompt_attention(device, xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], _offsets(lens), out, scale=scale)
        torch.cuda.synchronize()
        _check(out, x, lens, hq, hkv, dtype, scale or 1 / np.sqrt(dim), what=f"scale {scale}")


def test_layouts_and_rows_of_no_sequence(device):
    """Heads-first and padded layouts; rows before the first and behind the last sequence stay as they were, whatever
    the inputs hold there."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    dtype, dim, hq, hkv, lens, total, first = "bfloat16", 64, 4, 2, [100, 37], 180, 9
    x = _inputs(total, hq, hkv, dim, dtype, 8)
    x[:first], x[first + 137:] = float("nan"), float("inf")
    q = torch.full((hq, total, dim + 8), float("nan"), dtype=x.dtype, device="cuda")
    q[:, :, :dim] = x[:, :hq].transpose(0, 1).cuda()
    k, v = x[:, hq:hq + hkv].transpose(0, 1).contiguous().cuda(), x[:, hq + hkv:].cuda()
    out = torch.full((hq, total, dim), 3.0, dtype=x.dtype, device="cuda")
    batched.prompt_attention(device, q[:, :, :dim].transpose(0, 1), k.transpose(0, 1), v, _offsets(lens, first), out.transpose(0, 1))
    torch.cuda.synchronize()
    _check(out.transpose(0, 1), x, lens, hq, hkv, dtype, 1 / 8, first)
    assert bool((out[:, :first] == 3).all()) and bool((out[:, first + 137:] == 3).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
def test_non_finite_rows_reach_only_what_sees_them(device, dim, bad):
    """A K or V row with infinities or NaNs changes nothing for the queries before it, nor for other sequences."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    lens, hq, hkv, dtype = [150, 90], 2, 1, "float16"
    x = _inputs(240, hq, hkv, dim, dtype, 4)
    clean = x.clone()
    x[100, hq + hkv:, 3::7] = float(bad)  # V of token 100
    x[120, hq:hq + hkv] = float(bad)      # K of token 120
    xd, out = x.cuda(), torch.empty((240, hq, dim), dtype=x.dtype, device="cuda")
    batched.prompt_attention(device, xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], _offsets(lens), out)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    ref, size = _reference(*(clean[:150].double().numpy()[:, a:b] for a, b in ((0, 2), (2, 3), (3, 4))), 1 / np.sqrt(dim))
    lim = U[dtype] * (size + np.abs(ref)) * 1.001 + 2.0 ** -14 * size + 1e-6
    assert np.all(np.abs(got[:100] - ref[:100]) <= lim[:100])
    hit = np.zeros(dim, bool)
    hit[3::7] = True
    assert np.all(np.abs(got[100:120] - ref[100:120])[..., ~hit] <= lim[100:120][..., ~hit])
    want = float(bad)
    seen = got[100:120][..., hit]
    assert np.all(np.isnan(seen)) if np.isnan(want) else np.all(seen == want)
    assert np.all(~np.isfinite(got[120:150]) | np.isnan(got[120:150])) or bad == "-inf" or bad == "inf"
    ref2, size2 = _reference(*(clean[150:].double().numpy()[:, a:b] for a, b in ((0, 2), (2, 3), (3, 4))), 1 / np.sqrt(dim))
    assert np.all(np.abs(got[150:] - ref2) <= U[dtype] * (size2 + np.abs(ref2)) * 1.001 + 2.0 ** -14 * size2 + 1e-6)


def test_lowest_values(device):
    """Keys of the type's lowest and highest values: logits beyond any exponent, weights 0 and 1, no NaN."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    x = _inputs(130, 2, 1, 64, "bfloat16", 2)
    x[:, :2] = x[:, :2].abs() + 0.1
    x[40, 2], x[70, 2] = -3e4, 3e4
    xd, out = x.cuda(), torch.empty((130, 2, 64), dtype=x.dtype, device="cuda")
    batched.prompt_attention(device, xd[:, :2], xd[:, 2:3], xd[:, 3:], _offsets([130]), out)
    torch.cuda.synchronize()
    _check(out[:70], x[:70], [70], 2, 1, "bfloat16", 1 / 8)
    assert torch.equal(out[70:], xd[70:71, 3:].expand(60, 2, 64))


@pytest.mark.parametrize("sequences", [2, 63, 64, 65, 129])
def test_every_tile_of_mixed_sequences(device, sequences):
    """Lengths from none to many tiles of 128 rows, in any order: each row of each sequence is written once, whatever
    order the tiles start in."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    dtype, dim, hq, hkv = "float16", 64, 2, 1
    lens = [int(n) for n in np.random.RandomState(sequences).permutation([(37 * i * i) % 700 if i % 5 else 0 for i in range(sequences)])]
    lens[sequences // 2] = 1300
    x = _inputs(sum(lens), hq, hkv, dim, dtype, sequences)
    xd, out = x.cuda(), torch.full((sum(lens), hq, dim), float("nan"), dtype=x.dtype, device="cuda")
    batched.prompt_attention(device, xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], _offsets(lens), out)
    torch.cuda.synchronize()
    _check(out, x, lens, hq, hkv, dtype, 1 / 8, what=f"{sequences} sequences")


def test_many_sequences_and_bad_offsets(device):
    """Thousands of short sequences (the search for a tile's sequence takes several rounds); offsets outside the rows
    are clamped to them."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    rng = np.random.RandomState(1)
    lens = [int(n) for n in rng.randint(0, 6, 9000)]
    x = _inputs(sum(lens), 1, 1, 64, "float16", 1)
    xd, out = x.cuda(), torch.empty((sum(lens), 1, 64), dtype=x.dtype, device="cuda")
    batched.prompt_attention(device, xd[:, :1], xd[:, 1:2], xd[:, 2:], _offsets(lens), out)
    torch.cuda.synchronize()
    _check(out, x, lens, 1, 1, "float16", 1 / 8)
    out2 = torch.full((300, 1, 64), 5.0, dtype=x.dtype, device="cuda")
    y = xd[:300]
    off = torch.tensor([-7, 100, 2 ** 30], dtype=torch.int32, device="cuda")  # sequences 0..99 and 100..299
    batched.prompt_attention(device, y[:, :1], y[:, 1:2], y[:, 2:], off, out2)
    torch.cuda.synchronize()
    _check(out2, x[:300], [100, 200], 1, 1, "float16", 1 / 8)


def test_captured_and_replayed(device):
    """A graph of the call serves other offsets and inputs."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    hq, hkv, dim, total = 6, 2, 64, 400
    xd = torch.zeros((total, hq + 2 * hkv, dim), dtype=torch.bfloat16, device="cuda")
    out, off = torch.empty((total, hq, dim), dtype=torch.bfloat16, device="cuda"), _offsets([total, 0, 0])
    args = (xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], off, out)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        device.set_stream(side.cuda_stream)
        batched.prompt_attention(device, *args)
    batched.bind_torch_stream(device)
    for i, lens in enumerate(([400, 0, 0], [100, 200, 100], [1, 0, 399], [133, 133, 134])):
        x = _inputs(total, hq, hkv, dim, "bfloat16", i)
        xd.copy_(x)
        off.copy_(_offsets(lens))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, x, lens, hq, hkv, "bfloat16", 1 / 8, what=f"replay {i}")
        replayed = out.clone()
        batched.prompt_attention(device, *args)
        torch.cuda.synchronize()
        assert torch.equal(replayed, out)


def test_wrapper_refusals(device):
    import torch
    import bgtq
    from bgtq import batched
    x = torch.zeros((8, 4, 64), dtype=torch.float16, device="cuda")
    off = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    ok = dict(q=x[:, :2], k=x[:, 2:3], v=x[:, 3:], offsets=off, out=x[:, :2].clone())
    for bad in (dict(q=x[:, :2].float()), dict(k=x[:4, 2:3]), dict(v=x[:, 3:].bfloat16()), dict(offsets=off.long()), dict(scale=-1.0),
                dict(scale=float("nan")), dict(q=x[:, :2, :32]), dict(out=x[:, :1].clone()), dict(k=x[:, :0], v=x[:, :0]),
                dict(q=torch.zeros((8, 2, 65), dtype=torch.float16, device="cuda")[:, :, :64])):
        with pytest.raises((bgtq.RangeError, bgtq.UnsupportedError)):
            batched.prompt_attention(device, **{**ok, **bad})
    batched.prompt_attention(device, x[:0, :2], x[:0, 2:3], x[:0, 3:], off[:1], x[:0, :2].clone())  # nothing to do


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sink,n", [(0, 9000), (4500, 9000), (17, 300), (None, 4096)])
def test_many_small_weights_beside_a_large_one(device, dtype, dim, sink, n):
    """A key whose weight is 2^15 to 2^30 times every other's and whose V is zero: the others are the output. (None:
    logits that rise by 3.5 in the log2 domain from block to block of 64 keys, V random.)

    A weight p (of a sum of 1) is off by half a step u p of its type, an FP16 one below 2^-25 of the largest by 2^-36:
    u (sum p |v| + |ref|) + 2^-36 (sum |v| + n |ref|) with the sum's; the logits (below 32) and sums in FP32 by
    2^-14 of the same; the output's own rounding is u |ref|, FP16 2^-25 where it is subnormal."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    print(dtype, dim, sink, n, flush=True)
    gaps = [15.0, 20.5, 21.5, 25.0, 28.0, 30.0]
    hq, typ, g = len(gaps), getattr(torch, dtype), torch.Generator().manual_seed(n + dim)
    q, k, v = (torch.zeros((n, h, dim)) for h in (hq, 1, 1))
    q[:, :, 0] = torch.tensor(gaps) * np.log(2.0) / 4
    k[:, 0, 0] = 0.02 * torch.randn(n, generator=g)
    if sink is None:
        q[:, :, 0] = 3.5 * np.log(2.0) * torch.linspace(0.4, 1, hq)
        k[:, 0, 0] = (torch.arange(n) // 64) % 8
        v.normal_(generator=g)
    else:
        v[:, 0] = 1 + 0.25 * torch.rand((n, dim), generator=g)
        k[sink, 0, 0], v[sink] = 4, 0
    q, k, v = q.to(typ), k.to(typ), v.to(typ)
    out = torch.empty((n, hq, dim), dtype=typ, device="cuda")
    batched.prompt_attention(device, q.cuda(), k.cuda(), v.cuda(), _offsets([n]), out, scale=1.0)
    torch.cuda.synchronize()
    q, k, v, got = (x.double().cpu().numpy() for x in (q, k, v, out))
    u = U[dtype]
    for row in sorted({0, 1, 16, 17, 18, 63, 64, 128, n // 2 - 1, n // 2, n // 2 + 1, 3 * n // 4, n - 1}):
        s = q[row, :, 0, None] * k[None, :row + 1, 0, 0]
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        x = v[:row + 1, 0]
        ref, size = p @ x, p @ np.abs(x)
        lim = (u + 2.0 ** -14) * (size + np.abs(ref)) + u * np.abs(ref) * 1.001
        if dtype == "float16":
            lim += 2.0 ** -36 * (np.abs(x).sum(0) + (row + 1) * np.abs(ref)) + 2.0 ** -25
        err = np.abs(got[row] - ref)
        assert np.all(err <= lim), f"row {row}: {np.max(err / lim):.1f} of the limit, heads {np.max(err / lim, -1).round(2)}"


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("where", ["k", "v", "both"])
def test_non_finite_rows_in_64_bits(device, dtype, dim, bad, where):
    """K and V rows with infinities or NaNs, seen in a diagonal block and in whole ones: NaNs, infinities and finite
    values are where the formula in 64 bits has them. Head 0's queries are positive, so that an infinite K row has
    infinite logits (minus infinity: weight 0); the other head's signs are mixed, its logits NaN."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    print(dtype, dim, bad, where, flush=True)
    n, hq, value = 330, 2, float(bad)
    x = _inputs(n, hq, 1, dim, dtype, 6)
    x[:, 0] = x[:, 0].abs() * 0.25 + 0.01
    if where != "k":
        x[10, 3, 3::7], x[140, 3, 5::11] = value, value
    if where != "v":
        x[200, 2] = value
    xd, out = x.cuda(), torch.empty((n, hq, dim), dtype=x.dtype, device="cuda")
    batched.prompt_attention(device, xd[:, :hq], xd[:, 2:3], xd[:, 3:], _offsets([n]), out)
    torch.cuda.synchronize()
    got, y = out.double().cpu().numpy(), x.double().numpy()
    for h in range(hq):
        for i in range(n):
            with np.errstate(invalid="ignore"):
                s = (y[i, h] * y[:i + 1, 2]).sum(-1) / np.sqrt(dim)
                p = np.exp(s - s.max())
                p /= p.sum()
                live = ~(p == 0)  # (a key of weight 0 adds nothing, whatever its V)
                ref, size = (p[live, None] * y[:i + 1, 3][live]).sum(0), (p[live, None] * np.abs(y[:i + 1, 3][live])).sum(0)
            assert np.array_equal(np.isnan(got[i, h]), np.isnan(ref)), f"head {h} query {i}"
            assert np.array_equal(np.isinf(got[i, h]), np.isinf(ref)), f"head {h} query {i}"
            f = np.isfinite(ref)
            assert np.array_equal(got[i, h][np.isinf(ref)], ref[np.isinf(ref)])
            lim = U[dtype] * (size[f] + 2 * np.abs(ref[f])) * 1.001 + 2.0 ** -14 * size[f] + 1e-6
            assert np.all(np.abs(got[i, h][f] - ref[f]) <= lim), f"head {h} query {i}"


def test_two_calls_give_the_same_bits(device):
    """No order of workgroups shows in the result."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    lens = [700, 33, 1, 257]
    for dtype, dim in (("float16", 64), ("bfloat16", 64), ("bfloat16", 128)):
        x = _inputs(sum(lens), 9, 3, dim, dtype, 2).cuda()
        outs = [torch.full((sum(lens), 9, dim), float(i), dtype=x.dtype, device="cuda") for i in range(4)]
        for o in outs:
            batched.prompt_attention(device, x[:, :9], x[:, 9:12], x[:, 12:], _offsets(lens), o)
        torch.cuda.synchronize()
        assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_scales_that_fp32_does_not_hold(device):
    """A scale that is 0 in FP32 is refused: it would stand for the default. The smallest that is none gives equal weights."""
    import torch
    import bgtq
    from bgtq import batched
    batched.bind_torch_stream(device)
    x = _inputs(70, 1, 1, 64, "bfloat16", 1).cuda()
    out = torch.empty((70, 1, 64), dtype=x.dtype, device="cuda")
    args = (x[:, :1], x[:, 1:2], x[:, 2:], _offsets([70]), out)
    for scale in (1e-46, 1e-300, 0.0, 1e39, 2.5e38):
        with pytest.raises(bgtq.RangeError):
            batched.prompt_attention(device, *args, scale=scale)
    batched.prompt_attention(device, *args, scale=1e-45)
    torch.cuda.synchronize()
    _check(out, x.cpu() * torch.tensor([0, 1, 1], dtype=x.dtype)[:, None], [70], 1, 1, "bfloat16", 1.0)


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_far_apart(device, dim):
    """The largest row stride: offsets past 2^32 bytes, rows of q, k, v and out side by side in one buffer."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    lens, hq, hkv, stride, dtype = [300, 1, 339], 2, 1, 1 << 22, "bfloat16"
    total = sum(lens)
    x = _inputs(total, hq, hkv, dim, dtype, 3)
    buf = torch.empty((total, stride), dtype=x.dtype, device="cuda")
    part = buf[:, :(2 * hq + 2 * hkv) * dim].unflatten(1, (2 * hq + 2 * hkv, dim))
    part[:, :hq + 2 * hkv] = x.cuda()
    out = part[:, hq + 2 * hkv:]
    out.fill_(float("nan"))
    batched.prompt_attention(device, part[:, :hq], part[:, hq:hq + hkv], part[:, hq + hkv:hq + 2 * hkv], _offsets(lens), out)
    torch.cuda.synchronize()
    _check(out, x, lens, hq, hkv, dtype, 1 / np.sqrt(dim))


@pytest.mark.parametrize("sequences", [64, 65, 200])
def test_many_sequences_captured(device, sequences):
    """A graph over many sequences serves other lengths, empty ones among them; rows of none stay as they were."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    hq, hkv, dim, total, dtype = 3, 1, 64, 5000, "float16"
    xd = torch.zeros((total, hq + 2 * hkv, dim), dtype=torch.float16, device="cuda")
    out, off = torch.empty((total, hq, dim), dtype=torch.float16, device="cuda"), torch.zeros(sequences + 1, dtype=torch.int32, device="cuda")
    args = (xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], off, out)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        device.set_stream(side.cuda_stream)
        batched.prompt_attention(device, *args)
    batched.bind_torch_stream(device)
    for step in range(3):
        rng = np.random.RandomState(step)
        lens = [int(n) for n in rng.multinomial(total - 100, rng.dirichlet(np.full(sequences, 0.2)))]
        x = _inputs(total, hq, hkv, dim, dtype, step)
        xd.copy_(x), off.copy_(_offsets(lens, 60)), out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, x, lens, hq, hkv, dtype, 1 / 8, 60, f"replay {step}")
        assert bool((out[:60] == 7).all()) and bool((out[-40:] == 7).all())
        replayed = out.clone()
        batched.prompt_attention(device, *args)
        torch.cuda.synchronize()
        assert torch.equal(replayed, out)
