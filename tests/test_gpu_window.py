"""Sliding windows with sinks: decode over pages, and prompts, against 64 bits with the tolerances of the same calls
without a window (test_gpu_paged, test_gpu_prompt); what a window hides is garbage, or not there at all."""
import numpy as np
import pytest

from test_gpu_paged import CASES, Pool, _check, _fill, _rows, _table
from test_gpu_prompt import U, _inputs, _offsets

pytestmark = pytest.mark.gpu

LENGTHS = [0, 1, 5, 31, 32, 33, 64, 97, 130, 200, 515, 1000, 0]
WINDOWS = [(1, 0), (1, 3), (2, 64), (31, 1), (32, 32), (33, 0), (64, 33), (100, 4), (300, 100), (999, 1), (5000, 7),
           (2 ** 31 - 1, 2 ** 30)]


def _seen(n, window, sinks):
    """The tokens that the newest of n sees."""
    t = np.arange(n)
    return t[(t >= n - window) | (t < sinks)]


def _decode(pool, q, lengths, table, window, sinks, splits=0, max_length=None, workspace=None):
    import torch
    from bgtq import batched
    out = torch.full_like(q, float("nan"))
    args = dict(pages=pool.handle, q=q, out=out, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                page_table=table, max_length=max_length, splits=splits, window=window, sinks=sinks)
    if workspace is None:
        workspace = torch.zeros(batched.paged_decode_workspace_bytes(batched.paged_decode_desc(**args)), dtype=torch.uint8, device="cuda")
    batched.paged_decode(pool.device, batched.paged_decode_desc(workspace=workspace, **args))
    return out


def _decode_reference(pool, oracle, q, lengths, table, window, sinks):
    """Attention in 64 bits over the visible tokens whose page is the pool's."""
    B, Hq, D = q.shape
    G, out, tab = Hq // pool.heads, np.zeros((B, Hq, D)), table.cpu().numpy().astype(np.int64)
    for h in range(pool.heads):
        for b, n in enumerate(lengths):
            t = _seen(n, window, sinks)
            page = tab[b, t // pool.page]
            at = (page * pool.page + t % pool.page)[(page >= 0) & (page < pool.pages)]
            if not at.size:
                continue
            s = q[b, h * G:(h + 1) * G].double().cpu().numpy() @ pool.k_rows(oracle, h, at)[0].T / np.sqrt(D)
            e = np.exp(s - s.max(-1, keepdims=True))
            out[b, h * G:(h + 1) * G] = e @ pool.v_rows(h, at).astype(np.float64) / e.sum(-1, keepdims=True)
    return out


@pytest.mark.parametrize("layout,v,dim,heads,page", CASES)
@pytest.mark.parametrize("G,splits", [(1, 0), (3, 3), (16, 0), (2, 60)])
def test_decode(device, oracle, layout, v, dim, heads, page, G, splits):
    """Only what is seen was ever written: the rest of its pages is garbage (NaN scales and rows), other pages are given back."""
    import torch
    from bgtq import batched
    rng = np.random.RandomState(G)
    q = _rows(len(LENGTHS), heads * G, dim, "float32", G, 3).cuda()
    for window, sinks in WINDOWS:
        print(layout, v, dim, heads, page, G, splits, window, sinks, flush=True)
        lengths = [int(n) for n in rng.permutation(LENGTHS)]
        pool = Pool(device, layout, v, dim, heads, sum(-(-n // page) for n in lengths) + 2, page, gap=32)
        table = _table(pool, lengths, rng)
        tab = table.cpu().numpy().astype(np.int64)
        seen = [_seen(n, window, sinks) for n in lengths]
        slots = np.concatenate([tab[b, t // page] * page + t % page for b, t in enumerate(seen)]).astype(np.int64)
        for b, t in enumerate(seen):
            held = np.unique(t // page)
            gone = np.setdiff1d(np.arange(table.shape[1]), held)
            table[b, torch.from_numpy(gone)] = -1
        k, val = _rows(len(slots), heads, dim, "float16", G, 1), _rows(len(slots), heads, dim, "float16", G, 2)
        batched.paged_write(device, pool.handle, torch.from_numpy(slots).cuda(), k.cuda(), val.cuda())
        out = _decode(pool, q, lengths, table, window, sinks, splits)
        torch.cuda.synchronize()
        _check(out, _decode_reference(pool, oracle, q, lengths, table, window, sinks), f"window {window} sinks {sinks}")
        assert bool((out[[b for b, n in enumerate(lengths) if n == 0]] == 0).all())
        pool.destroy()


@pytest.mark.parametrize("layout,v,dim,heads", [("B", "q8", 64, 2), ("f16", "f16", 128, 1), ("S", "q8", 64, 3)])
@pytest.mark.parametrize("batch", [1, 2, 63, 65, 200])
def test_decode_batches(device, oracle, layout, v, dim, heads, batch):
    """Long and short sequences share the workgroups by what they stream; lengths beyond max_length count as it;
    one workspace serves several windows; a window that hides nothing gives the bits of none."""
    import torch
    from bgtq import batched
    rng = np.random.RandomState(batch)
    longest = 6000 if batch < 3 else 2000
    lengths = [int(longest * ((i + 1) / batch) ** 2) for i in range(batch)]
    lengths = [int(n) for n in rng.permutation(lengths)]
    pool = Pool(device, layout, v, dim, heads, sum(-(-n // 128) for n in lengths) + 1, 128)
    _fill(pool, batch)
    table = _table(pool, lengths, rng, spare=longest // 128 + 1)
    q = _rows(batch, heads * 3, dim, "float32", batch, scale=1.5).cuda()
    out = torch.empty_like(q)
    size = max(batched.paged_decode_workspace_bytes(batched.paged_decode_desc(
        pages=pool.handle, q=q, out=out, lengths=torch.zeros(batch, dtype=torch.int32, device="cuda"), page_table=table, max_length=longest, window=w))
        for w in (1, 100, 1500, 5000, None))
    workspace = torch.zeros(size, dtype=torch.uint8, device="cuda")
    for window, sinks in ((1500, 4), (100, 70), (1, 0), (5000, 1)):
        print(layout, dim, batch, window, sinks, flush=True)
        got = _decode(pool, q, lengths, table, window, sinks, max_length=longest, workspace=workspace)
        _check(got, _decode_reference(pool, oracle, q, lengths, table, window, sinks), f"{window} {sinks}")
    short = [min(n, 300) for n in lengths]
    _check(_decode(pool, q, lengths, table, 90, 5, max_length=300, workspace=workspace),
           _decode_reference(pool, oracle, q, short, table, 90, 5), "clamped")
    args = dict(pages=pool.handle, q=q, out=out, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), page_table=table,
                max_length=longest, workspace=workspace)
    batched.paged_decode(device, batched.paged_decode_desc(**args))
    assert torch.equal(out, _decode(pool, q, lengths, table, longest, 0, max_length=longest, workspace=workspace))
    pool.destroy()


def test_decode_pages_that_are_none(device, oracle):
    """Table entries outside the pool among the visible tokens: those are left out."""
    import torch
    rng = np.random.RandomState(5)
    pool = Pool(device, "B", "f16", 64, 2, 40, 32)
    _fill(pool, 4)
    lengths = [400, 333, 96, 1000]
    table = torch.from_numpy(rng.randint(0, pool.pages, (4, 33)).astype(np.int32))
    table[0, ::2], table[1, 3:], table[2], table[3, rng.permutation(32)[:20]] = -1, pool.pages, -2 ** 31, 2 ** 31 - 1
    table = table.cuda()
    q = _rows(4, pool.heads * 3, 64, "float32", 1).cuda()
    for window, sinks in ((100, 40), (31, 0), (600, 1)):
        out = _decode(pool, q, lengths, table, window, sinks)
        torch.cuda.synchronize()
        _check(out, _decode_reference(pool, oracle, q, lengths, table, window, sinks))
        assert bool((out[2] == 0).all())
    pool.destroy()


def _prompt_check(out, x, lens, hq, hkv, dtype, window, sinks, first=0):
    """As test_gpu_prompt's, behind a window."""
    x, got, at = x.double().numpy(), out.double().cpu().numpy(), first
    d = x.shape[-1]
    for i, n in enumerate(lens):
        t = np.arange(n)
        seen = (t[None] <= t[:, None]) & ((t[None] > t[:, None] - window) | (t[None] < sinks))
        for h in range(hq if n else 0):
            kv = hq + h // (hq // hkv)
            s = np.where(seen, x[at:at + n, h] @ x[at:at + n, kv].T / np.sqrt(d), -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            v = x[at:at + n, kv + hkv]
            ref, size = p @ v, p @ np.abs(v)
            err, lim = np.abs(got[at:at + n, h] - ref), U[dtype] * (size + np.abs(ref)) * 1.001 + 2.0 ** -14 * size + 1e-6
            assert np.all(err <= lim), f"{window} {sinks} sequence {i} of {n}: worst {np.nanmax(err / lim):.2f}, {np.isnan(err).sum()} NaN"
        at += n


@pytest.mark.parametrize("dtype,dim", [("float16", 64), ("bfloat16", 64), ("float16", 128), ("bfloat16", 128)])
@pytest.mark.parametrize("hq,hkv,lens", [(1, 1, [1]), (9, 3, [32, 33, 63, 64, 65, 0, 129]), (4, 2, [700, 1, 300]), (2, 2, [5] * 70),
                                         (2, 1, [0, 1100, 0])])
def test_prompts(device, dtype, dim, hq, hkv, lens):
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    x = _inputs(sum(lens), hq, hkv, dim, dtype, len(lens) + hq)
    xd = x.cuda()
    for window, sinks in WINDOWS + [(65, 64), (128, 65), (127, 129), (257, 0), (448, 500)]:
        print(dtype, dim, hq, hkv, lens[:3], window, sinks, flush=True)
        out = torch.full((sum(lens), hq, dim), float("nan"), dtype=x.dtype, device="cuda")
        batched.prompt_attention(device, xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], _offsets(lens), out, window=window, sinks=sinks)
        torch.cuda.synchronize()
        _prompt_check(out, x, lens, hq, hkv, dtype, window, sinks)


def test_prompt_without_effect_and_twice(device):
    """A window as long as the prompts gives the bits of none; two calls give the same bits."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    lens = [900, 64, 333]
    x = _inputs(sum(lens), 4, 2, 64, "bfloat16", 1).cuda()
    outs = []
    for kw in (dict(), dict(window=900, sinks=3), dict(window=77, sinks=3), dict(window=77, sinks=3)):
        out = torch.empty((sum(lens), 4, 64), dtype=x.dtype, device="cuda")
        batched.prompt_attention(device, x[:, :4], x[:, 4:6], x[:, 6:], _offsets(lens), out, **kw)
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[2], outs[3]) and not torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("dtype,dim", [("float16", 64), ("bfloat16", 128)])
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
def test_prompt_non_finite_rows_reach_only_what_sees_them(device, dtype, dim, bad):
    """K and V rows of infinities or NaNs: rows that do not see them are as if they were zeros; V's reach who sees them."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    n, hq, window, sinks = 500, 2, 70, 5
    x = _inputs(n, hq, 1, dim, dtype, 3)
    rows = [2, 6, 63, 64, 130, 333]
    clean = x.clone()
    clean[rows, hq:] = 0
    x[rows, hq, ::3] = float(bad)      # K
    x[rows, hq + 1, 1::4] = float(bad)  # V
    out = torch.empty((n, hq, dim), dtype=x.dtype, device="cuda")
    want = torch.empty_like(out)
    for src, dst in ((x, out), (clean, want)):
        src = src.cuda()
        batched.prompt_attention(device, src[:, :hq], src[:, hq:hq + 1], src[:, hq + 1:], _offsets([n]), dst, window=window, sinks=sinks)
    torch.cuda.synchronize()
    t = torch.arange(n)
    sees = torch.zeros(n, dtype=torch.bool)
    for r in rows:
        sees |= (t >= r) & ((t < r + window) | (r < sinks))
    assert torch.equal(out[~sees], want[~sees]) and int((~sees).sum()) == 2  # (row 2 is a sink: all but two rows see it)
    only = x.clone()
    only[2] = clean[2]
    src = only.cuda()
    batched.prompt_attention(device, src[:, :hq], src[:, hq:hq + 1], src[:, hq + 1:], _offsets([n]), out, window=window, sinks=sinks)
    torch.cuda.synchronize()
    sees = torch.zeros(n, dtype=torch.bool)
    for r in rows[1:]:
        sees |= (t >= r) & (t < r + window)
    assert torch.equal(out[~sees], want[~sees]) and int((~sees).sum()) > 100
    assert bool((~out[sees][:, :, 1::4].isfinite()).any())


def test_captured(device, oracle):
    """A captured windowed decode and prompt replay over new lengths, tables and rows, eager calls between."""
    import torch
    from bgtq import batched
    rng = np.random.RandomState(1)
    pool = Pool(device, "B", "q8", 64, 2, 70, 32)
    _fill(pool, 1)
    q, out = _rows(3, 6, 64, "float32", 1).cuda(), torch.empty((3, 6, 64), device="cuda")
    lengths, table = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros((3, 32), dtype=torch.int32, device="cuda")
    args = dict(pages=pool.handle, q=q, out=out, lengths=lengths, page_table=table, max_length=1000, window=200, sinks=4)
    workspace = torch.zeros(batched.paged_decode_workspace_bytes(batched.paged_decode_desc(**args)), dtype=torch.uint8, device="cuda")
    desc = batched.paged_decode_desc(workspace=workspace, **args)
    x, pout = _inputs(300, 4, 2, 64, "float16", 1).cuda(), torch.empty((300, 4, 64), dtype=torch.float16, device="cuda")
    offsets = _offsets([100, 200])

    def both():
        batched.paged_decode(device, desc)
        batched.prompt_attention(device, x[:, :4], x[:, 4:6], x[:, 6:], offsets, pout, window=33, sinks=2)
    both()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        device.set_stream(torch.cuda.current_stream().cuda_stream)
        both()
    batched.bind_torch_stream(device)
    for seed in (3, 4, 5):
        lens = [int(n) for n in rng.randint(0, 1001, 3)]
        lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        table.copy_(torch.from_numpy(rng.randint(0, pool.pages, (3, 32)).astype(np.int32)))
        q.copy_(_rows(3, 6, 64, "float32", seed))
        x.copy_(_inputs(300, 4, 2, 64, "float16", seed))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, _decode_reference(pool, oracle, q, lens, table, 200, 4), f"replay {seed}")
        got, pgot = out.clone(), pout.clone()
        both()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(pgot, pout)
    pool.destroy()


def test_wrapper_refusals(device):
    import torch
    import bgtq
    from bgtq import batched
    batched.bind_torch_stream(device)
    x, offsets = _inputs(4, 2, 1, 64, "float16", 1).cuda(), _offsets([4])
    for kw in (dict(sinks=3), dict(window=-1), dict(window=1 << 31), dict(window=5, sinks=-1), dict(window=5, sinks=(1 << 30) + 1)):
        with pytest.raises(bgtq.RangeError):
            batched.prompt_attention(device, x[:, :2], x[:, 2:3], x[:, 3:], offsets, torch.empty_like(x[:, :2]), **kw)
    pool = Pool(device, "f16", "f16", 64, 1, 2, 32)
    q = torch.zeros((1, 1, 64), device="cuda")
    with pytest.raises(bgtq.RangeError):
        batched.paged_decode_desc(pages=pool.handle, q=q, out=q.clone(), lengths=torch.zeros(1, dtype=torch.int32, device="cuda"),
                                  page_table=torch.zeros((1, 2), dtype=torch.int32, device="cuda"), sinks=1)
