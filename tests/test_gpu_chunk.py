"""Attention of chunks of new tokens over pages, against 64 bits over the rows that the pages hold.

An output may be off by its own rounding (half a step u of its type, of |ref|), that of the probabilities
to FP16 (2^-11 of sum p |v|), and its logits' errors: a logit off by e moves a weight by e^2e - 1, below 2.1 e of sum p |v|
for small e. FP32 sums: 2^-14 covers d 2^-24 times logits below 60. Packed K by BF16 rows: query, table entry and
product each rounded to FP16 (2^-11 each; 3.1 2^-11 of sum |q'_i| |k'_i| scale in the code domain); FP16 rows: pairs of
FP16 values, whose missing product and tails are below 2^-20 of the same. Over a whole output the errors are random: its
relative 2-norm error stays below u (BF16) and 2 u (FP16), where a rounding's own is at most 0.58 u.
"""
import numpy as np
import pytest

from test_gpu_paged import CASES, Pool, _fill, _rows, _table

pytestmark = pytest.mark.gpu

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _call(pool, q, new, lengths, table, window=0, sinks=0, max_length=None, scale=None, workspace=None, out=None, first=0):
    """Chunks of `new` rows each, packed from row `first` of q on."""
    import torch
    from bgtq import batched
    out = torch.full_like(q, float("nan")) if out is None else out
    args = dict(pages=pool.handle, q=q, out=out, offsets=torch.tensor(first + np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda"),
                lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), page_table=table, max_length=max_length,
                window=window, sinks=sinks, scale=scale)
    if workspace is None:
        workspace = torch.zeros(batched.paged_prefill_workspace_bytes(batched.paged_prefill_desc(**args)), dtype=torch.uint8, device="cuda")
    batched.paged_prefill(pool.device, batched.paged_prefill_desc(workspace=workspace, **args))
    return out


def _check(pool, oracle, q, out, new, lengths, table, window=0, sinks=0, scale=None, first=0, what=""):
    dtype, D = str(q.dtype)[6:], pool.dim
    scale = scale or 1 / np.sqrt(D)
    G, tab = q.shape[1] // pool.heads, table.cpu().numpy().astype(np.int64)
    qn, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    want = np.zeros_like(qn)
    at = first
    for b, (c, n) in enumerate(zip(new, lengths)):
        t = np.arange(n)
        page = tab[b, t // pool.page] if n else t
        ok = (page >= 0) & (page < pool.pages)
        t, slots = t[ok], (page * pool.page + np.arange(n) % pool.page)[ok]
        pos = n - c + np.arange(c)
        seen = t[None] <= pos[:, None]
        if window:
            seen &= (t[None] > pos[:, None] - window) | (t[None] < sinks)
        used = seen.any(0)  # (the others may be garbage)
        seen, t, slots = seen[:, used], t[used], slots[used]
        for h in range(pool.heads if c else 0):
            k, _ = pool.k_rows(oracle, h, slots)
            v = pool.v_rows(h, slots).astype(np.float64)
            if pool.k is None:
                p = pool.params[h]
                rot, perm = np.asarray(p.rotation, np.float64).reshape(D, D), np.asarray(p.permutation, np.int64)
                rows, norms = pool.k_bytes(h, slots)
                codes = oracle.unpack(rows, D, p.nibbleDims).astype(np.int64)
                cent = np.asarray(p.centroids, np.float64).reshape(D, -1)
                cs = np.abs(cent[np.arange(D), codes] * norms.astype(np.float64)[:, np.asarray(p.groupOf, np.int64)])
            for g in range(G):
                x = qn[at:at + c, h * G + g]
                s = np.where(seen, x @ k.T * scale, -np.inf)
                any_ = seen.any(1)
                w = np.where(seen, np.exp(s - np.where(any_, s.max(1, initial=-np.inf), 0)[:, None]), 0)
                w /= np.where(any_, w.sum(1), 1)[:, None]
                ref, size = w @ v, w @ np.abs(v)
                want[at:at + c, h * G + g] = ref
                e = np.zeros(c)
                if pool.k is None and len(t):
                    turned = np.abs(x[:, perm] @ rot.T)
                    e = np.where(seen, turned @ cs.T, 0).max(1) * scale * (3.1 * 2.0 ** -11 if dtype == "bfloat16" else 2.0 ** -20)
                lim = U[dtype] * np.abs(ref) * 1.001 + (2.0 ** -11 + 2.0 ** -14 + 2.1 * e)[:, None] * size + 1e-6
                err = np.abs(got[at:at + c, h * G + g] - ref)
                assert np.all(err <= lim), (f"{what} sequence {b} ({c} of {n}) head {h * G + g}: worst {np.nanmax(err / lim):.2f} of the limit, "
                                            f"{np.isnan(err).sum()} NaN")
        at += c
    rows = slice(first, at)
    off, norm = np.linalg.norm(got[rows] - want[rows]), np.linalg.norm(want[rows])
    assert off <= (1 if dtype == "bfloat16" else 2) * U[dtype] * norm + 1e-6, f"{what}: {off / norm:.2e} of the norm"


def _written(device, layout, v, dim, heads, page, lengths, rng, seed, spare=2):
    """A pool with the sequences' tokens alone written (the rest garbage), and its table."""
    import torch
    from bgtq import batched
    pool = Pool(device, layout, v, dim, heads, sum(-(-n // page) for n in lengths) + 2, page, gap=32)
    table = _table(pool, lengths, rng, spare)
    tab = table.cpu().numpy().astype(np.int64)
    slots = np.concatenate([tab[b, np.arange(n) // page] * page + np.arange(n) % page for b, n in enumerate(lengths)]).astype(np.int64)
    k, val = _rows(len(slots), heads, dim, "float16", seed, 1, scale=1.5), _rows(len(slots), heads, dim, "float16", seed, 2)
    batched.paged_write(device, pool.handle, torch.from_numpy(slots).cuda(), k.cuda(), val.cuda())
    return pool, table


# (new rows, tokens with them)
MIXED = [(1, 1), (1, 33), (0, 0), (5, 5), (0, 70), (2, 64), (17, 200), (1, 515), (40, 40), (33, 97), (130, 333)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("layout,v,dim,heads,page", CASES)
@pytest.mark.parametrize("G", [1, 3, 16])
def test_mixed_chunks(device, oracle, dtype, layout, v, dim, heads, page, G):
    import torch
    print(dtype, layout, v, dim, heads, page, G, flush=True)
    rng = np.random.RandomState(G)
    order = rng.permutation(len(MIXED))
    new, lengths = [MIXED[i][0] for i in order], [MIXED[i][1] for i in order]
    pool, table = _written(device, layout, v, dim, heads, page, lengths, rng, G)
    q = _rows(sum(new), heads * G, dim, dtype, G, 3).cuda()
    out = _call(pool, q, new, lengths, table)
    torch.cuda.synchronize()
    _check(pool, oracle, q, out, new, lengths, table)
    again = _call(pool, q, new, lengths, table)
    assert torch.equal(out, again), "two calls give the same bits"
    pool.destroy()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("layout,v,dim,heads,page", CASES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 3), (64, 64), (100, 33), (400, 1)])
def test_windows(device, oracle, dtype, layout, v, dim, heads, page, window, sinks):
    """Behind a window only what is seen by some row was ever written; other pages are given back."""
    import torch
    from bgtq import batched
    print(dtype, layout, v, dim, heads, page, window, sinks, flush=True)
    rng = np.random.RandomState(window)
    new, lengths = [c for c, _ in MIXED], [n for _, n in MIXED]
    pool = Pool(device, layout, v, dim, heads, sum(-(-n // page) for n in lengths) + 2, page, gap=32)
    table = _table(pool, lengths, rng)
    tab = table.cpu().numpy().astype(np.int64)
    slots = []
    for b, (c, n) in enumerate(MIXED):
        t = np.arange(n)
        t = t[(t > n - c - window) | (t < sinks)]
        slots.append(tab[b, t // page] * page + t % page)
        table[b, torch.from_numpy(np.setdiff1d(np.arange(table.shape[1]), np.unique(t // page)))] = -1
    slots = np.concatenate(slots).astype(np.int64)
    k, val = _rows(len(slots), heads, dim, "float16", 5, 1), _rows(len(slots), heads, dim, "float16", 5, 2)
    batched.paged_write(device, pool.handle, torch.from_numpy(slots).cuda(), k.cuda(), val.cuda())
    q = _rows(sum(new), heads * 2, dim, dtype, 1, 3).cuda()
    out = _call(pool, q, new, lengths, table, window, sinks)
    torch.cuda.synchronize()
    _check(pool, oracle, q, out, new, lengths, table, window, sinks)
    pool.destroy()


@pytest.mark.parametrize("dtype,layout,v,dim,heads", [("bfloat16", "B", "q8", 64, 2), ("float16", "S", "q8", 64, 3), ("bfloat16", "f16", "f16", 128, 2),
                                                      ("float16", "B", "f16", 128, 1)])
def test_long_histories(device, oracle, dtype, layout, v, dim, heads):
    """Few units and long histories: their tokens split over workgroups, wide and narrow units, one workspace for all."""
    import torch
    from bgtq import batched
    rng = np.random.RandomState(3)
    lengths = [6001, 40, 2500]
    pool, table = _written(device, layout, v, dim, heads, 64, lengths, rng, 2)
    G = 4
    workspace = torch.zeros(512 << 20, dtype=torch.uint8, device="cuda")
    for new in ([1, 1, 1], [300, 0, 0], [70, 40, 9], [8, 0, 8], [0, 0, 700]):
        for window, sinks in ((0, 0), (1100, 5)):
            print(layout, dim, new, window, flush=True)
            q = _rows(sum(new), heads * G, dim, dtype, sum(new), 3, scale=1.5).cuda()
            out = _call(pool, q, new, lengths, table, window, sinks, workspace=workspace)
            torch.cuda.synchronize()
            _check(pool, oracle, q, out, new, lengths, table, window, sinks, what=f"{new}")
    assert not workspace[:batched._lib.PAGED_PREFILL_COUNTER_BYTES].any()
    pool.destroy()


@pytest.mark.parametrize("layout,v,dim,heads,dtype", [("S", "q8", 64, 3, "float16"), ("B", "q8", 64, 2, "bfloat16"), ("f16", "q8", 128, 2, "bfloat16")])
@pytest.mark.parametrize("max_length", [1 << 18, 1 << 20])
def test_groups_of_sequences(device, oracle, layout, v, dim, heads, dtype, max_length):
    """Sequences that may be long take the rebuilt rows' workspace in turns."""
    import torch
    rng = np.random.RandomState(4)
    new, lengths = [c for c, _ in MIXED] * 2, [n for _, n in MIXED] * 2
    pool, table = _written(device, layout, v, dim, heads, 64, lengths, rng, 6, spare=max_length // 64)
    q = _rows(sum(new), heads * 3, dim, dtype, 4, 3).cuda()
    for window, sinks in ((0, 0), (50, 3)):
        print(layout, max_length, window, flush=True)
        out = _call(pool, q, new, lengths, table, window, sinks, max_length=max_length)
        torch.cuda.synchronize()
        _check(pool, oracle, q, out, new, lengths, table, window, sinks)
    pool.destroy()


def test_two_rounds_of_items(device, oracle):
    """100 equal units on 256 workgroups: two splits each leave 56 idle, five are two rounds."""
    import torch
    rng = np.random.RandomState(7)
    pool, table = _written(device, "B", "q8", 128, 1, 64, [6500], rng, 5)
    q = _rows(1600, 16, 128, "float16", 2, 3).cuda()
    out = _call(pool, q, [1600], [6500], table)
    torch.cuda.synchronize()
    _check(pool, oracle, q, out, [1600], [6500], table)
    pool.destroy()


@pytest.mark.parametrize("new", [1, 30, 400])
def test_a_query_of_nans(device, oracle, new):
    """Its head's output is NaN, whether its tokens are split or not. The others' keep their limits (not their bits:
    32 columns raise their maxima together, and FP16 probabilities are rounded relative to those)."""
    import torch
    rng = np.random.RandomState(8)
    for layout, dim, dtype in (("f16", 64, "bfloat16"), ("B", 128, "bfloat16"), ("S", 64, "float16")):
        heads = 3 if layout == "S" else 1
        for n in (400, 5000):
            pool, table = _written(device, layout, "q8", dim, heads, 64, [n], rng, 5)
            q = _rows(new, 2 * heads, dim, dtype, 2, 3).cuda()
            bad = q.clone()
            bad[new // 2, 1, 3] = float("nan")
            out = _call(pool, bad, [new], [n], table)
            torch.cuda.synchronize()
            assert bool(out[new // 2, 1].isnan().all())
            out[new // 2, 1] = _call(pool, q, [new], [n], table)[new // 2, 1]
            _check(pool, oracle, q, out, [new], [n], table)
            pool.destroy()


@pytest.mark.parametrize("sequences", [1, 64, 65, 200])
def test_many_sequences(device, oracle, sequences):
    import torch
    rng = np.random.RandomState(sequences)
    lengths = [int(n) for n in rng.randint(0, 150, sequences)]
    lengths[0] = 1500
    new = [min(n, int(rng.choice([0, 1, 1, 1, 3, 60]))) for n in lengths]
    new[0] = 200
    pool, table = _written(device, "B", "q8", 64, 1, 32, lengths, rng, 1)
    q = _rows(sum(new), 3, 64, "bfloat16", 1, 3).cuda()
    out = _call(pool, q, new, lengths, table)
    torch.cuda.synchronize()
    _check(pool, oracle, q, out, new, lengths, table)
    pool.destroy()


def test_rows_that_see_nothing_and_rows_of_no_sequence(device, oracle):
    """More new rows than tokens, pages that are none, clamped lengths and offsets, rows before and behind the sequences'."""
    import torch
    rng = np.random.RandomState(1)
    pool = Pool(device, "S", "q8", 64, 3, 40, 32)
    _fill(pool, 4)
    table = torch.from_numpy(rng.randint(0, pool.pages, (4, 40)).astype(np.int32))
    table[0, ::2], table[1], table[2, 5:9] = -1, pool.pages, 2 ** 31 - 1
    table = table.cuda()
    for dtype in ("float16", "bfloat16"):
        new, lengths, first = [70, 9, 300, 2], [500, 400, 1200, 300], 7
        q = _rows(sum(new) + 20, 6, 64, dtype, 1, 3).cuda()
        out = torch.full_like(q, 7.0)
        _call(pool, q, new, lengths, table, out=out, first=first)
        torch.cuda.synchronize()
        _check(pool, oracle, q, out, new, lengths, table, first=first)
        assert bool((out[:first] == 7).all()) and bool((out[first + sum(new):] == 7).all())
        assert bool((out[first + 70:first + 79] == 0).all())  # no page of its is in the pool
        # rows at negative positions
        out = torch.full_like(q, 7.0)
        _call(pool, q, [100, 0, 3, 1], [40, 0, 0, 1], table, out=out)
        torch.cuda.synchronize()
        assert bool((out[:60] == 0).all()) and bool((out[100:103] == 0).all()) and bool((out[104:] == 7).all())
        _check(pool, oracle, q, out, [40], [40], table[:1], first=60)
        # lengths beyond max_length count as it; a chunk's rows end there
        out = _call(pool, q, [10, 0, 5, 1], [2 ** 31 - 1, 33, 700, 90], table, max_length=600)
        torch.cuda.synchronize()
        _check(pool, oracle, q, out, [10, 0, 5, 1], [600, 33, 600, 90], table)
    pool.destroy()


@pytest.mark.parametrize("layout,dim", [("f16", 64), ("f16", 128), ("B", 64)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_non_finite_rows_reach_only_what_sees_them(device, oracle, layout, dim, dtype):
    """K and V rows of infinities and NaNs among the new tokens: rows before them are as if they were not there."""
    import torch
    from bgtq import batched
    n, c = 300, 150
    for new, window in ((c, 0), (c, 40), (7, 0), (7, 3)):
        pool = Pool(device, layout, "f16" if layout == "f16" else "q8", dim, 1, 6, 64)
        k, v = _rows(n, 1, dim, "float16", 1, 1), _rows(n, 1, dim, "float16", 1, 2)
        bad = [n - new + 2, n - new // 2, n - 1]
        kb, vb = k.clone(), v.clone()
        kb[bad[0], 0, 5], vb[bad, 0, 1::4] = float("nan"), torch.tensor([float("inf"), float("nan"), float("-inf")], dtype=torch.float16)[:, None]
        table = torch.tensor([[3, 0, 5, 1, 4]], dtype=torch.int32, device="cuda")
        slots = table[0].long()[torch.arange(n, device="cuda") // 64] * 64 + torch.arange(n, device="cuda") % 64
        q = _rows(new, 2, dim, dtype, 1, 3).cuda()
        outs = []
        for kk, vv in ((k, v), (kb, vb)):
            batched.paged_write(device, pool.handle, slots, kk.cuda(), vv.cuda())
            outs.append(_call(pool, q, [new], [n], table, window, 0))
        torch.cuda.synchronize()
        pos = torch.arange(n - new, n)
        sees = torch.zeros(new, dtype=torch.bool)
        for b in bad:
            sees |= (pos >= b) & ((pos < b + window) if window else True)
        assert torch.equal(outs[0][~sees], outs[1][~sees]) and int((~sees).sum()) >= 2
        assert bool(outs[0].isfinite().all()) and not bool(outs[1][sees][..., 1::4].isfinite().all())
        pool.destroy()


def test_strides_scale_and_large_logits(device, oracle):
    """q and out as slices of wider rows; a given scale; logits of a few hundred."""
    import torch
    rng = np.random.RandomState(2)
    lengths, new = [200, 77, 300], [50, 1, 300]
    for layout, dim in (("B", 64), ("f16", 128)):
        pool, table = _written(device, layout, "f16", dim, 2, 32, lengths, rng, 3)
        for dtype in ("float16", "bfloat16"):
            wide = _rows(sum(new), 10, dim, dtype, 1, 3).cuda()
            q, out = wide[:, 2:6], torch.full((sum(new), 12, dim), 3.0, dtype=wide.dtype, device="cuda")
            for mult, scale in ((1.0, 0.02), (1.0, None), (0.0, None)):
                x = q * mult
                qq = wide.clone()[:, 2:6]
                qq.copy_(x)
                _call(pool, qq, new, lengths, table, scale=scale, out=out[:, 1:9:2])
                torch.cuda.synchronize()
                _check(pool, oracle, qq, out[:, 1:9:2], new, lengths, table, scale=scale)
                assert bool((out[:, ::2] == 3).all())
        pool.destroy()


def test_captured_and_on_another_stream(device, oracle):
    """A captured call replays over new offsets, lengths, tables and queries; eager calls on another stream between."""
    import torch
    import bgtq
    from bgtq import batched
    rng = np.random.RandomState(1)
    pool = Pool(device, "B", "q8", 64, 2, 70, 32)
    _fill(pool, 1)
    q, out = _rows(300, 6, 64, "bfloat16", 1).cuda(), torch.zeros((300, 6, 64), dtype=torch.bfloat16, device="cuda")
    offsets, lengths = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    table = torch.zeros((4, 64), dtype=torch.int32, device="cuda")
    args = dict(pages=pool.handle, q=q, out=out, offsets=offsets, lengths=lengths, page_table=table)
    size = batched.paged_prefill_workspace_bytes(batched.paged_prefill_desc(**args))
    desc = batched.paged_prefill_desc(workspace=torch.zeros(size, dtype=torch.uint8, device="cuda"), **args)
    batched.paged_prefill(device, desc)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        device.set_stream(torch.cuda.current_stream().cuda_stream)
        batched.paged_prefill(device, desc)
    batched.bind_torch_stream(device)
    eager, want = bgtq.Device(0), torch.zeros_like(out)
    other = batched.paged_prefill_desc(workspace=torch.zeros(size, dtype=torch.uint8, device="cuda"), **{**args, "out": want})
    for new, lens in (([1, 1, 1, 1], [2000, 5, 64, 900]), ([200, 1, 0, 99], [1999, 70, 0, 1000]), ([0, 0, 0, 300], [0, 0, 0, 2048])):
        offsets.copy_(torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32))
        lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        table.copy_(torch.from_numpy(rng.randint(0, pool.pages, (4, 64)).astype(np.int32)))
        q.copy_(_rows(300, 6, 64, "bfloat16", sum(new)))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            batched.bind_torch_stream(eager)
            batched.paged_prefill(eager, other)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _check(pool, oracle, q, out, new, lens, table)
        n = sum(new)
        assert torch.equal(out[:n], want[:n])
    eager.destroy()
    pool.destroy()


@pytest.mark.parametrize("rows,max_length", [(100, 1024), (2000, 1024), (2000, 1 << 17)])
def test_offsets_out_of_order(device, oracle, rows, max_length):
    """Offsets count as no less than those before them, whatever they hold; also where the sequences take turns."""
    import torch
    from bgtq import batched
    rng = np.random.RandomState(9)
    S = 70
    lengths = [int(n) for n in rng.randint(1, 400, S)]
    pool, table = _written(device, "B", "q8", 64, 2, 64, lengths, rng, 5, spare=max_length // 64)
    q = _rows(rows, 4, 64, "bfloat16", 4, 3).cuda()
    for kind in range(3):
        given = rng.randint(-rows, 2 * rows, S + 1) if kind == 0 else np.where(np.arange(S + 1) % 2, rows, 0) if kind == 1 else -np.arange(S + 1)
        meant = np.maximum.accumulate(np.clip(given, 0, rows))
        args = dict(pages=pool.handle, q=q, offsets=torch.tensor(given, dtype=torch.int32, device="cuda"),
                    lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), page_table=table, max_length=max_length)
        out = torch.full_like(q, 7.0)
        size = batched.paged_prefill_workspace_bytes(batched.paged_prefill_desc(out=out, **args))
        batched.paged_prefill(device, batched.paged_prefill_desc(out=out, workspace=torch.zeros(size, dtype=torch.uint8, device="cuda"), **args))
        torch.cuda.synchronize()
        _check(pool, oracle, q, out, list(np.diff(meant)), lengths, table, first=int(meant[0]))
        assert bool((out[:meant[0]] == 7).all()) and bool((out[meant[-1]:] == 7).all())
    pool.destroy()


@pytest.mark.parametrize("layout,v,dim", [("f16", "f16", 128), ("B", "q8", 64)])
def test_pages_beyond_32_bits(device, layout, v, dim):
    """Pages several hundred million entries apart: the same bits as from a compact pool."""
    import torch
    from bgtq import batched
    rows, got = 700, []
    k, val = _rows(rows, 1, dim, "bfloat16", 1, 1).cuda(), _rows(rows, 1, dim, "bfloat16", 1, 2).cuda()
    q = _rows(rows, 4, dim, "bfloat16", 1, 3).cuda()
    rope = batched.rope(table=batched.rope_table(1000, dim, 1e4))
    positions = torch.arange(rows, device="cuda")
    table = torch.tensor(np.random.RandomState(1).permutation(12)[None], dtype=torch.int32, device="cuda")
    slots = table[0].long()[positions // 64] * 64 + positions % 64
    for gap in (32, 400_000_000):
        pool = Pool(device, layout, v, dim, 1, 12, 64, gap=gap)
        qr = torch.empty_like(q)
        batched.paged_append(device, pool.handle, slots, rope, positions, k, val, q=q, q_out=qr)
        outs = [qr]
        for new in (5, 300):
            for window, sinks in ((0, 0), (100, 5)):
                outs.append(_call(pool, qr[rows - new:].contiguous(), [new], [rows], table, window, sinks))
        q1, o1 = qr[-1:].float().contiguous(), torch.empty((1, 4, dim), device="cuda")
        args = dict(pages=pool.handle, q=q1, out=o1, lengths=torch.tensor([rows], dtype=torch.int32, device="cuda"), page_table=table, window=200, sinks=4)
        ws = torch.zeros(batched.paged_decode_workspace_bytes(batched.paged_decode_desc(**args)), dtype=torch.uint8, device="cuda")
        batched.paged_decode(device, batched.paged_decode_desc(workspace=ws, **args))
        kr, vr = torch.empty_like(k), torch.empty_like(val)
        batched.paged_read(device, pool.handle, slots, kr, vr)
        torch.cuda.synchronize()
        got.append([t.clone() for t in (*outs, o1, kr, vr)])
        pool.destroy()
        del pool
    for a, b in zip(*got):
        assert torch.equal(a, b) and bool(a.isfinite().all())


@pytest.mark.parametrize("layout,v,dim,heads", [("S", "q8", 64, 3), ("f16", "f16", 128, 2)])
def test_shared_and_large_pages(device, oracle, layout, v, dim, heads):
    """Sequences that share their first pages; pages of 4096 tokens; no sequences; sequences without rows."""
    import torch
    from bgtq import batched
    rng = np.random.RandomState(11)
    pool, table = _written(device, layout, v, dim, heads, 4096, [6000, 4096], rng, 5)
    table = table[[0, 0, 1, 0]].contiguous()
    new, lengths = [50, 1, 200, 7], [6000, 4500, 4096, 3000]
    q = _rows(sum(new), 2 * heads, dim, "bfloat16", 4, 3).cuda()
    for window, sinks in ((0, 0), (4100, 10)):
        out = _call(pool, q, new, lengths, table, window, sinks)
        torch.cuda.synchronize()
        _check(pool, oracle, q, out, new, lengths, table, window, sinks)
    out = _call(pool, q, [0, 0, 0, 0], lengths, table)
    none = _call(pool, q, [], [], table[:0])
    torch.cuda.synchronize()
    assert bool(out.isnan().all()) and bool(none.isnan().all())
    pool.destroy()


def test_two_calls_at_once(device, oracle):
    """Two contexts on streams of their own over one pool, a workspace each."""
    import bgtq
    import torch
    from bgtq import batched
    rng = np.random.RandomState(10)
    lengths = [3000, 700, 64]
    pool, table = _written(device, "S", "q8", 64, 3, 64, lengths, rng, 5)
    calls = []
    for new in ([600, 1, 0], [1, 1, 20]):
        q = _rows(sum(new), 9, 64, "float16", sum(new), 3).cuda()
        calls.append((new, q, _call(pool, q, new, lengths, table)))
    torch.cuda.synchronize()
    others, descs = [], []
    for new, q, _ in calls:
        stream, ctx = torch.cuda.Stream(), bgtq.Device(0)
        ctx.set_stream(stream.cuda_stream)
        args = dict(pages=pool.handle, q=q, out=torch.zeros_like(q), offsets=torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda"),
                    lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), page_table=table)
        size = batched.paged_prefill_workspace_bytes(batched.paged_prefill_desc(**args))
        descs.append((args["out"], batched.paged_prefill_desc(workspace=torch.zeros(size, dtype=torch.uint8, device="cuda"), **args)))
        others.append((ctx, stream))
    torch.cuda.synchronize()
    for _ in range(20):
        for (ctx, _s), (_o, desc) in zip(others, descs):
            batched.paged_prefill(ctx, desc)
    torch.cuda.synchronize()
    for (_n, _q, want), (got, _d) in zip(calls, descs):
        assert torch.equal(want, got)
    for ctx, _s in others:
        ctx.destroy()
    pool.destroy()


def test_a_step_from_rows_to_outputs(device, oracle):
    """A layer's step as a serving loop runs it: rows rotated into the pages, then all chunks attended, then single
    tokens decoded behind a window, against 64 bits from the rows themselves with K as the pages hold it."""
    import torch
    from bgtq import batched
    from test_gpu_window import _decode, _decode_reference
    from test_gpu_paged import _check as _check_decode
    batched.bind_torch_stream(device)
    rng = np.random.RandomState(4)
    pool = Pool(device, "S", "q8", 64, 3, 60, 32)
    rope = batched.rope(table=batched.rope_table(4096, 64, 1e5))
    lens, table = [0, 0, 0], torch.from_numpy(rng.permutation(60)[:48].reshape(3, 16).astype(np.int32)).cuda()
    for step, new in enumerate(([100, 7, 0], [60, 0, 300], [1, 1, 1], [1, 30, 1])):
        n = sum(new)
        x = _rows(n, 9 + 6, 64, "bfloat16", step, 9).cuda()
        positions = torch.cat([torch.arange(have, have + c) for have, c in zip(lens, new)]).cuda()
        seq = torch.cat([torch.full((c,), b) for b, c in enumerate(new)]).cuda()
        slots = table[seq, positions // 32].long() * 32 + positions % 32
        q = torch.empty((n, 9, 64), dtype=x.dtype, device="cuda")
        batched.paged_append(device, pool.handle, slots, rope, positions, x[:, 9:12], x[:, 12:], x[:, :9], q)
        lens = [have + c for have, c in zip(lens, new)]
        out = _call(pool, q, new, lens, table)
        torch.cuda.synchronize()
        _check(pool, oracle, q, out, new, lens, table, what=f"step {step}")
    q32 = _rows(3, 9, 64, "float32", 1).cuda()
    _check_decode(_decode(pool, q32, lens, table, 50, 4), _decode_reference(pool, oracle, q32, lens, table, 50, 4))
    pool.destroy()


def test_wrapper_refusals(device):
    import torch
    import bgtq
    from bgtq import batched
    batched.bind_torch_stream(device)
    pool = Pool(device, "f16", "f16", 64, 2, 4, 32)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.zeros((5, 4, 64), dtype=torch.float16, device="cuda")
    good = dict(pages=pool.handle, q=q, out=q.clone(), offsets=i32(0, 5), lengths=i32(9), page_table=i32(0, 1)[None])
    for bad in (dict(q=q.float()), dict(out=q.bfloat16()), dict(q=q[..., :32]), dict(q=q.cpu()), dict(out=q[:4]), dict(offsets=i32(0, 2, 5)),
                dict(offsets=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(lengths=i32(9, 9)), dict(page_table=i32(0, 1)),
                dict(max_length=65), dict(sinks=1), dict(window=-1), dict(scale=0.0), dict(scale=-1.0), dict(q=q.transpose(0, 1))):
        with pytest.raises(bgtq.RangeError):
            batched.paged_prefill_desc(**{**good, **bad})
    with pytest.raises(bgtq.RangeError, match="workspace"):
        batched.paged_prefill(device, batched.paged_prefill_desc(**good))
    odd = torch.zeros((5, 4, 72), dtype=torch.float16, device="cuda")[..., 4:68]
    with pytest.raises(bgtq.RangeError, match="aligned"):
        batched.paged_prefill(device, batched.paged_prefill_desc(**{**good, "q": odd}))
    empty = dict(good, q=q[:0], out=q[:0], offsets=i32(0, 0))
    batched.paged_prefill(device, batched.paged_prefill_desc(workspace=torch.zeros(1 << 28, dtype=torch.uint8, device="cuda"), **empty))
