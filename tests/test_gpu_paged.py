"""The paged cache: rows written into pages, read back, and decode attention over them.

Written K codes and scales must equal the oracle's encode bit for bit, 8-bit V the
definition in 64 bits exactly; outputs of the decode within 1e-5 + 1e-4 |ref| of
attention in 64 bits over the rows that the pages hold (the batched decode's tolerance).
"""
import numpy as np
import pytest

from conftest import REF

pytestmark = pytest.mark.gpu

ATOL, RTOL = 1e-5, 1e-4
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _params(layout, dim, heads):
    """BlockGTQParameters per KV head."""
    import bgtq
    from bgtq import calibrate, calibration
    if layout == "S":
        blobs = calibration.read(REF / "model")[2]
        return [bgtq.BlockGTQParameters.from_serialized(blobs[7 + h].config, blobs[7 + h].table) for h in range(heads)]
    make = {"A": calibrate.layout_a, "B": calibrate.layout_b}[layout]
    return [make(dim)] * heads


def _olayout(oracle, p):
    return oracle.Layout(dim=p.dim, groups=p.groups, row_bytes=p.rowBytes, norm_stride=p.normStride,
                         nibble_dims=p.nibbleDims, max_centroids=p.maxCentroids, perm=p.permutation,
                         group_of=p.groupOf, pos_to_cb=p.positionToCodebook, code_lut=p.codeLut,
                         rotation=p.rotation, centroids=p.centroids, offsets=p.offsets, inv_scales=p.inverseScales)


class Pool:
    """A pool of pages on the GPU whose every byte starts as garbage: scales and FP16 rows as NaN."""

    def __init__(self, device, layout, v, dim, heads, pages, page, gap=0):
        import torch
        import bgtq
        from bgtq import batched
        batched.bind_torch_stream(device)
        self.layout, self.q8, self.dim, self.heads, self.pages, self.page = layout, v == "q8", dim, heads, pages, page
        self.device, self.params = device, _params(layout, dim, heads) if layout != "f16" else []
        self.tables = [bgtq.Tables(device, p) for p in self.params]

        def garbage(dtype, *shape):  # `gap` more entries per head, in whole 16 bytes
            n = int(np.prod(shape[2:])) + gap
            flat = torch.full((pages, heads, n), 0x7e7f if dtype == torch.float16 else 0x7f, dtype=torch.int16 if dtype == torch.float16 else torch.uint8,
                              device="cuda")
            flat = flat.view(dtype) if dtype != torch.uint8 else flat
            return flat[:, :, :n - gap].unflatten(2, shape[2:])
        self.v = garbage(torch.int8 if self.q8 else torch.float16, pages, heads, page, dim)
        self.v_scales = garbage(torch.float16, pages, heads, page) if self.q8 else None
        self.packed = self.norms = self.k = None
        if self.params:
            self.packed = garbage(torch.uint8, pages, heads, page * max(p.rowBytes for p in self.params))
            self.norms = garbage(torch.float16, pages, heads, page * max(p.normStride for p in self.params))
        else:
            self.k = garbage(torch.float16, pages, heads, page, dim)
        self.handle = batched.pages(page_tokens=page, tables=self.tables or None, packed=self.packed, norms=self.norms,
                                    k_f16=self.k, v=self.v, v_scales=self.v_scales)

    def destroy(self):
        for t in self.tables:
            t.destroy()

    def k_bytes(self, h, slots):
        """The packed rows and FP16 scale bits of head h at the slots (numpy)."""
        p, (pg, at) = self.params[h], np.divmod(np.asarray(slots), self.page)
        rows = self.packed[:, h, :self.page * p.rowBytes].cpu().numpy().reshape(self.pages, self.page, p.rowBytes)
        norms = self.norms.view_as(self.norms)[:, h, :self.page * p.normStride].cpu().numpy().reshape(self.pages, self.page, p.normStride)
        return rows[pg, at], norms[pg, at]

    def k_rows(self, oracle, h, slots):
        """The K rows in 64 bits, and per dimension the sum of |factor| products that rebuild it."""
        pg, at = np.divmod(np.asarray(slots), self.page)
        if self.k is not None:
            k = self.k[:, h].cpu().numpy()[pg, at].astype(np.float64)
            return k, np.abs(k)
        p = self.params[h]
        rows, norms = self.k_bytes(h, slots)
        codes = oracle.unpack(rows, self.dim, p.nibbleDims).astype(np.int64)
        cent = np.asarray(p.centroids, np.float64).reshape(self.dim, -1)
        cs = cent[np.arange(self.dim), codes] * norms.astype(np.float64)[:, np.asarray(p.groupOf, np.int64)]
        rot, perm = np.asarray(p.rotation, np.float64).reshape(self.dim, self.dim), np.asarray(p.permutation, np.int64)
        k, size = np.empty_like(cs), np.empty_like(cs)
        k[:, perm], size[:, perm] = cs @ rot, np.abs(cs) @ np.abs(rot)
        return k, size

    def v_rows(self, h, slots):
        """The V rows' FP16 values."""
        pg, at = np.divmod(np.asarray(slots), self.page)
        v = self.v[:, h].cpu().numpy()[pg, at]
        if not self.q8:
            return v
        with np.errstate(over="ignore"):
            return (v.astype(np.float32) * self.v_scales[:, h].cpu().numpy()[pg, at].astype(np.float32)[:, None]).astype(np.float16)

    def snapshot(self):
        return [None if t is None else t.clone() for t in (self.v, self.v_scales, self.packed, self.norms, self.k)]


def _same_bits(a, b):
    import torch
    kind = {1: torch.uint8, 2: torch.int16}[a.element_size()]
    return torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


def _rows(n, heads, dim, dtype, seed, salt=0, scale=1.0):
    import torch
    g = torch.Generator().manual_seed(1000 * seed + salt)
    return (torch.randn((n, heads, dim), generator=g) * scale).to(getattr(torch, dtype))


def _quantise(v):
    """(codes, FP16 scales) of FP16 rows by the definition, in 64 bits."""
    top = np.abs(v.astype(np.float64)).max(-1)
    s = (top / 127).astype(np.float16)
    s = np.where(s.astype(np.float64) * 127 < top, np.nextafter(s, np.float16(np.inf)), s)
    d = s.astype(np.float64)[..., None]
    return np.where(d > 0, np.rint(v.astype(np.float64) / np.where(d > 0, d, 1)), 0).astype(np.int8), s


def _check_write(pool, oracle, slots, k, v):
    """Every written row holds the definition's codes."""
    k16, v16 = k.half().numpy(), v.half().numpy()
    pg, at = np.divmod(np.asarray(slots), pool.page)
    for h in range(pool.heads):
        if pool.k is not None:
            assert np.array_equal(pool.k[:, h].cpu().numpy()[pg, at].view(np.uint16), k16[:, h].view(np.uint16))
        else:
            rows, norms = pool.k_bytes(h, slots)
            want_rows, want_norms = oracle.encode_pack(_olayout(oracle, pool.params[h]), np.ascontiguousarray(k16[:, h]).view(np.uint16))[:2]
            assert np.array_equal(rows, want_rows), f"packed K of head {h}"
            assert np.array_equal(norms.view(np.uint16), np.asarray(want_norms).view(np.uint16)), f"scales of head {h}"
        got = pool.v[:, h].cpu().numpy()[pg, at]
        if pool.q8:
            codes, s = _quantise(v16[:, h])
            assert np.array_equal(pool.v_scales[:, h].cpu().numpy()[pg, at].view(np.uint16), s.view(np.uint16))
            assert np.array_equal(got, codes)
        else:
            assert np.array_equal(got.view(np.uint16), v16[:, h].view(np.uint16))


def _check_read(pool, oracle, slots, k, v):
    """K, V read at the slots: K within the split product's 3 2^-20 and FP32 sums' 2^-24 per term (together
    below 2^-18 of the sum of magnitudes) and the output's half step, V exactly its FP16 value rounded."""
    import torch
    for h in range(pool.heads):
        ref, size = pool.k_rows(oracle, h, slots)
        got = k[:, h].double().cpu().numpy()
        lim = (0 if pool.k is not None else 2.0 ** -18) * size + HALF_STEP[str(k.dtype)[6:]] * np.abs(ref) * 1.001 + 1e-7
        assert np.all(np.abs(got - ref) <= lim), f"K head {h}: {np.max(np.abs(got - ref) / lim):.2f} of the limit"
        want = torch.from_numpy(pool.v_rows(h, slots)).to(v.dtype)
        assert torch.equal(v[:, h].cpu(), want), f"V head {h}"


CASES = [("S", "q8", 64, 3, 64), ("B", "q8", 64, 2, 32), ("B", "f16", 128, 2, 64), ("A", "q8", 128, 1, 32),
         ("A", "f16", 64, 2, 256), ("f16", "q8", 64, 1, 64), ("f16", "f16", 128, 4, 32)]


@pytest.mark.parametrize("layout,v,dim,heads,page", CASES)
@pytest.mark.parametrize("rows,dtype", [(1, "float32"), (17, "float16"), (300, "bfloat16"), (5000, "float32"), (4999, "float16"), (9000, "bfloat16")])
def test_write_and_read(device, oracle, layout, v, dim, heads, page, rows, dtype):
    """Few rows (a wave each) and many (16 to a wave), consecutive and scattered slots, every source type."""
    import torch
    from bgtq import batched
    print(layout, v, dim, heads, page, rows, dtype, flush=True)
    pages = -(-rows // page) + 2
    pool = Pool(device, layout, v, dim, heads, pages, page, gap=16)
    rng = np.random.RandomState(rows)
    if rows % 2:  # pages in any order, the first one entered in its middle
        order = rng.permutation(pages)
        t = np.arange(rows) + (page // 2 + 3 if rows > 1 else 0)
        slots = order[t // page] * page + t % page
    else:
        slots = rng.permutation(pages * page)[:rows]
    k, val = _rows(rows, heads, dim, dtype, rows, 1, 2.0), _rows(rows, heads, dim, dtype, rows, 2)
    if rows > 10:
        val[3], val[5] = 0, 1e-7  # a row of zeros, one of the smallest values
        k[4] = 0
        val[6, :, 0] = 60000.0
    before = pool.snapshot()
    sd = torch.from_numpy(slots).cuda()
    batched.paged_write(device, pool.handle, sd, k.cuda(), val.cuda())
    torch.cuda.synchronize()
    _check_write(pool, oracle, slots, k, val)
    # nothing else changed
    mask = torch.zeros(pages * page, dtype=torch.bool)
    mask[slots] = True
    keep = ~mask.view(pages, 1, page).expand(pages, heads, page).cuda()
    now = pool.snapshot()
    for x, y in ((before[0], now[0]), (before[1], now[1]), (before[4], now[4])):
        if x is not None:
            assert _same_bits(x[keep], y[keep])
    for h, p in enumerate(pool.params):
        for x, y, w in ((before[2], now[2], p.rowBytes), (before[3], now[3], p.normStride)):
            x, y = (a[:, h, :page * w].reshape(pages, page, w)[keep[:, h]] for a in (x, y))
            assert _same_bits(x, y)
    for out in ("float32", "float16", "bfloat16"):
        ko, vo = (torch.empty((rows, heads, dim), dtype=getattr(torch, out), device="cuda") for _ in range(2))
        batched.paged_read(device, pool.handle, sd, ko, vo)
        torch.cuda.synchronize()
        _check_read(pool, oracle, slots, ko, vo)
    pool.destroy()


@pytest.mark.parametrize("rows", [5, 6000])
def test_rows_strided_unaligned_and_skipped(device, oracle, rows):
    """Rows inside wider tensors at odd offsets; slots outside the pool are skipped on both ways."""
    import torch
    from bgtq import batched
    heads, dim, page = 3, 64, 64
    pages = rows // page + 2
    pool = Pool(device, "S", "q8", dim, heads, pages, page)
    wide = torch.zeros((rows, 2 * heads, dim + 5), dtype=torch.float16)
    wide[:, :, 3:3 + dim] = _rows(rows, 2 * heads, dim, "float16", 11)
    w = wide.cuda()
    k, v = w[:, :heads, 3:3 + dim], w[:, heads:, 3:3 + dim]
    slots = np.random.RandomState(3).permutation(pages * page)[:rows].astype(np.int64)
    bad = slots.copy()
    bad[::3] = [-1, pages * page, 2 ** 62, -2 ** 63][rows % 4]
    before = pool.snapshot()
    batched.paged_write(device, pool.handle, torch.from_numpy(bad).cuda(), k, v)
    torch.cuda.synchronize()
    good = np.ones(rows, bool)
    good[::3] = False
    _check_write(pool, oracle, slots[good], k.cpu()[good], v.cpu()[good])
    pg, at = np.divmod(slots[~good], page)
    assert _same_bits(before[0].cpu()[pg, :, at], pool.v.cpu()[pg, :, at])
    out = torch.full((rows, 2 * heads, dim + 3), 7.0, device="cuda")
    ko, vo = out[:, :heads, 1:1 + dim], out[:, heads:, 2:2 + dim]
    batched.paged_read(device, pool.handle, torch.from_numpy(bad).cuda(), ko, vo)
    torch.cuda.synchronize()
    _check_read(pool, oracle, slots[good], ko[good], vo[good])
    assert bool((out[~torch.from_numpy(good).cuda()] == 7.0).all()) and bool((out[:, :heads, 0] == 7.0).all())
    only = torch.empty((rows, heads, dim), device="cuda")
    batched.paged_read(device, pool.handle, torch.from_numpy(slots).cuda(), v=only)
    only_k = torch.empty((rows, heads, dim), device="cuda")
    batched.paged_read(device, pool.handle, torch.from_numpy(slots).cuda(), k=only_k)
    torch.cuda.synchronize()
    assert torch.equal(only[good], vo[good]) and torch.equal(only_k[good], ko[good])
    pool.destroy()


def test_non_finite_rows(device):
    """A V row with an infinity or a NaN reads back as NaN; other rows of the call, and K, keep their own."""
    import torch
    from bgtq import batched
    pool = Pool(device, "B", "q8", 64, 2, 3, 32)
    k, v = _rows(40, 2, 64, "float32", 1), _rows(40, 2, 64, "float32", 2)
    v[3, 0, 5], v[9, 1, 63], v[11, 0, 0] = float("inf"), float("nan"), 1e6  # 1e6: an infinity in FP16
    slots = torch.arange(40, device="cuda") + 7
    batched.paged_write(device, pool.handle, slots, k.cuda(), v.cuda())
    ko, vo = torch.empty((40, 2, 64), device="cuda"), torch.empty((40, 2, 64), device="cuda")
    batched.paged_read(device, pool.handle, slots, ko, vo)
    torch.cuda.synchronize()
    bad = torch.zeros((40, 2), dtype=torch.bool)
    bad[3, 0] = bad[9, 1] = bad[11, 0] = True
    assert bool(vo[bad.cuda()].isnan().all()) and bool(vo[~bad.cuda()].isfinite().all()) and bool(ko.isfinite().all())
    pool.destroy()


def test_slot_named_twice_leaves_the_others(device, oracle):
    import torch
    from bgtq import batched
    pool = Pool(device, "B", "q8", 64, 2, 3, 32)
    k, v = _rows(40, 2, 64, "float32", 1), _rows(40, 2, 64, "float32", 2)
    slots = np.arange(40) + 5
    slots[7] = slots[20]
    batched.paged_write(device, pool.handle, torch.from_numpy(slots).cuda(), k.cuda(), v.cuda())
    torch.cuda.synchronize()
    one = np.array([i for i in range(40) if i not in (7, 20)])
    _check_write(pool, oracle, slots[one], k[one], v[one])
    pool.destroy()


def _fill(pool, seed):
    """Every slot of the pool written, with rows of N(0, 1) (K decaying)."""
    import torch
    from bgtq import batched
    n = pool.pages * pool.page
    k, v = _rows(n, pool.heads, pool.dim, "float16", seed, 1), _rows(n, pool.heads, pool.dim, "float16", seed, 2)
    batched.paged_write(pool.device, pool.handle, torch.arange(n, device="cuda"), k.cuda(), v.cuda())


def _decode(pool, q, lengths, table, splits=0, max_length=None, workspace=None, q_rotated=False):
    import torch
    from bgtq import batched
    out = torch.full_like(q, float("nan"))
    args = dict(pages=pool.handle, q=q, out=out, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                page_table=table, max_length=max_length, splits=splits, q_rotated=q_rotated)
    if workspace is None:
        workspace = torch.zeros(batched.paged_decode_workspace_bytes(batched.paged_decode_desc(**args)), dtype=torch.uint8, device="cuda")
    batched.paged_decode(pool.device, batched.paged_decode_desc(workspace=workspace, **args))
    return out


def _reference(pool, oracle, q, lengths, table):
    """Attention in 64 bits over the rows of the pages that are the pool's."""
    B, Hq, D = q.shape
    G, out = Hq // pool.heads, np.zeros((B, Hq, D))
    tab = table.cpu().numpy().astype(np.int64)
    for h in range(pool.heads):
        for b, n in enumerate(lengths):
            t = np.arange(n)
            page = tab[b, t // pool.page]
            at = (page * pool.page + t % pool.page)[(page >= 0) & (page < pool.pages)]
            if not at.size:
                continue
            s = q[b, h * G:(h + 1) * G].double().cpu().numpy() @ pool.k_rows(oracle, h, at)[0].T / np.sqrt(D)
            e = np.exp(s - s.max(-1, keepdims=True))
            out[b, h * G:(h + 1) * G] = e @ pool.v_rows(h, at).astype(np.float64) / e.sum(-1, keepdims=True)
    return out


def _check(out, ref, what=""):
    err, lim = np.abs(out.double().cpu().numpy() - ref), ATOL + RTOL * np.abs(ref)
    assert np.all(err <= lim), f"{what}: max err {np.nanmax(err):.3e}, worst ratio {np.nanmax(err / lim):.2f}, {np.isnan(err).sum()} NaN"


def _table(pool, lengths, rng, spare=2):
    """Pages of the sequences in any order of the pool; entries past a sequence's tokens name no page."""
    import torch
    need = [-(-n // pool.page) for n in lengths]
    order = rng.permutation(pool.pages)
    table = np.full((len(lengths), max(max(need), 1) + spare), 2 ** 31 - 1, np.int32)
    table[:, -1] = -5
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    assert at <= pool.pages
    return torch.from_numpy(table).cuda()


LENGTHS = [0, 1, 31, 32, 33, 64, 65, 127, 200, 515, 0]


@pytest.mark.parametrize("layout,v,dim,heads,page", CASES)
@pytest.mark.parametrize("G,splits", [(1, 0), (3, 0), (7, 1), (3, 3), (16, 0), (2, 60)])
def test_decode(device, oracle, layout, v, dim, heads, page, G, splits):
    """Sequences from none to many tokens that end anywhere in a page whose rest is garbage."""
    import torch
    print(layout, v, dim, heads, page, G, splits, flush=True)
    rng = np.random.RandomState(G)
    pool = Pool(device, layout, v, dim, heads, sum(-(-n // page) for n in LENGTHS) + 2, page, gap=32)
    lengths = [int(n) for n in rng.permutation(LENGTHS)]
    table = _table(pool, lengths, rng)
    # only the sequences' own tokens are written; the rest of the pool stays garbage
    from bgtq import batched
    tab = table.cpu().numpy().astype(np.int64)
    slots = np.concatenate([tab[b, np.arange(n) // page] * page + np.arange(n) % page for b, n in enumerate(lengths)]).astype(np.int64)
    k, val = _rows(len(slots), heads, dim, "float16", G, 1), _rows(len(slots), heads, dim, "float16", G, 2)
    batched.paged_write(device, pool.handle, torch.from_numpy(slots).cuda(), k.cuda(), val.cuda())
    q = _rows(len(lengths), heads * G, dim, "float32", G, 3).cuda()
    out = _decode(pool, q, lengths, table, splits)
    torch.cuda.synchronize()
    _check(out, _reference(pool, oracle, q, lengths, table))
    assert bool((out[[b for b, n in enumerate(lengths) if n == 0]] == 0).all())
    pool.destroy()


@pytest.mark.parametrize("layout,v", [("B", "q8"), ("S", "q8"), ("f16", "f16")])
def test_decode_pages_that_are_none(device, oracle, layout, v):
    """Tokens of table entries outside the pool are left out, also whole sequences of them."""
    import torch
    rng = np.random.RandomState(5)
    pool = Pool(device, layout, v, 64, 3 if layout == "S" else 2, 40, 32)
    _fill(pool, 4)
    lengths = [400, 333, 96, 1000]
    table = torch.from_numpy(rng.randint(0, pool.pages, (4, 33)).astype(np.int32))  # pages shared between sequences
    table[0, ::2] = -1
    table[1, 3:] = torch.tensor(pool.pages, dtype=torch.int32)
    table[2] = -2 ** 31
    table[3, rng.permutation(32)[:20]] = 2 ** 31 - 1
    table = table.cuda()
    q = _rows(4, pool.heads * 3, 64, "float32", 1).cuda()
    out = _decode(pool, q, lengths, table)
    torch.cuda.synchronize()
    _check(out, _reference(pool, oracle, q, lengths, table))
    assert bool((out[2] == 0).all())
    pool.destroy()


def test_decode_long(device, oracle):
    """A long sequence beside short ones: every merge of splits, several chunks per wave."""
    import torch
    rng = np.random.RandomState(9)
    for layout, v, dim, heads in (("B", "q8", 64, 2), ("B", "q8", 128, 1), ("S", "f16", 64, 3)):
        lengths = [9001, 40, 0, 4097]
        pool = Pool(device, layout, v, dim, heads, sum(-(-n // 64) for n in lengths) + 1, 64)
        _fill(pool, 8)
        table = _table(pool, lengths, rng)
        q = _rows(4, heads * 7, dim, "float32", 6, scale=2.0).cuda()
        ref = _reference(pool, oracle, q, lengths, table)
        for splits in (0, 1, 2, 8, 20, 40, 50, 200):
            print(layout, v, dim, splits, flush=True)
            _check(_decode(pool, q, lengths, table, splits), ref, f"{layout} {dim} splits {splits}")
        # max_length clamps the lengths
        _check(_decode(pool, q, [2 ** 31 - 1] * 4, table, max_length=33),
               _reference(pool, oracle, q, [33] * 4, table), "clamped") if layout == "B" and dim == 64 else None
        pool.destroy()


@pytest.mark.parametrize("layout,v,dim,heads", [("B", "q8", 64, 2), ("f16", "f16", 128, 1), ("S", "q8", 64, 3)])
@pytest.mark.parametrize("batch", [2, 31, 64, 65])
def test_decode_workgroups_shared_by_length(device, oracle, layout, v, dim, heads, batch):
    """Sequences share the workgroups by their lengths: one long among short ones, mixed, equal, and none at all,
    in one workspace; lengths beyond max_length count as it."""
    import torch
    rng = np.random.RandomState(batch)
    longest = 6000 if batch == 2 else 2500
    kinds = {"one long": [longest] + [int(n) for n in rng.randint(0, 40, batch - 1)],
             "mixed": [int(longest * (i / batch) ** 3) for i in range(batch)],
             "equal": [700] * batch, "short": [1] * batch, "none": [0] * batch}
    need = max(sum(-(-n // 128) for n in lens) for lens in kinds.values())
    pool = Pool(device, layout, v, dim, heads, need + 1, 128)
    _fill(pool, batch)
    q = _rows(batch, heads * 3, dim, "float32", batch, scale=1.5).cuda()
    for kind, lens in kinds.items():
        lens = [int(n) for n in rng.permutation(lens)]
        print(layout, dim, batch, kind, flush=True)
        table = _table(pool, lens, rng, spare=longest // 128 + 1)
        _check(_decode(pool, q, lens, table, max_length=longest), _reference(pool, oracle, q, lens, table), kind)
    short = [min(n, 300) for n in kinds["mixed"]]
    table = _table(pool, kinds["mixed"], rng)
    _check(_decode(pool, q, kinds["mixed"], table, max_length=300), _reference(pool, oracle, q, short, table), "clamped")
    pool.destroy()


@pytest.mark.parametrize("layout,dim", [("S", 64), ("B", 64), ("B", 128), ("f16", 64)])
def test_decode_of_tiny_queries(device, oracle, layout, dim):
    """Queries down to the smallest FP32 numbers give all but equal weights, and none NaN; zeros the mean."""
    pool = Pool(device, layout, "q8", dim, 2, 12, 32)
    _fill(pool, 4)
    table = _table(pool, [70, 200], np.random.RandomState(0))
    for size in (0.0, 1e-45, 1e-39, 1e-36, 1e-30, 1e-20):
        print(layout, dim, size, flush=True)
        q = (_rows(2, 6, dim, "float32", 9) * size).cuda()
        _check(_decode(pool, q, [70, 200], table), _reference(pool, oracle, q * 0, [70, 200], table), f"{layout} {dim} {size}")
    pool.destroy()


def test_decode_equals_dense(device):
    """8-bit V equals FP16 V pages of the values it stands for, bit for bit. And the same rows in one contiguous cache
    per sequence: bgtq_decode sorts a code's high and low parts into products of their own and multiplies the
    logits' factor in by itself, so the two agree as two results that are each within the tolerance of 64 bits."""
    import torch
    from bgtq import batched
    for layout, dim, heads in (("B", 64, 2), ("S", 64, 3), ("B", 128, 2)):
        pool = Pool(device, layout, "q8", dim, heads, 70, 64)
        _fill(pool, 3)
        rng = np.random.RandomState(2)
        lengths, T = [1000, 77, 2048], 2048
        table = _table(pool, lengths, rng, spare=1)
        q = _rows(3, heads * 3, dim, "float32", 5).cuda()
        out = _decode(pool, q, lengths, table, max_length=T)
        plain = Pool(device, layout, "f16", dim, heads, 70, 64)
        n = torch.arange(70 * 64, device="cuda")
        vals = torch.empty((70 * 64, heads, dim), dtype=torch.float16, device="cuda")
        batched.paged_read(device, pool.handle, n, v=vals)
        plain.packed.copy_(pool.packed)
        plain.norms.copy_(pool.norms)
        plain.v.copy_(vals.view(70, 64, heads, dim).transpose(1, 2))
        assert torch.equal(_decode(plain, q, lengths, table, max_length=T), out)
        # dense copies
        rb, ns = max(p.rowBytes for p in pool.params), max(p.normStride for p in pool.params)
        packed = torch.zeros((3, heads, (T * rb + 15) // 16 * 16), dtype=torch.uint8, device="cuda")
        norms = torch.zeros((3, heads, (T * ns + 7) // 8 * 8), dtype=torch.float16, device="cuda")
        v = torch.zeros((3, heads, T, dim), dtype=torch.float16, device="cuda")
        for b, L in enumerate(lengths):
            t = torch.arange(L, device="cuda")
            page, at = table[b].long()[t // 64], t % 64
            for h, p in enumerate(pool.params):
                rows = pool.packed[:, h, :64 * p.rowBytes].reshape(70, 64, p.rowBytes)[page, at]
                packed[b, h, :L * p.rowBytes] = rows.reshape(-1)
                norms[b, h, :L * p.normStride] = pool.norms[:, h, :64 * p.normStride].reshape(70, 64, p.normStride)[page, at].reshape(-1)
                v[b, h, :L] = plain.v[page, h, at]
        dense = torch.empty_like(q)
        kw = dict(batch=3, q_heads=3 * heads, kv_heads=heads, dim=dim, q=q, out=dense, max_length=T, tables=pool.tables,
                  lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), packed=packed, v=v,
                  packed_seq_stride=packed.stride(0), packed_head_stride=packed.stride(1), norms=norms,
                  norms_seq_stride=norms.stride(0), norms_head_stride=norms.stride(1), v_seq_stride=v.stride(0), v_head_stride=v.stride(1))
        ws = torch.zeros(batched.workspace_bytes(batched.decode_desc(**kw)), dtype=torch.uint8, device="cuda")
        batched.decode(device, batched.decode_desc(workspace=ws, **kw))
        torch.cuda.synchronize()
        off = (dense - out).abs()
        assert (off <= 2 * (ATOL + RTOL * dense.abs())).all(), (layout, dim, off.max().item())
        pool.destroy()
        plain.destroy()


def test_pages_far_apart(device, oracle):
    """Byte offsets past 2^32 between pages, for the writes, the reads and the decode."""
    import torch
    from bgtq import batched
    batched.bind_torch_stream(device)
    dim, heads, page, far = 64, 1, 32, 5 << 29  # 2.5 GiB from page to page
    import bgtq
    p = _params("B", dim, 1)
    tables = [bgtq.Tables(device, p[0])]
    buf = torch.empty(2 * far + (1 << 20), dtype=torch.uint8, device="cuda")

    def view(dtype, offset, *shape):
        size = torch.empty((), dtype=dtype).element_size()
        flat = buf.view(dtype)
        inner = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
        return flat.as_strided((3, heads) + shape, (far // size, int(np.prod(shape))) + tuple(inner), offset // size)
    pool = Pool.__new__(Pool)
    pool.layout, pool.q8, pool.dim, pool.heads, pool.pages, pool.page, pool.params, pool.k = "B", True, dim, heads, 3, page, p, None
    pool.packed, pool.norms = view(torch.uint8, 0, page * p[0].rowBytes), view(torch.float16, 4096, page * p[0].normStride)
    pool.v, pool.v_scales = view(torch.int8, 8192, page, dim), view(torch.float16, 16384, page)
    pool.device, pool.tables = device, tables
    pool.handle = batched.pages(page_tokens=page, tables=tables, packed=pool.packed, norms=pool.norms, v=pool.v, v_scales=pool.v_scales)
    k, v = _rows(96, 1, dim, "float16", 1), _rows(96, 1, dim, "float16", 2)
    slots = np.arange(96)
    batched.paged_write(device, pool.handle, torch.from_numpy(slots).cuda(), k.cuda(), v.cuda())
    torch.cuda.synchronize()
    _check_write(pool, oracle, slots, k, v)
    ko, vo = torch.empty((96, 1, dim), device="cuda"), torch.empty((96, 1, dim), device="cuda")
    batched.paged_read(device, pool.handle, torch.from_numpy(slots).cuda(), ko, vo)
    torch.cuda.synchronize()
    _check_read(pool, oracle, slots, ko, vo)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    q = _rows(1, 3, dim, "float32", 3).cuda()
    out = _decode(pool, q, [90], table)
    torch.cuda.synchronize()
    _check(out, _reference(pool, oracle, q, [90], table))
    pool.destroy()


def test_decode_queries_in_the_code_domain(device, oracle):
    import torch
    pool = Pool(device, "S", "q8", 64, 3, 12, 32)
    _fill(pool, 2)
    lengths, rng = [100, 222], np.random.RandomState(1)
    table = _table(pool, lengths, rng)
    q = _rows(2, 9, 64, "float32", 3)
    qr = torch.empty_like(q)
    for h, p in enumerate(pool.params):
        rot, perm = torch.from_numpy(np.array(p.rotation, np.float32).reshape(64, 64)), torch.from_numpy(np.array(p.permutation, np.int64))
        qr[:, 3 * h:3 * h + 3] = q[:, 3 * h:3 * h + 3][..., perm] @ rot.T
    out = _decode(pool, qr.cuda(), lengths, table, q_rotated=True)
    torch.cuda.synchronize()
    _check(out, _reference(pool, oracle, q, lengths, table))
    pool.destroy()


def test_step_of_write_and_decode_captured(device, oracle):
    """One serving step, a token's write and the attention over the cache with it, captured as a graph and replayed
    with eager work between; rows of a padded batch (no slot, length 0) do nothing."""
    import torch
    from bgtq import batched
    rng = np.random.RandomState(3)
    pool = Pool(device, "S", "q8", 64, 3, 20, 64)
    _fill(pool, 6)
    lengths = [130, 0, 64, 513]
    table = _table(pool, [n + 8 for n in lengths], rng)
    tab = table.cpu().numpy().astype(np.int64)
    ln = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    slots = torch.empty(4, dtype=torch.int64, device="cuda")
    k, v = (torch.empty((4, 3, 64), device="cuda") for _ in range(2))
    q, out = torch.empty((4, 9, 64), device="cuda"), torch.empty((4, 9, 64), device="cuda")
    args = dict(pages=pool.handle, q=q, out=out, lengths=ln, page_table=table)
    ws = torch.zeros(batched.paged_decode_workspace_bytes(batched.paged_decode_desc(**args)), dtype=torch.uint8, device="cuda")
    desc = batched.paged_decode_desc(workspace=ws, **args)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        device.set_stream(side.cuda_stream)
        batched.paged_write(device, pool.handle, slots, k, v)
        batched.paged_decode(device, desc)
    batched.bind_torch_stream(device)
    for step in range(4):
        now = [n + step + 1 if n else 0 for n in lengths]
        nk, nv = _rows(4, 3, 64, "float32", step, 1), _rows(4, 3, 64, "float32", step, 2)
        s = np.array([tab[b, (n - 1) // 64] * 64 + (n - 1) % 64 if n else -1 for b, n in enumerate(now)])
        slots.copy_(torch.from_numpy(s))
        k.copy_(nk), v.copy_(nv), ln.copy_(torch.tensor(now, dtype=torch.int32)), q.copy_(_rows(4, 9, 64, "float32", step, 3))
        graph.replay()
        torch.cuda.synchronize()
        live = np.array([b for b, n in enumerate(now) if n])
        _check_write(pool, oracle, s[live], nk[live], nv[live])
        _check(out, _reference(pool, oracle, q, now, table), f"step {step}")
        replayed = out.clone()
        batched.paged_decode(device, desc)  # eager, on the same workspace
        torch.cuda.synchronize()
        assert torch.equal(replayed, out)
    pool.destroy()


def test_workspace_shared_across_geometries(device, oracle):
    import torch
    rng = np.random.RandomState(8)
    pool = Pool(device, "B", "q8", 64, 2, 60, 32)
    _fill(pool, 1)
    ws = torch.zeros(8 << 20, dtype=torch.uint8, device="cuda")
    for lengths, G, splits in (([900, 20], 3, 0), ([33] * 20, 7, 0), ([1500], 1, 9), ([0, 700, 64], 2, 4)):
        table = _table(pool, lengths, rng)
        q = _rows(len(lengths), 2 * G, 64, "float32", G).cuda()
        out = _decode(pool, q, lengths, table, splits, workspace=ws)
        torch.cuda.synchronize()
        _check(out, _reference(pool, oracle, q, lengths, table))
    pool.destroy()


def test_other_stream_and_current_device_kept(device, oracle):
    """Calls run on the stream that the context is given, in order with it; the current device stays."""
    import torch
    from bgtq import batched
    pool = Pool(device, "B", "q8", 64, 2, 40, 32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    k, v = _rows(1200, 2, 64, "float16", 1), _rows(1200, 2, 64, "float16", 2)
    with torch.cuda.stream(s):
        batched.bind_torch_stream(device)
        kd, vd = k.cuda(), v.cuda()
        slots = torch.arange(1200, device="cuda")
        batched.paged_write(device, pool.handle, slots, kd, vd)
        ko = torch.empty_like(kd, dtype=torch.float32)
        vo = torch.empty_like(ko)
        batched.paged_read(device, pool.handle, slots, ko, vo)
        s.synchronize()
        _check_read(pool, oracle, np.arange(1200), ko, vo)
    batched.bind_torch_stream(device)
    assert torch.cuda.current_device() == 0
    pool.destroy()


def test_refusals_on_the_gpu(device):
    """What the Python wrappers refuse before any call."""
    import torch
    import bgtq
    from bgtq import batched
    pool = Pool(device, "f16", "f16", 64, 2, 4, 32)
    x = torch.zeros((3, 2, 64), device="cuda")
    slots = torch.arange(3, device="cuda")
    for bad in (dict(k=x[:2], v=x), dict(k=x, v=x.double()), dict(k=x.cpu(), v=x), dict(k=x.transpose(1, 2), v=x)):
        with pytest.raises(bgtq.RangeError):
            batched.paged_write(device, pool.handle, slots, **bad)
    with pytest.raises(bgtq.RangeError):
        batched.paged_write(device, pool.handle, slots.int(), x, x)
    with pytest.raises(bgtq.RangeError):
        batched.paged_read(device, pool.handle, slots)
    batched.paged_write(device, pool.handle, slots[:0], x[:0], x[:0])  # nothing to do
    q, ln = torch.zeros((2, 4, 64), device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    table = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    for bad in (dict(max_length=97), dict(lengths=ln[:1]), dict(q=q[:, :, :32]), dict(page_table=table.long()), dict(out=q[:1])):
        with pytest.raises(bgtq.RangeError):
            batched.paged_decode_desc(**{**dict(pages=pool.handle, q=q, out=q.clone(), lengths=ln, page_table=table), **bad})
    with pytest.raises(bgtq.RangeError):  # no workspace
        batched.paged_decode(device, batched.paged_decode_desc(pages=pool.handle, q=q, out=q.clone(), lengths=ln, page_table=table))
    pool.destroy()


def test_prompts_to_pages_to_steps(device, oracle):
    """The operators as a server runs them for a layer: packed prompts attend to themselves, their rows enter the pages,
    then tokens are appended and attended to, against 64 bits over the rows the cache holds."""
    import torch
    from bgtq import batched
    rng = np.random.RandomState(12)
    pool = Pool(device, "S", "q8", 64, 3, 24, 64)
    prompts = [70, 1, 0, 257]
    total, D, H, Hq = sum(prompts), 64, 3, 9
    x = _rows(total, Hq + 2 * H, D, "bfloat16", 5)
    xd = x.cuda()
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(prompts)]), dtype=torch.int32, device="cuda")
    out = torch.empty((total, Hq, D), dtype=torch.bfloat16, device="cuda")
    batched.prompt_attention(device, xd[:, :Hq], xd[:, Hq:Hq + H], xd[:, Hq + H:], offsets, out)
    table = _table(pool, [n + 3 for n in prompts], rng)
    tab = table.cpu().numpy().astype(np.int64)
    slot = lambda b, t: tab[b, t // 64] * 64 + t % 64  # noqa: E731
    slots = np.concatenate([slot(b, np.arange(n)) for b, n in enumerate(prompts)]).astype(np.int64)
    batched.paged_write(device, pool.handle, torch.from_numpy(slots).cuda(), xd[:, Hq:Hq + H], xd[:, Hq + H:])
    torch.cuda.synchronize()
    _check_write(pool, oracle, slots, x[:, Hq:Hq + H], x[:, Hq + H:])
    at = 0
    for n in prompts:
        q, k, v = (a[at:at + n].double().numpy() for a in (x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]))
        for h in range(Hq if n else 0):
            s = q[:, h] @ k[:, h // 3].T / 8
            s[np.triu_indices(n, 1)] = -np.inf
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            ref, size = p @ v[:, h // 3], p @ np.abs(v[:, h // 3])
            got = out[at:at + n, h].double().cpu().numpy()
            assert np.all(np.abs(got - ref) <= 2.0 ** -8 * (size + np.abs(ref)) + 2.0 ** -14 * size + 1e-6)
        at += n
    lengths = list(prompts)
    for step in range(3):
        k, v, q = _rows(4, H, D, "bfloat16", step, 1), _rows(4, H, D, "bfloat16", step, 2), _rows(4, Hq, D, "float32", step, 3).cuda()
        batched.paged_write(device, pool.handle, torch.tensor([slot(b, n) for b, n in enumerate(lengths)], device="cuda"), k.cuda(), v.cuda())
        lengths = [n + 1 for n in lengths]
        o = _decode(pool, q, lengths, table)
        torch.cuda.synchronize()
        _check(o, _reference(pool, oracle, q, lengths, table), f"step {step}")
    pool.destroy()


@pytest.mark.parametrize("layout,dim,heads", [("B", 64, 2), ("B", 128, 2), ("f16", 64, 3)])
@pytest.mark.parametrize("rows,dtype", [(20, "float32"), (6000, "float16"), (6001, "float32")])
def test_largest_values_in_8_bits_stay_finite(device, oracle, layout, dim, heads, rows, dtype):
    """Rows up to FP16's largest value: the scale is at most 515.5 (516 times 127 rounds to an infinity), codes pass no
    127, every value comes back finite and within half a scale (and its FP16 rounding), and the decode over them is finite."""
    import torch
    from bgtq import batched
    print(layout, dim, rows, dtype, flush=True)
    pages = -(-rows // 32) + 1
    pool = Pool(device, layout, "q8", dim, heads, pages, 32)
    k, v = _rows(rows, heads, dim, dtype, 1), _rows(rows, heads, dim, dtype, 2).clamp(-4, 4) * 15000.0
    tops = [65504.0, -65504.0, 65472.0, -65472.0, 65440.0, 65408.0, 32752.0]
    tops += [65519.0, 65488.0, 65456.0] if dtype == "float32" else []  # these round to FP16's last values
    for i in range(0, rows, 2):
        v[i, i % heads, i % dim] = tops[i // 2 % len(tops)]
    slots = torch.arange(rows, device="cuda")
    batched.paged_write(device, pool.handle, slots, k.cuda(), v.cuda())
    torch.cuda.synchronize()
    v16 = v.half().numpy()
    assert np.all(np.isfinite(v16))
    pg, at = np.divmod(np.arange(rows), 32)
    got = {}
    for out in ("float32", "float16", "bfloat16"):
        got[out] = torch.empty((rows, heads, dim), dtype=getattr(torch, out), device="cuda")
        batched.paged_read(device, pool.handle, slots, v=got[out])
    torch.cuda.synchronize()
    for h in range(heads):
        _, s = _quantise(v16[:, h])
        s = np.minimum(s, np.float16(515.5)).astype(np.float64)
        codes = np.rint(v16[:, h].astype(np.float64) / s[:, None])
        assert np.abs(codes).max() == 127
        assert np.array_equal(pool.v_scales[:, h].cpu().numpy()[pg, at].astype(np.float64), s)
        assert np.array_equal(pool.v[:, h].cpu().numpy()[pg, at].astype(np.float64), codes)
        value = (codes * s[:, None]).astype(np.float16)
        assert np.all(np.isfinite(value))
        for out, x in got.items():
            assert torch.equal(x[:, h].cpu(), torch.from_numpy(value).to(x.dtype)), f"{out} V of head {h}"
        err = np.abs(value.astype(np.float64) - v16[:, h].astype(np.float64))
        assert np.all(err <= s[:, None] / 2 + np.abs(value.astype(np.float64)) * 2.0 ** -11)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    q = _rows(1, heads * 3, dim, "float32", 4).cuda()
    out = _decode(pool, q, [rows], table)
    torch.cuda.synchronize()
    ref = _reference(pool, oracle, q, [rows], table)
    assert np.all(np.isfinite(ref))
    # values up to 2^16 of either sign cancel: the tolerance is relative to what is summed
    err = np.abs(out.double().cpu().numpy() - ref)
    assert np.all(err <= ATOL + RTOL * 65504.0), f"max err {err.max():.3e}"
    pool.destroy()


@pytest.mark.parametrize("layout,dim", [("B", 64), ("A", 64), ("B", 128)])
@pytest.mark.parametrize("factor", [1.0, 3.7, 6.0, 300.0, 0.02])
def test_rotations_that_are_not_orthogonal(device, oracle, layout, dim, factor):
    """Tables take any finite transform: rows under a scaled one are written, read back and attended to as the
    definition has them, entries of any size."""
    import dataclasses
    import torch
    import bgtq
    from bgtq import batched
    print(layout, dim, factor, flush=True)
    pool = Pool(device, layout, "q8", dim, 2, 9, 32)
    pool.destroy()
    p = dataclasses.replace(pool.params[0], rotation=(np.asarray(pool.params[0].rotation) * np.float32(factor)).astype(np.float32))
    pool.params, pool.tables = [p, p], [bgtq.Tables(device, p) for _ in range(2)]
    pool.handle = batched.pages(page_tokens=32, tables=pool.tables, packed=pool.packed, norms=pool.norms, v=pool.v, v_scales=pool.v_scales)
    n = 9 * 32
    slots = np.arange(n)
    k, v = _rows(n, 2, dim, "float16", 5), _rows(n, 2, dim, "float16", 6)
    batched.paged_write(device, pool.handle, torch.arange(n, device="cuda"), k.cuda(), v.cuda())
    torch.cuda.synchronize()
    _check_write(pool, oracle, slots, k, v)
    for out in ("float32", "bfloat16"):
        ko, vo = (torch.empty((n, 2, dim), dtype=getattr(torch, out), device="cuda") for _ in range(2))
        batched.paged_read(device, pool.handle, torch.arange(n, device="cuda"), ko, vo)
        torch.cuda.synchronize()
        _check_read(pool, oracle, slots, ko, vo)
    q = (_rows(1, 6, dim, "float32", 7) / max(1.0, factor)).cuda()  # (logits of a few units)
    table = torch.arange(9, dtype=torch.int32, device="cuda")[None]
    out = _decode(pool, q, [270], table)
    torch.cuda.synchronize()
    _check(out, _reference(pool, oracle, q, [270], table))
    pool.destroy()


@pytest.mark.parametrize("layout,v,dim,heads,page", [("S", "q8", 64, 3, 64), ("B", "q8", 64, 2, 32), ("A", "f16", 64, 2, 256),
                                                     ("B", "f16", 128, 2, 64), ("A", "q8", 128, 1, 32)])
@pytest.mark.parametrize("rows,scattered", [(39, False), (40, True), (9003, False), (8200, True)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_non_finite_keys(device, oracle, layout, v, dim, heads, page, rows, scattered, dtype):
    """K rows with infinities and NaNs (and FP32 and BF16 values that FP16 does not hold) among others: a wave's
    row, and the tile encoder's second pass, whose blocks have skipped slots and end inside a tile. Each keeps to its
    groups as in an encode call of few rows; no other slot changes."""
    import torch
    from bgtq import batched
    from test_gpu_encode import _encode_nonfinite
    print(layout, dim, rows, scattered, dtype, flush=True)
    pages = -(-rows // page) + 2
    pool = Pool(device, layout, v, dim, heads, pages, page, gap=16)
    rng = np.random.RandomState(rows + dim)
    slots = (rng.permutation(pages * page)[:rows] if scattered else np.arange(rows) + 5).astype(np.int64)
    k, val = _rows(rows, heads, dim, dtype, rows, 1, 2.0), _rows(rows, heads, dim, dtype, rows, 2)
    odd = np.unique(np.concatenate([rng.choice(rows, min(rows, 50), replace=False)[:max(8, rows // 200)], [0, rows - 1, rows - 2]]))
    kinds = [float("inf"), -float("inf"), float("nan")] + ([1e6, -70000.0] if dtype != "float16" else [])
    for r in odd:
        for h in range(heads):
            for c in rng.choice(dim, rng.choice([0, 1, 1, 2, dim // 3]), replace=False):
                k[r, h, c] = kinds[rng.randint(len(kinds))]
    k[odd[1]] = float("inf")
    given = slots.copy()
    skipped = np.unique(np.concatenate([odd[::4] if rows > 100 else odd[3:5], odd[2:3] + 1])) % rows
    given[skipped] = rng.choice([-1, pages * page, 2 ** 40], len(skipped))
    kept = np.ones(rows, bool)
    kept[skipped] = False
    before = pool.snapshot()
    batched.paged_write(device, pool.handle, torch.from_numpy(given).cuda(), k.cuda(), val.cuda())
    torch.cuda.synchronize()
    k16 = k.half().numpy()
    for h, p in enumerate(pool.params):
        got_p, got_n = pool.k_bytes(h, slots[kept])
        want_p, want_n = _encode_nonfinite(oracle, p, np.ascontiguousarray(k16[kept, h]).view(np.uint16), True)
        got_n, want_n = got_n.view(np.uint16), np.asarray(want_n).view(np.uint16)
        same = (got_n == want_n) | (np.isnan(got_n.view(np.float16)) & np.isnan(want_n.view(np.float16)))
        bad = np.nonzero(np.any(got_p != want_p, 1) | ~same.all(1))[0]
        assert bad.size == 0, f"head {h}: {bad.size} rows differ, first {np.nonzero(kept)[0][bad[:5]]}"
    mask = torch.zeros(pages * page, dtype=torch.bool)
    mask[slots[kept]] = True
    keep = ~mask.view(pages, page).cuda()
    now = pool.snapshot()
    for h, p in enumerate(pool.params):
        for x, y, w in ((before[2], now[2], p.rowBytes), (before[3], now[3], p.normStride)):
            x, y = (a[:, h, :page * w].reshape(pages, page, w)[keep] for a in (x, y))
            assert _same_bits(x, y)
        assert _same_bits(before[0][:, h][keep], now[0][:, h][keep])
    pool.destroy()


def _relay(pool, heads_first):
    """The pool's arrays in other storage: heads outermost, or pages with other pages between them."""
    import torch
    from bgtq import batched

    def again(t):
        if t is None:
            return None
        if heads_first:
            return torch.empty((t.shape[1], t.shape[0], *t.shape[2:]), dtype=t.dtype, device="cuda").transpose(0, 1).copy_(t)
        n = (int(np.prod(t.shape[2:])) * t.element_size() + 15) // 16 * 16 // t.element_size()
        flat = torch.empty((t.shape[0], 3, t.shape[1], n), dtype=t.dtype, device="cuda")[:, 1, :, :int(np.prod(t.shape[2:]))]
        return flat.unflatten(2, t.shape[2:]).copy_(t)
    pool.v, pool.v_scales, pool.packed, pool.norms, pool.k = (again(t) for t in (pool.v, pool.v_scales, pool.packed, pool.norms, pool.k))
    pool.handle = batched.pages(page_tokens=pool.page, tables=pool.tables or None, packed=pool.packed, norms=pool.norms,
                                k_f16=pool.k, v=pool.v, v_scales=pool.v_scales)


@pytest.mark.parametrize("layout,v,dim,heads,page", [("S", "q8", 64, 3, 64), ("B", "q8", 64, 16, 32), ("B", "f16", 128, 2, 4096), ("f16", "q8", 64, 2, 32),
                                                     ("f16", "f16", 128, 3, 128)])
@pytest.mark.parametrize("heads_first", [True, False])
def test_other_pool_strides(device, oracle, layout, v, dim, heads, page, heads_first):
    """Heads outermost, or a pool inside a larger one; few and many rows; a page table inside a wider one, lengths of
    uint32; 16 KV heads of 16 query heads."""
    import torch
    from bgtq import batched
    print(layout, v, dim, heads, page, heads_first, flush=True)
    pages = 4 if page == 4096 else 12000 // page // heads + 3
    pool = Pool(device, layout, v, dim, heads, pages, page)
    _relay(pool, heads_first)
    n, rng = pages * page, np.random.RandomState(1)
    k, val = _rows(n, heads, dim, "bfloat16", 1), _rows(n, heads, dim, "float32", 2)
    slots = rng.permutation(n)
    few = 37
    for part in (slice(0, few), slice(few, n)):
        batched.paged_write(device, pool.handle, torch.from_numpy(slots[part].copy()).cuda(), k[part].cuda(), val[part].cuda())
    torch.cuda.synchronize()
    _check_write(pool, oracle, slots, k, val)
    sd = torch.from_numpy(slots).cuda()
    ko, vo = torch.empty((n, heads, dim), device="cuda"), torch.empty((n, heads, dim), device="cuda")
    batched.paged_read(device, pool.handle, sd, ko, vo)
    torch.cuda.synchronize()
    _check_read(pool, oracle, slots, ko, vo)
    G = 16 if heads == 16 else 3
    lengths = [min(page * 2 - 5, 300), 0, page + 1]
    wide = torch.full((3, 9), 2 ** 31 - 1, dtype=torch.int32)
    wide[0, 2:4], wide[2, 2:4] = torch.tensor([1, 3]), torch.tensor([2, 0])
    table = wide.cuda()[:, 2:5]
    q = _rows(3, heads * G, dim, "float32", 3).cuda()
    out = torch.full_like(q, float("nan"))
    args = dict(pages=pool.handle, q=q, out=out, lengths=torch.tensor(lengths, dtype=torch.uint32, device="cuda"), page_table=table)
    ws = torch.zeros(batched.paged_decode_workspace_bytes(batched.paged_decode_desc(**args)), dtype=torch.uint8, device="cuda")
    batched.paged_decode(device, batched.paged_decode_desc(workspace=ws, **args))
    torch.cuda.synchronize()
    _check(out, _reference(pool, oracle, q, lengths, table))
    pool.destroy()


@pytest.mark.parametrize("batch", [200, 1100])
def test_decode_of_many_sequences(device, oracle, batch):
    """More sequences than share workgroups by their lengths, and more (sequence, head) units than the counters' prefix
    holds, twice in one workspace."""
    import torch
    from bgtq import batched
    rng = np.random.RandomState(batch)
    pool = Pool(device, "B", "q8", 64, 1, 64, 32)
    _fill(pool, 2)
    table = torch.from_numpy(rng.randint(0, 64, (batch, 24)).astype(np.int32)).cuda()
    lengths = [int(x) for x in rng.randint(0, 24 * 32 + 1, batch)]
    q = _rows(batch, 2, 64, "float32", 3).cuda()
    outs = [_decode(pool, q, lengths, table) for _ in range(2)]
    torch.cuda.synchronize()
    assert torch.equal(*outs)
    some = [0, 1, batch // 2, batch - 1] + [int(x) for x in rng.randint(0, batch, 40)]
    ref = _reference(pool, oracle, q[some], [lengths[i] for i in some], table[some])
    _check(outs[0][some], ref)
    assert bool((outs[0][[i for i, n in enumerate(lengths) if n == 0]] == 0).all())
    pool.destroy()


def test_two_contexts_at_once(device, oracle):
    """Two contexts on two streams write different rows of one pool, neighbours in memory among them, while one of
    them decodes; neither touches the other's rows."""
    import torch
    import bgtq
    from bgtq import batched
    pool = Pool(device, "S", "q8", 64, 3, 130, 64)
    other = bgtq.Device(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    n = 130 * 64
    k, v = _rows(n, 3, 64, "float16", 1), _rows(n, 3, 64, "float16", 2)
    kd, vd = k.cuda(), v.cuda()
    slots = torch.arange(n, device="cuda")
    table = torch.arange(128, dtype=torch.int32, device="cuda").view(4, 32)
    q = _rows(4, 9, 64, "float32", 3).cuda()
    torch.cuda.synchronize()
    pool2 = batched.pages(page_tokens=64, tables=pool.tables, packed=pool.packed, norms=pool.norms, v=pool.v, v_scales=pool.v_scales)
    odd = [torch.arange(n, device="cuda")[i::2] for i in range(2)]
    parts = [(slots[o], kd[o].contiguous(), vd[o].contiguous()) for o in odd]
    torch.cuda.synchronize()
    for dev, s in zip((device, other), streams):
        dev.set_stream(s.cuda_stream)
    for dev, handle, (at, kk, vv) in zip((device, other), (pool.handle, pool2), parts):
        batched.paged_write(dev, handle, at, kk, vv)
    torch.cuda.synchronize()
    _check_write(pool, oracle, np.arange(n), k, v)
    outs = [torch.empty_like(q) for _ in range(2)]
    descs = []
    for handle, o in zip((pool.handle, pool2), outs):
        args = dict(pages=handle, q=q, out=o, lengths=torch.tensor([2048, 100, 0, 1999], dtype=torch.int32, device="cuda"), page_table=table)
        ws = torch.zeros(batched.paged_decode_workspace_bytes(batched.paged_decode_desc(**args)), dtype=torch.uint8, device="cuda")
        descs.append(batched.paged_decode_desc(workspace=ws, **args))
    torch.cuda.synchronize()
    for _ in range(3):
        for dev, d in zip((device, other), descs):
            batched.paged_decode(dev, d)
    torch.cuda.synchronize()
    assert torch.equal(*outs)
    _check(outs[0], _reference(pool, oracle, q, [2048, 100, 0, 1999], table))
    batched.bind_torch_stream(device)
    other.destroy()
    pool.destroy()


@pytest.mark.parametrize("layout,v,rows", [("S", "q8", 6000), ("f16", "f16", 500), ("B", "q8", 3)])
def test_write_and_read_captured(device, oracle, layout, v, rows):
    """A graph of a write and the read back, replayed with other rows and slots."""
    import torch
    from bgtq import batched
    heads = 3 if layout == "S" else 2
    pool = Pool(device, layout, v, 64, heads, rows // 64 + 3, 64)
    n = (rows // 64 + 3) * 64
    slots = torch.zeros(rows, dtype=torch.int64, device="cuda")
    k, val, ko, vo = (torch.empty((rows, heads, 64), device="cuda") for _ in range(4))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        device.set_stream(side.cuda_stream)
        batched.paged_write(device, pool.handle, slots, k, val)
        batched.paged_read(device, pool.handle, slots, ko, vo)
    batched.bind_torch_stream(device)
    for step in range(4):
        s = np.random.RandomState(step).permutation(n)[:rows]
        nk, nv = _rows(rows, heads, 64, "float32", step, 1), _rows(rows, heads, 64, "float32", step, 2)
        slots.copy_(torch.from_numpy(s)), k.copy_(nk), val.copy_(nv)
        graph.replay()
        torch.cuda.synchronize()
        _check_write(pool, oracle, s, nk, nv)
        _check_read(pool, oracle, s, ko, vo)
        again = [torch.empty_like(ko), torch.empty_like(vo)]
        batched.paged_read(device, pool.handle, slots, *again)
        torch.cuda.synchronize()
        assert torch.equal(again[0], ko) and torch.equal(again[1], vo)
    pool.destroy()
