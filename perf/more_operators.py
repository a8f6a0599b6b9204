"""Performance cases of a model step over the paged cache: rotation, append, chunks and windows.

Four operators that a serving loop calls per layer with the rows of its
projections: head norms and position rotation of queries and keys in one pass;
the same with the rotated keys and the values entering the paged cache on the
way; attention of chunks of new tokens (one token to whole chunks, mixed in a
batch) over the pages; and attention with a sliding window and a few first
tokens that stay visible, for single tokens over pages and for prompts.
Geometries are those of the repository's own benchmark and tests: SmolLM2-135M
(9 query / 3 KV heads, d=64, its calibration tables: layout "S"), Qwen2.5-0.5B
(14 / 2 heads, d=64) and d=128 heads; layout "B" has a 4-bit and an 8-bit group
of equal size, "f16" pages hold plain FP16 K.

Rotation: the pairs are (i, i + dim / 2), with table row p holding the cosines
of position p's dim / 2 angles, then the sines, in FP32. A head's norm divides
its row by sqrt(mean(x^2) + eps) and multiplies by a weight per dimension.
Window w with s sinks: position p sees token t <= p where t > p - w or t < s.
A page holds `page` tokens of every KV head; a slot is page * page_tokens +
place. V rows are FP16, or ("q8") 8-bit codes c with one FP16 scale s per row,
s = max|v| / 127 rounded up, c = round(v / s), standing for the FP16 value
nearest s c.
"""
from __future__ import annotations

import json
import math
import os
import sys

import numpy as np
import torch

own = False  # set by the tools: plain torch (False) or the library's calls (True)

CALIBRATION = os.path.join(os.getcwd(), "tests", "golden", "reference", "model")
EPS = 1e-6
POSITIONS = 32768  # rows of the rotation table


def listed():
    return [
        # One token's queries and keys of a SmolLM2 layer: latency.
        dict(name="rotate_one", kind="rotate", dtype="f32", dim=64, q_heads=9, kv_heads=3, rows=1, norm=False),
        # A batch's prompt rows (Qwen geometry), slices of a fused projection, with head norms: memory bound.
        dict(name="rotate_prompt", kind="rotate", dtype="bf16", dim=64, q_heads=14, kv_heads=2, rows=16384, norm=True),
        # One token of one sequence enters the cache of a SmolLM2 layer: latency.
        dict(name="append_one_cal", kind="append", layout="S", v="q8", dim=64, q_heads=9, kv_heads=3, rows=1, dtype="f32",
             norm=False, page=64),
        # A batch's prompts enter the cache of a layer (Qwen geometry), heads normed.
        dict(name="append_prompt", kind="append", layout="B", v="q8", dim=64, q_heads=14, kv_heads=2, rows=16384,
             dtype="bf16", norm=True, page=64),
        # An odd number of rows of wide heads on FP16 pages.
        dict(name="append_d128", kind="append", layout="f16", v="f16", dim=128, q_heads=16, kv_heads=4, rows=5003,
             dtype="f16", norm=True, page=32),
        # Continuous batching (SmolLM2 on its calibration tables): some sequences bring parts of their prompts, most one token.
        dict(name="chunk_mixed", kind="chunk", layout="S", v="q8", dim=64, q_heads=9, kv_heads=3, dtype="f16", sequences=13,
             rows=301, mix=True, ctx=8001, window=0, sinks=0, page=64),
        # The last 2048 rows of a long prompt (Qwen geometry): the largest, matrix-core work.
        dict(name="chunk_long", kind="chunk", layout="B", v="q8", dim=64, q_heads=14, kv_heads=2, dtype="bf16", sequences=1,
             rows=2048, mix=False, ctx=32768, window=0, sinks=0, page=64),
        # A few drafted tokens of each sequence are verified at once: wide heads, FP16 pages.
        dict(name="chunk_verify", kind="chunk", layout="f16", v="f16", dim=128, q_heads=16, kv_heads=4, dtype="bf16",
             sequences=16, rows=5, mix=False, ctx=4099, window=0, sinks=0, page=128),
        # A chunk of one sequence behind a window, short pages.
        dict(name="chunk_window", kind="chunk", layout="B", v="q8", dim=128, q_heads=8, kv_heads=8, dtype="bf16", sequences=2,
             rows=1000, mix=False, ctx=9001, window=2048, sinks=16, page=32),
        # One layer of a batch-1 SmolLM2 step behind a window: latency.
        dict(name="decode_one_window", kind="decode", layout="S", v="q8", dim=64, q_heads=9, kv_heads=3, batch=1, ctx=8001,
             ragged=False, window=1024, sinks=4, page=64),
        # 64 sequences of up to 32768 tokens behind a window (Qwen geometry), odd lengths, an empty one among them.
        dict(name="decode_b64_window", kind="decode", layout="B", v="q8", dim=64, q_heads=14, kv_heads=2, batch=64, ctx=32768,
             ragged=True, window=4096, sinks=4, page=64),
        # A batch of prompts of mixed odd lengths behind a window (Qwen geometry).
        dict(name="prompt_window", kind="prompt", dtype="bf16", dim=64, q_heads=14, kv_heads=2, sequences=11, longest=2777,
             window=511, sinks=4),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of lo..hi, both ends included."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "append", "chunk", "chunk", "chunk", "decode", "prompt"])
    dim = rng.choice([64, 64, 128])
    if kind in ("rotate", "prompt"):
        q, kv = rng.choice([(9, 3), (14, 2), (16, 4), (8, 8), (4, 1)])
        if kind == "rotate":
            return dict(kind=kind, dtype=rng.choice(["f32", "f16", "bf16"]), dim=dim, q_heads=q, kv_heads=kv,
                        rows=_log(rng, 1, 16384), norm=rng.random() < 0.5)
        longest = _log(rng, 1, 6000)
        return dict(kind=kind, dtype=rng.choice(["f16", "bf16"]), dim=dim, q_heads=q, kv_heads=kv,
                    sequences=_log(rng, 1, max(1, min(200, (1 << 27) // (longest * longest)))), longest=longest,
                    window=_log(rng, 1, 4096), sinks=rng.choice([0, 4, 33]))
    layout = rng.choice(["S", "S", "B", "B", "f16"]) if dim == 64 else rng.choice(["B", "f16"])
    kv, g = (3, 3) if layout == "S" else rng.choice([(1, 1), (1, 3), (2, 7), (4, 4), (8, 1)])
    v, page = rng.choice(["q8", "q8", "f16"]), rng.choice([32, 64, 64, 256])
    if kind == "append":
        return dict(kind=kind, layout=layout, v=v, dim=dim, q_heads=kv * g, kv_heads=kv, rows=_log(rng, 1, 16384),
                    dtype=rng.choice(["f32", "f16", "bf16"]), norm=rng.random() < 0.5, page=page)
    ctx = _log(rng, 1, 32768)
    window, sinks = rng.choice([(0, 0), (_log(rng, 1, 8192), rng.choice([0, 4, 33]))])
    if kind == "decode":
        return dict(kind=kind, layout=layout, v=v, dim=dim, q_heads=kv * g, kv_heads=kv,
                    batch=_log(rng, 1, max(1, min(200, (1 << 21) // (kv * ctx)))), ctx=ctx, ragged=rng.random() < 0.7,
                    window=window or _log(rng, 1, 8192), sinks=sinks, page=page)
    rows = _log(rng, 1, min(ctx, 2048))
    most = (1 << 28) // (rows * g * ctx)
    return dict(kind=kind, layout=layout, v=v, dim=dim, q_heads=kv * g, kv_heads=kv, dtype=rng.choice(["f16", "bf16"]),
                sequences=_log(rng, 1, max(1, min(100, most, (1 << 20) // ctx))), rows=rows, mix=rng.random() < 0.5, ctx=ctx,
                window=window, sinks=sinks, page=page)


DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- calibration tables and the rotation's: what a program loads once

_CACHE: dict = {}


def _once(key, make):
    if key not in _CACHE:
        _CACHE[key] = make()
    return _CACHE[key]


def _blobs(layout, dim, head):
    """A KV head's serialised tables (integers, floats): the SmolLM2 calibration's, or layout B's."""
    if layout == "S":
        def load():
            with open(os.path.join(CALIBRATION, "calibration.json"), encoding="utf-8") as f:
                meta = json.load(f)
            return meta["arrays"], np.fromfile(os.path.join(CALIBRATION, meta["binary"]), np.uint8)
        arrays, payload = _once("calibration", load)
        part = [payload[a["offset"]:a["offset"] + a["nbytes"]] for a in (arrays[f"h{head}_config"], arrays[f"h{head}_table"])]
        return part[0].view(np.uint32), part[1].view(np.float32)

    def make():
        m, pairs = dim // 2, dim // 2
        low = [i for i in range(pairs) if i >= pairs // 2]  # the low-energy frequency pairs take the 4-bit group
        high = [i for i in range(pairs) if i < pairs // 2]
        perm = [d for p in (low, high) for d in [*p, *(i + pairs for i in p)]]
        rot, cent = np.zeros((dim, dim)), np.zeros((dim, 256))
        lut, off, inv = [], np.zeros(dim), np.zeros(dim)
        for g, n in enumerate((16, 256)):
            q, r = np.linalg.qr(np.random.RandomState(42 + g).standard_normal((m, m)))
            s = slice(g * m, (g + 1) * m)
            rot[s, s] = q * np.sign(np.diag(r))
            # the quantiser of least squared error for many codes: quantiles of the normal density's cube root
            u = torch.special.ndtri((torch.arange(n, dtype=torch.float64) + 0.5) / n).numpy()
            c = math.sqrt(3.0 / m) * u
            cent[s, :n] = c
            width = (c[-1] - c[0]) * 1.02 / 256
            off[s], inv[s] = c[0] - 0.01 * (c[-1] - c[0]), 1 / width
            centres = off[g * m] + (np.arange(256) + 0.5) * width
            lut.append(np.abs(centres[:, None] - c[None]).argmin(1))
        ints = [dim, 2, dim * 3 // 4, 2, m, 256, 10, 10 + dim, 10 + 2 * dim, 10 + 3 * dim, *perm, *([0] * m + [1] * m),
                *([0] * m + [1] * m), *np.concatenate(lut)]
        return (np.asarray(ints, np.uint32),
                np.concatenate([x.reshape(-1) for x in (rot, cent, off, inv)]).astype(np.float32))
    return _once(("B", dim), make)


class _Book:
    """A KV head's tables as torch tensors on the GPU."""

    def __init__(self, ints, floats):
        def t(x, dtype):
            return torch.as_tensor(np.ascontiguousarray(x).astype(dtype), device="cuda")
        c = ints.astype(np.int64)
        d = self.dim = int(c[0])
        self.groups, self.row_bytes, self.norm_stride, self.nib, mc = (int(x) for x in c[1:6])
        self.perm, self.group_of, self.pos_cb = (t(c[c[k]:c[k] + d], np.int64) for k in (6, 7, 8))
        self.lut = t(c[c[9]:], np.int64)
        self.rot, self.cent = t(floats[:d * d], np.float32).reshape(d, d), t(floats[d * d:d * d + d * mc], np.float32).reshape(d, mc)
        self.off, self.inv = t(floats[d * d + d * mc:][:d], np.float32), t(floats[d * d + d * mc + d:][:d], np.float32)
        self.sizes = torch.bincount(self.group_of).tolist()
        self.pos = torch.arange(d, device="cuda")


def _books(case):
    if case.get("layout", "f16") == "f16":
        return []
    key = lambda h: (case["layout"], case["dim"], h if case["layout"] == "S" else 0)  # noqa: E731
    return [_once(("book", key(h)), lambda h=h: _Book(*_blobs(case["layout"], case["dim"], h))) for h in range(case["kv_heads"])]


def _table(dim):
    """Cosines and sines of the positions' angles, base 10^6, from angles in 64 bits."""
    def make():
        freq = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
        angle = torch.arange(POSITIONS, dtype=torch.float64, device="cuda")[:, None] * freq
        return torch.cat([angle.cos(), angle.sin()], 1).float()
    return _once(("rotation", dim), make)


# ---- inputs

def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)
    return g


def _randn(seed, salt, *shape):
    return torch.randn(shape, generator=_gen(seed, salt), device="cuda")


def _energies(dim):
    """Frequency pairs whose energy decays geometrically, as a rotary model's keys have."""
    return (0.9 ** (torch.arange(dim, device="cuda") % (dim // 2)).double()).sqrt().float()


def _pool(case, pages):
    """An empty pool. K: rows of each head's own row bytes and norm stride from the start of its part of the page."""
    H, D, P, books = case["kv_heads"], case["dim"], case["page"], _books(case)
    z = lambda dtype, *s: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    pool = dict(v=z(torch.int8 if case["v"] == "q8" else torch.float16, pages, H, P, D))
    if case["v"] == "q8":
        pool["v_scales"] = z(torch.float16, pages, H, P)
    if books:
        pool["packed"] = z(torch.uint8, pages, H, P * max(b.row_bytes for b in books))
        pool["norms"] = z(torch.float16, pages, H, P * max(b.norm_stride for b in books))
    else:
        pool["k"] = z(torch.float16, pages, H, P, D)
    return pool


def _filled(case, pages, seed):
    """A pool whose every row holds what written rows hold: codes of rotated unit-norm groups, V of N(0, 1)."""
    pool, D = _pool(case, pages), case["dim"]
    n = pages * case["page"]
    for h, b in enumerate(_books(case)):
        sizes = torch.tensor(b.sizes, device="cuda", dtype=torch.float32)[b.group_of]
        y = _randn(seed, 10 + h, n, D) / sizes.sqrt()
        codes = b.lut[b.pos_cb * 256 + ((y - b.off) * b.inv).clamp(0, 255).long()]
        del y
        scales = (sizes.new_tensor(b.sizes).sqrt() * 1.5 * torch.exp(0.3 * _randn(seed, 50 + h, n, b.groups))).half()
        rows, norms = _pack(b, codes, scales)
        pool["packed"][:, h, :case["page"] * b.row_bytes] = rows.view(pages, -1)
        pool["norms"][:, h, :case["page"] * b.norm_stride] = norms.view(pages, -1)
    if "k" in pool:
        pool["k"].copy_(_randn(seed, 90, *pool["k"].shape) * _energies(D))
    v = _randn(seed, 91, *pool["v"].shape)
    if "v_scales" in pool:
        pool["v_scales"].copy_(v.abs().amax(-1) / 127)
        pool["v"].copy_((v / pool["v_scales"].float()[..., None]).round().clamp(-127, 127))
    else:
        pool["v"].copy_(v)
    return pool


def _permutation(n, seed):
    return np.random.RandomState(int(seed) % (1 << 31)).permutation(n)


def _lengths(case, seed):
    """Sequence lengths: all ctx, or spread evenly from an empty one to ctx, in an order of the seed's."""
    B, ctx = case["batch"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * B
    lens = [ctx * (i + 1) // B if i else 0 for i in range(B)]
    return [lens[i] for i in _permutation(B, seed)]


def _prompt_lengths(case, seed):
    """Prompt lengths: the longest, the others spread over its eighth and up, odd ones among them."""
    n, longest = case["sequences"], case["longest"]
    low = (longest + 7) // 8
    return [low + (longest - low) * (int(i) + 1) // n for i in _permutation(n, seed)]


def _chunks(case, seed):
    """(new rows, tokens with them) of each sequence, in an order of the seed's. Mixed: every fourth sequence brings a
    part of its prompt (rows down to half), one nothing at all, the others one token. Histories from none to the longest."""
    n, rows, ctx = case["sequences"], case["rows"], case["ctx"]
    got = []
    for i in range(n):
        c = rows if not case["mix"] else rows - (rows // 2) * i // n if i % 4 == 0 else 0 if i == 5 else 1
        got.append((c, c + (ctx - rows) * (n - i) // n if c else 0))
    return [got[i] for i in _permutation(n, seed)]


def _paged(case, lens, seed):
    """A filled pool and the page table of sequences that lie anywhere in it (-1: no page)."""
    P = case["page"]
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 3
    order = torch.from_numpy(_permutation(pages, seed))
    table = torch.full((len(lens), -(-case["ctx"] // P)), -1, dtype=torch.int32)
    for b, (at, n) in enumerate(zip(np.cumsum([0] + need), need)):
        table[b, :n] = order[at:at + n]
    return _filled(case, pages, seed), table.cuda()


def _places(lens):
    """Rows of packed sequences: [sequences, longest] indexes (past a sequence: its last row's, or any) and the offsets."""
    offsets = np.cumsum([0] + list(lens))
    index = [torch.arange(max(1, max(lens))).clamp(max=max(n - 1, 0)) + min(o, max(offsets[-1] - 1, 0)) for n, o in zip(lens, offsets)]
    return torch.stack(index).cuda(), torch.tensor(offsets, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    D, kind, seed = case["dim"], case["kind"], int(seed)
    Hq, Hkv = case["q_heads"], case["kv_heads"]
    st = dict(case=case)
    if kind == "prompt":
        lens = _prompt_lengths(case, seed)
        # the rows of a fused projection: queries, keys and values side by side
        x = _randn(seed, 1, sum(lens), Hq + 2 * Hkv, D).to(DTYPES[case["dtype"]])
        st.update(q=x[:, :Hq], k=x[:, Hq:Hq + Hkv], v=x[:, Hq + Hkv:], lens=lens, lengths=torch.tensor(lens, device="cuda"))
        st["out"] = torch.empty((sum(lens), Hq, D), dtype=x.dtype, device="cuda")
        st["index"], st["offsets"] = _places(lens)
    elif kind == "chunk":
        chunks = _chunks(case, seed)
        st["pool"], st["table"] = _paged(case, [n for _, n in chunks], seed)
        news = [c for c, _ in chunks]
        st["index"], st["offsets"] = _places(news)
        st.update(chunks=chunks, new=torch.tensor(news, device="cuda"),
                  lengths=torch.tensor([n for _, n in chunks], dtype=torch.int32, device="cuda"),
                  q=_randn(seed, 1, sum(news), Hq, D).to(DTYPES[case["dtype"]]))
        st["out"] = torch.empty_like(st["q"])
    elif kind == "decode":
        lens = _lengths(case, seed)
        st["pool"], st["table"] = _paged(case, lens, seed)
        st.update(lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"), q=_randn(seed, 1, case["batch"], Hq, D))
        st["out"] = torch.empty_like(st["q"])
    else:
        n = case["rows"]
        x = _randn(seed, 2, n, Hq + 2 * Hkv, D)
        x[:, Hq:Hq + Hkv] *= 3 * _energies(D)
        x = x.to(DTYPES[case["dtype"]])
        start = int(np.random.RandomState(seed % (1 << 31)).randint(0, POSITIONS - n + 1))
        st.update(q=x[:, :Hq], k=x[:, Hq:Hq + Hkv], v=x[:, Hq + Hkv:], table=_table(D),
                  positions=torch.arange(start, start + n, device="cuda"))
        st["weights"] = [1 + 0.1 * _randn(seed, 3 + i, D) for i in range(2)] if case["norm"] else [None, None]
        st["q_out"], st["k_out"] = torch.empty((n, Hq, D), dtype=x.dtype, device="cuda"), torch.empty((n, Hkv, D), dtype=x.dtype, device="cuda")
        if kind == "append":
            P = case["page"]
            pages = -(-n // P) + 3
            order = torch.from_numpy(_permutation(pages, seed)).cuda()  # consecutive tokens fill pages that lie anywhere
            t = torch.arange(n, device="cuda")
            st["slots"] = order[t // P] * P + t % P
            st["pool"], st["v_out"] = _pool(case, pages), torch.empty_like(st["k_out"])
    if own:  # the library's handles: tables on the device, the pool's description, a workspace
        _bind(st)
    return st


# ---- the plain forms

def _turned(x, weight, table, positions):
    """Rows [n, heads, dim] normed (weight given) and rotated, in FP32; a rotated pair is x1 cos - x2 sin and
    x2 cos + x1 sin with the second product rounded first, a norm's factor comes from sums in 64 bits: K enters a
    codec, where a value next to a code's border decides the code."""
    x, half = x.float(), x.shape[-1] // 2
    if weight is not None:
        mean = x.double().square().mean(-1, keepdim=True)
        x = (x * (mean + EPS).rsqrt().float()) * weight
    c, s = table[positions][:, None].split(half, -1)
    a, b = x.split(half, -1)
    mul = lambda u, v: u.double() * v.double()  # noqa: E731  (exact)
    return torch.cat([(mul(a, c) - (b * s).double()).float(), (mul(b, c) + (a * s).double()).float()], -1)


def _tree_sum(x):
    """FP32 sum over the last axis in the order that the codec's definition fixes: 8 lanes of 4 interleaved partials."""
    n, d = x.shape
    v = x.reshape(n, d // 32, 4, 8)
    a = v[:, 0]
    for i in range(1, d // 32):
        a = a + v[:, i]
    s = ((a[:, 0] + a[:, 1]) + a[:, 2]) + a[:, 3]
    t = s[:, 0]
    for lane in range(1, 8):
        t = t + s[:, lane]
    return t


def _encode(b, k):
    """FP16 rows [n, dim] -> codes [n, dim] and scales [n, groups]: the Block-GTQ encode. Which code a value gets is
    fixed by one FP32 rounding per step, so the steps are the definition's (through 64 bits, rounded at each)."""
    x = k.float()[:, b.perm]
    raw, den = [], torch.empty_like(x)
    for g in range(b.groups):
        mask = b.group_of == g
        n = (_tree_sum(torch.where(mask, x * x, 0.0)) + 1e-30).double().sqrt().float()
        if b.groups > 1:
            rep = _tree_sum(torch.where(mask, n[:, None], 0.0).expand(-1, b.dim).contiguous())
            raw.append((rep.double() / b.sizes[g]).float())
        else:
            raw.append(n)
        den[:, mask] = torch.where(n > 1e-10, n, 1.0)[:, None]
    xn = (x.double() / den.double()).float().double()
    y, r = torch.zeros_like(x), b.rot.double()
    for i in range(b.dim):
        y = torch.addcmul(y.double(), xn[:, i:i + 1], r[:, i][None]).float()
    codes = b.lut[b.pos_cb * 256 + ((y - b.off) * b.inv).clamp(0, 255).long()]
    c = b.cent[b.pos, codes]
    scales = []
    for g in range(b.groups):
        s = _tree_sum(torch.where(b.group_of == g, c * c, 0.0)).double().sqrt().float().clamp_min(1e-10)
        scales.append((raw[g].double() / s.double()).float())
    return codes, torch.stack(scales, 1).half()


def _pack(b, codes, scales):
    """Codes and scales -> rows uint8 [n, row_bytes] and scale rows FP16 [n, norm_stride], zero padded."""
    n, nib = codes.shape[0], b.nib
    rows = torch.zeros((n, b.row_bytes), dtype=torch.uint8, device=codes.device)
    rows[:, :nib // 2] = codes[:, 0:nib:2] | codes[:, 1:nib:2] << 4
    rows[:, nib // 2:nib // 2 + b.dim - nib] = codes[:, nib:]
    norms = torch.zeros((n, b.norm_stride), dtype=torch.float16, device=codes.device)
    norms[:, :b.groups] = scales
    return rows, norms


def _keys(case, pool, h, page, place, dtype=torch.float32):
    """Head h's K rows at (page, place), in the model's order of dimensions."""
    if "k" in pool:
        return pool["k"][page, h, place].to(dtype)
    b, P = _books(case)[h], case["page"]
    rows = pool["packed"][:, h, :P * b.row_bytes].unflatten(1, (P, b.row_bytes))[page, place].long()
    norms = pool["norms"][:, h, :P * b.norm_stride].unflatten(1, (P, b.norm_stride))[page, place]
    n, half = rows.shape[:-1], b.nib // 2
    codes = torch.cat([torch.stack([rows[..., :half] & 15, rows[..., :half] >> 4], -1).reshape(*n, b.nib),
                       rows[..., half:half + b.dim - b.nib]], -1)
    cs = b.cent.to(dtype)[b.pos, codes] * norms.to(dtype)[..., b.group_of]
    out = torch.empty_like(cs)
    out[..., b.perm] = torch.matmul(cs, b.rot.to(dtype))
    return out


def _values(pool, h, page, place):
    """Head h's V rows at (page, place): FP16 values."""
    v = pool["v"][page, h, place]
    return (v.float() * pool["v_scales"][page, h, place].float()[..., None]).half() if "v_scales" in pool else v


def _quantise_v(x):
    """FP16 rows -> (codes, scales): s = max|x| / 127 rounded up to FP16, c = round(x / s), ties to even."""
    top = x.float().abs().amax(-1)
    s = (top / 127).half()
    s = torch.where(s.float() * 127 < top, (s.view(torch.int16) + 1).view(torch.float16), s)
    return torch.where(s[..., None] > 0, x.double() / s.double()[..., None].clamp_min(1e-30), 0.0).round(), s


def _append(st):
    case, pool, P = st["case"], st["pool"], st["case"]["page"]
    page, place = st["slots"] // P, st["slots"] % P
    k, v = _turned(st["k"], st["weights"][1], st["table"], st["positions"]).half(), st["v"].half()
    for h, b in enumerate(_books(case)):
        rows, norms = _pack(b, *_encode(b, k[:, h]))
        pool["packed"][:, h, :P * b.row_bytes].unflatten(1, (P, b.row_bytes))[page, place] = rows
        pool["norms"][:, h, :P * b.norm_stride].unflatten(1, (P, b.norm_stride))[page, place] = norms
    if "k" in pool:
        pool["k"].transpose(1, 2)[page, place] = k
    if "v_scales" in pool:
        v, s = _quantise_v(v)
        pool["v_scales"].transpose(1, 2)[page, place] = s
    pool["v"].transpose(1, 2)[page, place] = v.to(pool["v"].dtype)
    heads = range(case["kv_heads"])
    back = [torch.stack([fn(h) for h in heads], 1).to(DTYPES[case["dtype"]])
            for fn in (lambda h: _keys(case, pool, h, page, place), lambda h: _values(pool, h, page, place))]
    return [_turned(st["q"], st["weights"][0], st["table"], st["positions"]).to(DTYPES[case["dtype"]]), *back]


def _seen(positions, tokens, window, sinks):
    """Whether each of `positions` sees each of `tokens` (a last axis of its own)."""
    p, t = positions[..., None], tokens
    seen = t <= p
    return seen & ((t > p - window) | (t < sinks)) if window else seen


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(dim)) over the seen entries, times v; rows that see nothing are zero."""
    logits = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(q.shape[-1])
    logits = torch.where(seen, logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def _over_pages(st, q, positions):
    """Queries [sequences, rows, heads, dim] at positions [sequences, rows] over the pages, in FP32."""
    case, pool, P = st["case"], st["pool"], st["case"]["page"]
    S, R, Hq, D = q.shape
    G = Hq // case["kv_heads"]
    t = torch.arange(case["ctx"], device="cuda")
    page, place = st["table"].long()[:, t // P].clamp_min(0), (t % P).expand(S, -1)
    seen = _seen(positions, t, case["window"], case["sinks"]).repeat(1, G, 1)
    outs = []
    for h in range(case["kv_heads"]):
        x = q[:, :, h * G:(h + 1) * G].float().transpose(1, 2).reshape(S, G * R, D)
        outs.append(_attend(x, _keys(case, pool, h, page, place), _values(pool, h, page, place).float(), seen).view(S, G, R, D))
    return torch.cat(outs, 1).transpose(1, 2)


def _decode(st):
    return _over_pages(st, st["q"][:, None], st["lengths"].long()[:, None] - 1)[:, 0]


def _chunk(st):
    r = torch.arange(st["index"].shape[1], device="cuda")
    inside = r < st["new"][:, None]
    positions = (st["lengths"].long() - st["new"])[:, None] + r
    return _over_pages(st, st["q"][st["index"]], torch.where(inside, positions, -1))[inside]


def _prompt(st):
    case = st["case"]
    G = case["q_heads"] // case["kv_heads"]
    q, k, v = (st[x][st["index"]].float().transpose(1, 2) for x in ("q", "k", "v"))  # [sequence, head, place, dim]
    k, v = (x.repeat_interleave(G, 1) for x in (k, v))
    t = torch.arange(q.shape[2], device="cuda")
    return _attend(q, k, v, _seen(t, t, case["window"], case["sinks"])).transpose(1, 2)[t < st["lengths"][:, None]]


# ---- the library's calls

def _library():
    def make():
        sys.path.insert(0, os.path.join(os.getcwd(), "block-gqt-webgpu_amd"))
        import bgtq
        from bgtq import batched
        dev = bgtq.Device(0)
        batched.bind_torch_stream(dev)
        return bgtq, batched, dev
    return _once("library", make)


def _bind(st):
    case, kind = st["case"], st["case"]["kind"]
    bgtq, batched, dev = _library()
    if kind in ("rotate", "append"):
        st["rope"] = batched.rope(table=st["table"], q_norm=st["weights"][0], k_norm=st["weights"][1], eps=EPS)
    if "pool" not in st:
        return
    tables = [_once(("tables", case["layout"], case["dim"], h if case["layout"] == "S" else 0),
                    lambda h=h: bgtq.Tables(dev, integer=_blobs(case["layout"], case["dim"], h)[0],
                                            floating=_blobs(case["layout"], case["dim"], h)[1]))
              for h in range(len(_books(case)))]
    p = st["pool"]
    st["pages"] = batched.pages(page_tokens=case["page"], tables=tables, packed=p.get("packed"), norms=p.get("norms"),
                                k_f16=p.get("k"), v=p["v"], v_scales=p.get("v_scales"))
    if kind == "append":
        return
    args = dict(pages=st["pages"], q=st["q"], out=st["out"], lengths=st["lengths"], page_table=st["table"],
                max_length=case["ctx"], window=case["window"], sinks=case["sinks"])
    if kind == "chunk":
        args["offsets"] = st["offsets"]
    make, size = ((batched.paged_decode_desc, batched.paged_decode_workspace_bytes) if kind == "decode" else
                  (batched.paged_prefill_desc, batched.paged_prefill_workspace_bytes))
    st["workspace"] = torch.zeros(size(make(**args)), dtype=torch.uint8, device="cuda")
    st["desc"] = make(workspace=st["workspace"], **args)


def run(st):
    case, kind = st["case"], st["case"]["kind"]
    if own:
        _, batched, dev = _library()
        if kind == "decode":
            batched.paged_decode(dev, st["desc"])
            return st["out"]
        if kind == "chunk":
            batched.paged_prefill(dev, st["desc"])
            return st["out"]
        if kind == "prompt":
            batched.prompt_attention(dev, st["q"], st["k"], st["v"], st["offsets"], st["out"], window=case["window"],
                                     sinks=case["sinks"])
            return st["out"]
        if kind == "rotate":
            batched.rotate(dev, st["rope"], st["positions"], st["q"], st["k"], st["q_out"], st["k_out"])
            return [st["q_out"], st["k_out"]]
        batched.paged_append(dev, st["pages"], st["slots"], st["rope"], st["positions"], st["k"], st["v"], st["q"], st["q_out"])
        batched.paged_read(dev, st["pages"], st["slots"], st["k_out"], st["v_out"])
        return [st["q_out"], st["k_out"], st["v_out"]]
    if kind == "decode":
        return _decode(st)
    if kind == "chunk":
        return _chunk(st).to(DTYPES[case["dtype"]])
    if kind == "prompt":
        return _prompt(st).to(DTYPES[case["dtype"]])
    if kind == "append":
        return _append(st)
    return [_turned(st[x], w, st["table"], st["positions"]).to(DTYPES[case["dtype"]]) for x, w in zip("qk", st["weights"])]


# ---- what a pass cannot do without

def _row_bytes(case):
    """Bytes of one token's rows in the pool, all KV heads."""
    k = sum(b.row_bytes + 2 * b.norm_stride for b in _books(case)) or case["kv_heads"] * 2 * case["dim"]
    return k + case["kv_heads"] * (case["dim"] + 2 if case["v"] == "q8" else 2 * case["dim"])


def _sees(first, last, window, sinks):
    """(query, token) pairs that positions first .. last see, and the tokens that any of them sees."""
    def upto(n):  # pairs of positions 0 .. n - 1
        if not window or n <= window:
            return n * (n + 1) // 2
        far = n - window  # positions window .. n - 1 miss 1, 2, ... tokens, but for the sinks
        kept = min(sinks, far)
        return n * (n + 1) // 2 - far * (far + 1) // 2 + kept * (kept + 1) // 2 + (far - kept) * kept
    low = max(0, first - window + 1) if window else 0
    return upto(last + 1) - upto(first), last + 1 - low + min(sinks, low)


def work(case):
    D, kind, Hq, Hkv = case["dim"], case["kind"], case["q_heads"], case["kv_heads"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case.get("dtype", "f32")]
    if kind == "prompt":
        lens = _prompt_lengths(case, 0)
        pairs = sum(_sees(0, n - 1, case["window"], case["sinks"])[0] for n in lens)
        return dict(bytes=sum(lens) * 2 * (Hq + Hkv) * D * size, flops=pairs * Hq * 4 * D)
    if kind in ("decode", "chunk"):
        chunks = _chunks(case, 0) if kind == "chunk" else [(min(n, 1), n) for n in _lengths(case, 0)]
        seen = [_sees(n - c, n - 1, case["window"], case["sinks"]) for c, n in chunks if c]
        return dict(bytes=sum(t for _, t in seen) * _row_bytes(case) + 2 * size * sum(c for c, _ in chunks) * Hq * D,
                    flops=sum(p for p, _ in seen) * Hq * 4 * D)
    n = case["rows"]
    if kind == "rotate":  # rows in and out, a table row and a position
        return dict(bytes=n * (2 * (Hq + Hkv) * D * size + 4 * D + 8), flops=n * (Hq + Hkv) * D * (8 if case["norm"] else 4))
    rotation = sum(2 * m * m for b in _books(case) for m in b.sizes)
    # in: q, k, v, a table row, a position, a slot; out: q, the pool's row, and it once more in and k and v out of the reading back
    each = (2 * Hq + 4 * Hkv) * D * size + 4 * D + 24 + 2 * _row_bytes(case)
    return dict(bytes=n * each, flops=n * (2 * rotation + (Hq + Hkv) * D * 4))


# ---- the definitions in 64 bits

def _exact_turned(st, name, weight):
    x = st[name].double()
    if weight is not None:
        x = x * weight.double() / torch.sqrt((x * x).mean(2, keepdim=True) + EPS)
    n, H, D = x.shape
    turn = torch.view_as_complex(st["table"][st["positions"]].double().view(n, 2, D // 2).transpose(1, 2).contiguous())
    z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_rows(case, st):
    """V after the write and the read; packed K has no value of its own in 64 bits: which code an entry gets is fixed by the
    codec's FP32 roundings (the format's contract is bit for bit), and an entry at a bin's border gets another one."""
    v = st["v"].half().double()
    if case["v"] == "q8":
        top = v.abs().amax(-1)
        s = (top / 127).float().half()
        s = (s.view(torch.int16) + (s.double() * 127 < top).short()).view(torch.float16).double()[..., None]
        v = (torch.where(s > 0, v / s.clamp_min(1e-30), 0.0).round() * s).float().half().double()
    k = _exact_turned(st, "k", st["weights"][1]).float().half().double() if case["layout"] == "f16" else None
    return [_exact_turned(st, "q", st["weights"][0]), k, v]


def _exact_heads(case, q, k, v, first):
    """One sequence: queries [rows, heads, dim] from position `first` on, k and v functions of a KV head."""
    G, out = case["q_heads"] // case["kv_heads"], torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for h in range(case["q_heads"]):
        if h % G == 0:
            kh, vh = k(h // G).double(), v(h // G).double()
        s = q[:, h].double() @ kh.T / math.sqrt(case["dim"])
        p = first + torch.arange(q.shape[0], device="cuda")[:, None]
        t = torch.arange(kh.shape[0], device="cuda")[None]
        hidden = t > p
        if case["window"]:
            hidden |= (p - t >= case["window"]) & (t >= case["sinks"])
        out[:, h] = torch.softmax(s.masked_fill_(hidden, -math.inf), -1) @ vh
    return out


def _exact_pages(case, st, spans):
    """Every sequence by itself over the rows that its pages hold; spans: (first row of q, rows, tokens)."""
    P, out = case["page"], torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, (at, c, n) in enumerate(spans):
        if not c:
            continue
        t = torch.arange(n, device="cuda")
        page = st["table"][b, t // P].long()
        out[at:at + c] = _exact_heads(case, st["q"][at:at + c], lambda h: _keys(case, st["pool"], h, page, t % P, torch.float64),
                                      lambda h: _values(st["pool"], h, page, t % P), n - c)
    return out


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "rotate":
        return [_exact_turned(st, x, w) for x, w in zip("qk", st["weights"])]
    if kind == "append":
        return _exact_rows(case, st)
    if kind == "prompt":
        out, at = [], 0
        for n in st["lens"]:
            rows = slice(at, at + n)
            out.append(_exact_heads(case, st["q"][rows], lambda h: st["k"][rows, h], lambda h: st["v"][rows, h], 0))
            at += n
        return torch.cat(out)
    if kind == "decode":
        return _exact_pages(case, st, [(b, min(n, 1), n) for b, n in enumerate(st["lengths"].tolist())])
    starts = np.cumsum([0] + [c for c, _ in st["chunks"]])
    return _exact_pages(case, st, [(int(at), c, n) for at, (c, n) in zip(starts, st["chunks"])])
