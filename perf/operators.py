"""Performance cases of the paged cache and of attention over packed prompts.

Four operators that a serving loop calls per layer: rows quantised into pages as
they are written (and read back), rows read back alone, attention of one new
token per sequence over the pages, and causal attention over a batch of prompts
of different lengths. Geometries are those of the repository's own benchmark and
tests: SmolLM2-135M (9 query / 3 KV heads, d=64, its calibration tables: layout
"S"), Qwen2.5-0.5B (14 / 2 heads, d=64) and d=128 heads; layout "B" has a 4-bit
and an 8-bit group of equal size, "f16" pages hold plain FP16 K.

A page holds PAGE tokens of every KV head; a slot is page * PAGE + place. K rows
are Block-GTQ codes with an FP16 scale per group, or FP16. V rows are FP16, or
("q8") 8-bit codes c with one FP16 scale s per row, s = max|v| / 127 rounded up,
c = round(v / s), standing for the FP16 value nearest s c.
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
PAGE = 64  # tokens per page where a case names no other


def listed():
    return [
        # One token of one sequence enters the cache of a SmolLM2 layer and is read back: latency.
        dict(name="write_one_cal", kind="write", layout="S", v="q8", dim=64, kv_heads=3, rows=1, src="f32", out="f32",
             page=PAGE),
        # A batch's prompts enter the cache of a layer (Qwen geometry) and are read back for checking or reuse.
        dict(name="write_prompt", kind="write", layout="B", v="q8", dim=64, kv_heads=2, rows=16384, src="bf16", out="bf16",
             page=PAGE),
        # An odd number of prompt rows of wide heads, V kept in FP16, short pages.
        dict(name="write_d128", kind="write", layout="B", v="f16", dim=128, kv_heads=4, rows=5003, src="f16", out="f16",
             page=32),
        # One sequence's history read back on the real calibration tables (rows of 34 to 44 bytes).
        dict(name="read_cal", kind="read", layout="S", v="q8", dim=64, kv_heads=3, rows=4001, out="f16", page=PAGE),
        # Many sequences' histories leave the pool as FP32 rows.
        dict(name="read_many", kind="read", layout="B", v="q8", dim=64, kv_heads=2, rows=131072, out="f32", page=PAGE),
        # One layer of a batch-1 SmolLM2 step on its calibration tables: latency.
        dict(name="decode_one_cal", kind="decode", layout="S", v="q8", dim=64, q_heads=9, kv_heads=3, batch=1, ctx=4097,
             ragged=False, page=PAGE),
        # One layer of serving 64 sequences of 32768 tokens (Qwen geometry): the largest, memory bound.
        dict(name="decode_b64_32k", kind="decode", layout="B", v="q8", dim=64, q_heads=14, kv_heads=2, batch=64,
             ctx=32768, ragged=False, page=PAGE),
        # Continuous batching: odd lengths from none to the longest, FP16 K and V pages of wide heads.
        dict(name="decode_ragged_f16", kind="decode", layout="f16", v="f16", dim=128, q_heads=16, kv_heads=4, batch=29,
             ctx=8191, ragged=True, page=128),
        # The same on packed K and 8-bit V, fewer and longer sequences, short pages.
        dict(name="decode_ragged_d128", kind="decode", layout="B", v="q8", dim=128, q_heads=8, kv_heads=8, batch=7,
             ctx=16001, ragged=True, page=32),
        # A few short prompts of one step (SmolLM2 geometry): latency.
        dict(name="prompt_short", kind="prompt", dtype="f16", dim=64, q_heads=9, kv_heads=3, sequences=3, longest=45),
        # A batch of prompts of mixed odd lengths (Qwen geometry).
        dict(name="prompt_packed", kind="prompt", dtype="bf16", dim=64, q_heads=14, kv_heads=2, sequences=11,
             longest=2777),
        # One long prompt of wide heads: matrix-core work.
        dict(name="prompt_long", kind="prompt", dtype="bf16", dim=128, q_heads=16, kv_heads=4, sequences=1, longest=8192),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of lo..hi, both ends included."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "write", "read", "decode", "decode", "prompt", "prompt"])
    if kind == "prompt":
        dim = rng.choice([64, 128])
        q, kv = rng.choice([(9, 3), (14, 2), (16, 4), (8, 8), (4, 1)])
        longest = _log(rng, 1, 6000)
        return dict(kind=kind, dtype=rng.choice(["f16", "bf16"]), dim=dim, q_heads=q, kv_heads=kv,
                    sequences=_log(rng, 1, max(1, min(200, (1 << 27) // (longest * longest)))), longest=longest)
    dim = rng.choice([64, 64, 128])
    layout = rng.choice(["S", "S", "B", "B", "f16"]) if dim == 64 else rng.choice(["B", "f16"])
    kv, g = (3, 3) if layout == "S" else rng.choice([(1, 1), (1, 3), (2, 7), (4, 4), (8, 1)])
    v, page = rng.choice(["q8", "q8", "f16"]), rng.choice([32, 64, 64, 256])
    if kind == "decode":
        ctx = min(_log(rng, 1, 32768), (1 << 22) // kv)
        return dict(kind=kind, layout=layout, v=v, dim=dim, q_heads=kv * g, kv_heads=kv,
                    batch=_log(rng, 1, max(1, min(200, (1 << 21) // (kv * ctx)))), ctx=ctx, ragged=rng.random() < 0.7,
                    page=page)
    if kind == "read":
        return dict(kind=kind, layout=layout, v=v, dim=dim, kv_heads=kv, rows=_log(rng, 1, 65536),
                    out=rng.choice(["f32", "f16", "bf16"]), page=page)
    return dict(kind=kind, layout=layout, v=v, dim=dim, kv_heads=kv, rows=_log(rng, 1, 16384),
                src=rng.choice(["f32", "f16", "bf16"]), out=rng.choice(["f32", "f16", "bf16"]), page=page)


DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- calibration tables: what a program loads once

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
    if case["layout"] == "f16":
        return []
    key = lambda h: (case["layout"], case["dim"], h if case["layout"] == "S" else 0)  # noqa: E731
    return [_once(("book", key(h)), lambda h=h: _Book(*_blobs(case["layout"], case["dim"], h))) for h in range(case["kv_heads"])]


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


def _shuffled(n, seed):
    return torch.from_numpy(np.random.RandomState(int(seed) % (1 << 31)).permutation(n)).cuda()


def _lengths(case, seed):
    """Sequence lengths: all ctx, or spread evenly from an empty one to ctx, in an order of the seed's."""
    B, ctx = case["batch"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * B
    return [int(x) for x in np.random.RandomState(int(seed) % (1 << 31)).permutation([ctx * (i + 1) // B if i else 0 for i in range(B)])]


def _prompt_lengths(case, seed):
    """Prompt lengths: the longest, the others spread over its eighth and up, odd ones among them."""
    n, longest = case["sequences"], case["longest"]
    low = (longest + 7) // 8
    return [int(x) for x in np.random.RandomState(int(seed) % (1 << 31)).permutation([low + (longest - low) * (i + 1) // n for i in range(n)])]


def prepare(case, seed):
    D, seed = case["dim"], int(seed)
    st = dict(case=case)
    if case["kind"] == "prompt":
        lens = _prompt_lengths(case, seed)
        Hq, Hkv, total = case["q_heads"], case["kv_heads"], sum(lens)
        # the rows of a fused projection: queries, keys and values side by side
        x = _randn(seed, 1, total, Hq + 2 * Hkv, D).to(DTYPES[case["dtype"]])
        st.update(q=x[:, :Hq], k=x[:, Hq:Hq + Hkv], v=x[:, Hq + Hkv:], lens=lens,
                  offsets=torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda"))
        st["out"] = torch.empty((total, Hq, D), dtype=x.dtype, device="cuda")
        st["index"] = torch.stack([torch.arange(max(lens)).clamp(max=n - 1) + o for n, o in zip(lens, np.cumsum([0] + lens))]).cuda()
        st["lengths"] = torch.tensor(lens, device="cuda")
    elif case["kind"] == "decode":
        lens, P = _lengths(case, seed), case["page"]
        need = [-(-n // P) for n in lens]
        pages = sum(need) + 3
        st["pool"] = _filled(case, pages, seed)
        order, width = _shuffled(pages, seed), -(-case["ctx"] // P)
        table = torch.full((case["batch"], width), -1, dtype=torch.int32)
        for b, (at, n) in enumerate(zip(np.cumsum([0] + need), need)):
            table[b, :n] = order[at:at + n]
        st.update(table=table.cuda(), lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                  q=_randn(seed, 1, case["batch"], case["q_heads"], D))
        st["out"] = torch.empty_like(st["q"])
    else:
        n, P, H = case["rows"], case["page"], case["kv_heads"]
        pages = -(-n // P) + 3
        order = _shuffled(pages, seed)  # consecutive tokens fill pages that lie anywhere
        t = torch.arange(n, device="cuda")
        st["slots"] = order[t // P] * P + t % P
        for name in ("k", "v"):
            st[name + "_out"] = torch.empty((n, H, D), dtype=DTYPES[case["out"]], device="cuda")
        if case["kind"] == "read":
            st["pool"] = _filled(case, pages, seed)
        else:
            st["pool"] = _pool(case, pages)
            x = _randn(seed, 2, n, 2 * H, D)
            x[:, :H] *= 3 * _energies(D)
            x = x.to(DTYPES[case["src"]])
            st.update(k=x[:, :H], v=x[:, H:])
    if own:  # the library's handles: tables on the device, the pool's description, a workspace
        _bind(st)
    return st


# ---- the plain forms

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


def _coded(case, pool, h, page, place, dtype=torch.float32):
    """The code-domain K rows c s [n, dim] of head h at (page, place)."""
    b, P = _books(case)[h], case["page"]
    rows = pool["packed"][:, h, :P * b.row_bytes].unflatten(1, (P, b.row_bytes))[page, place].long()
    norms = pool["norms"][:, h, :P * b.norm_stride].unflatten(1, (P, b.norm_stride))[page, place]
    n, half = rows.shape[:-1], b.nib // 2
    codes = torch.cat([torch.stack([rows[..., :half] & 15, rows[..., :half] >> 4], -1).reshape(*n, b.nib),
                       rows[..., half:half + b.dim - b.nib]], -1)
    return b.cent.to(dtype)[b.pos, codes] * norms.to(dtype)[..., b.group_of]


def _keys(case, pool, h, page, place, dtype=torch.float32):
    """Head h's K rows at (page, place), in the model's order of dimensions."""
    if "k" in pool:
        return pool["k"][page, h, place].to(dtype)
    b, cs = _books(case)[h], _coded(case, pool, h, page, place, dtype)
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


def _write(st):
    case, pool, P = st["case"], st["pool"], st["case"]["page"]
    page, place = st["slots"] // P, st["slots"] % P
    k, v = st["k"].half(), st["v"].half()
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


def _read(st):
    case, P = st["case"], st["case"]["page"]
    page, place = st["slots"] // P, st["slots"] % P
    heads = range(case["kv_heads"])
    return [torch.stack([fn(h) for h in heads], 1).to(DTYPES[case["out"]])
            for fn in (lambda h: _keys(case, st["pool"], h, page, place), lambda h: _values(st["pool"], h, page, place))]


def _attend(logits, seen, v):
    """softmax over the seen entries of the last axis, times v; rows that see nothing are zero."""
    logits = torch.where(seen, logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def _decode(st):
    case, pool, P = st["case"], st["pool"], st["case"]["page"]
    B, D, G = case["batch"], case["dim"], case["q_heads"] // case["kv_heads"]
    t = torch.arange(case["ctx"], device="cuda")
    page, place = st["table"].long()[:, t // P].clamp_min(0), (t % P).expand(B, -1)
    seen = (t < st["lengths"][:, None])[:, None]
    outs = []
    for h in range(case["kv_heads"]):
        q = st["q"][:, h * G:(h + 1) * G] / math.sqrt(D)
        if "k" in pool:
            k = _keys(case, pool, h, page, place)
        else:  # the query rotated once instead of every key
            b = _books(case)[h]
            q, k = torch.matmul(q[..., b.perm], b.rot.T.contiguous()), _coded(case, pool, h, page, place)
        logits = torch.matmul(q, k.transpose(1, 2).contiguous())
        outs.append(_attend(logits, seen, _values(pool, h, page, place).float()))
    return torch.cat(outs, 1)


def _prompt(st, dtype=torch.float32):
    G, D = st["case"]["q_heads"] // st["case"]["kv_heads"], st["case"]["dim"]
    q, k, v = (st[x][st["index"]].to(dtype).transpose(1, 2) for x in ("q", "k", "v"))  # [sequence, head, place, dim]
    k, v = (x.repeat_interleave(G, 1) for x in (k, v))
    t = torch.arange(q.shape[2], device="cuda")
    out = _attend(torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(D), t[None] <= t[:, None], v)
    return out.transpose(1, 2)[t < st["lengths"][:, None]]


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
    case = st["case"]
    bgtq, batched, dev = _library()
    if case["kind"] == "prompt":
        return
    tables = [_once(("tables", case["layout"], case["dim"], h if case["layout"] == "S" else 0),
                    lambda h=h: bgtq.Tables(dev, integer=_blobs(case["layout"], case["dim"], h)[0],
                                            floating=_blobs(case["layout"], case["dim"], h)[1]))
              for h in range(len(_books(case)))]
    p = st["pool"]
    st["pages"] = batched.pages(page_tokens=case["page"], tables=tables, packed=p.get("packed"), norms=p.get("norms"),
                                k_f16=p.get("k"), v=p["v"], v_scales=p.get("v_scales"))
    if case["kind"] == "decode":
        args = dict(pages=st["pages"], q=st["q"], out=st["out"], lengths=st["lengths"], page_table=st["table"],
                    max_length=case["ctx"])
        size = batched.paged_decode_workspace_bytes(batched.paged_decode_desc(**args))
        st["workspace"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
        st["desc"] = batched.paged_decode_desc(workspace=st["workspace"], **args)


def run(st):
    kind = st["case"]["kind"]
    if own:
        _, batched, dev = _library()
        if kind == "decode":
            batched.paged_decode(dev, st["desc"])
            return st["out"]
        if kind == "prompt":
            batched.prompt_attention(dev, st["q"], st["k"], st["v"], st["offsets"], st["out"])
            return st["out"]
        if kind == "write":
            batched.paged_write(dev, st["pages"], st["slots"], st["k"], st["v"])
        batched.paged_read(dev, st["pages"], st["slots"], st["k_out"], st["v_out"])
        return [st["k_out"], st["v_out"]]
    if kind == "decode":
        return _decode(st)
    if kind == "prompt":
        return _prompt(st).to(DTYPES[st["case"]["dtype"]])
    if kind == "write":
        _write(st)
    return _read(st)


# ---- what a pass cannot do without

def _row_bytes(case):
    """Bytes of one token's rows in the pool, all KV heads."""
    k = sum(b.row_bytes + 2 * b.norm_stride for b in _books(case)) or case["kv_heads"] * 2 * case["dim"]
    return k + case["kv_heads"] * (case["dim"] + 2 if case["v"] == "q8" else 2 * case["dim"])


def work(case):
    D, kind = case["dim"], case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if kind == "prompt":
        lens = _prompt_lengths(case, 0)
        rows = 2 * case["q_heads"] + 2 * case["kv_heads"]
        return dict(bytes=sum(lens) * rows * D * 2, flops=sum(n * (n + 1) // 2 for n in lens) * case["q_heads"] * 4 * D)
    if kind == "decode":
        n = sum(_lengths(case, 0))
        return dict(bytes=n * _row_bytes(case) + 8 * case["batch"] * case["q_heads"] * D,
                    flops=n * case["q_heads"] * 4 * D)
    n, H = case["rows"], case["kv_heads"]
    rotation = sum(2 * m * m for b in _books(case) for m in b.sizes)
    each = _row_bytes(case) + 8 + 2 * H * D * size[case["out"]]
    if kind == "write":  # in, written, read back, out
        each += _row_bytes(case) + 2 * H * D * size[case["src"]]
    return dict(bytes=n * each, flops=n * rotation * (2 if kind == "write" else 1))


# ---- the definitions in 64 bits

def _exact_rows(case, st):
    """K and V after a write and a read. Packed K has no value of its own in 64 bits: which code an entry gets is fixed by
    the codec's FP32 roundings (the format's contract is bit for bit), and an entry at a bin's border gets another one."""
    v = st["v"].half().double()
    if case["v"] == "q8":
        top = v.abs().amax(-1)
        s = (top / 127).float().half()
        s = (s.view(torch.int16) + (s.double() * 127 < top).short()).view(torch.float16).double()[..., None]
        v = (torch.where(s > 0, v / s.clamp_min(1e-30), 0.0).round() * s).float().half().double()
    return [st["k"].half().double() if case["layout"] == "f16" else None, v]


def _exact_decode(case, st):
    """Every sequence by itself over the rows that its pages hold, K rebuilt in the model's order."""
    P, G, out = case["page"], case["q_heads"] // case["kv_heads"], torch.zeros_like(st["q"], dtype=torch.float64)
    for b, n in enumerate(st["lengths"].tolist()):
        t = torch.arange(n, device="cuda")
        page = st["table"][b, t // P].long()
        for h in range(case["kv_heads"] if n else 0):
            q = st["q"][b, h * G:(h + 1) * G].double()
            s = q @ _keys(case, st["pool"], h, page, t % P, torch.float64).T / math.sqrt(case["dim"])
            out[b, h * G:(h + 1) * G] = torch.softmax(s, -1) @ _values(st["pool"], h, page, t % P).double()
    return out


def _exact_prompt(case, st):
    """Every sequence and head by itself."""
    G, out = case["q_heads"] // case["kv_heads"], torch.empty(st["out"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for n in st["lens"]:
        past = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
        for h in range(case["q_heads"]):
            q, k, v = (x[at:at + n].double() for x in (st["q"][:, h], st["k"][:, h // G], st["v"][:, h // G]))
            s = (q @ k.T / math.sqrt(case["dim"])).masked_fill(~past, -math.inf)
            out[at:at + n, h] = torch.softmax(s, -1) @ v
        at += n
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "prompt":
        return _exact_prompt(case, st)
    if case["kind"] == "decode":
        return _exact_decode(case, st)
    if case["kind"] == "write":
        return _exact_rows(case, st)
    P = case["page"]
    page, place = st["slots"] // P, st["slots"] % P
    heads = range(case["kv_heads"])
    return [torch.stack([_keys(case, st["pool"], h, page, place, torch.float64) for h in heads], 1),
            torch.stack([_values(st["pool"], h, page, place) for h in heads], 1).double()]
