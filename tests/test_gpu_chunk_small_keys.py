"""Chunk attention over packed K rows that are small numbers: FP16 queries take 22 bits of a row whatever its scale is.

The limits are test_gpu_chunk.py's. Of the packed K, an FP16 row's pair of FP16 values leaves 2^-23 of a value (the high one
rounded to nearest, the low one held times 2^11), or 2^-36 where that is more: below 2^-20 of a row's largest for rows down to scales of
2^-16. Queries are cut to 2^-21, and of the products only low times low is missing, 2^-21. Logits stay below 60.
"""
import numpy as np
import pytest

from test_gpu_chunk import _call, _check
from test_gpu_paged import Pool, _rows, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exp", [0, -8, -12, -16])
@pytest.mark.parametrize("layout,v,dim,heads", [("S", "q8", 64, 3), ("B", "f16", 64, 2), ("B", "q8", 128, 1)])
def test_small_keys_keep_their_bits(device, oracle, layout, v, dim, heads, exp):
    """Few and many new rows (straight from the pages, and rebuilt), long and short histories."""
    import torch
    from bgtq import batched
    print(layout, v, dim, exp, flush=True)
    rng = np.random.RandomState(1)
    lengths = [700, 90, 33]
    pool = Pool(device, layout, v, dim, heads, 20, 64, gap=32)
    table = _table(pool, lengths, rng)
    tab = table.cpu().numpy().astype(np.int64)
    slots = np.concatenate([tab[b, np.arange(n) // 64] * 64 + np.arange(n) % 64 for b, n in enumerate(lengths)]).astype(np.int64)
    k, val = _rows(len(slots), heads, dim, "float16", 1, 1, scale=2.0 ** exp), _rows(len(slots), heads, dim, "float16", 1, 2)
    batched.paged_write(device, pool.handle, torch.from_numpy(slots).cuda(), k.cuda(), val.cuda())
    for new in ([5, 1, 7], [300, 60, 33]):
        q = _rows(sum(new), 3 * heads, dim, "float16", sum(new), 3).cuda()
        scale = 8 * 2.0 ** -exp / np.sqrt(dim)  # (logits with a standard deviation of 8)
        out = _call(pool, q, new, lengths, table, scale=scale)
        torch.cuda.synchronize()
        _check(pool, oracle, q, out, new, lengths, table, scale=scale, what=f"{new}")
    pool.destroy()
