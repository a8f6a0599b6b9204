"""How chunk attention cuts long units into items, by the partials that a call leaves in its workspace.

The rule is chunk_wave.h's (find_item) with chunk.h's constants, read from there: should they change so that a case no longer
takes two rounds of items, its test says so. Behind the workspace's counters lie the slots of split units' items, each
`columns` x dim FP32 sums, then (maximum, sum) of each column.
"""
import math
import re
from pathlib import Path

import numpy as np
import pytest

from test_gpu_chunk import _call, _check, _written
from test_gpu_paged import _rows

pytestmark = pytest.mark.gpu

CHUNK_H = Path(__file__).resolve().parents[1] / "block-gqt-webgpu_amd" / "csrc" / "chunk.h"


def _plan(new, lengths, G, columns, aim, max_length):
    """(whether wide units take two rounds, units of each sequence, splits of each) of one KV head."""
    c = {name: int(value) for name, value in re.findall(r"\b(k\w+) = (\d+)\b", CHUNK_H.read_text())}
    keys, setup, wide, least, most = (c[k] for k in ("kChunkKeys", "kChunkSetup", "kChunkWide", "kChunkLeast", "kChunkMostSplits"))
    units = [-(-n * G // columns) if n * G > 32 else 0 for n in new]
    cost = [setup + wide * -(-n // keys) for n in lengths]
    # the host's part
    rows = sum(new) * G
    bound = rows // columns + min(len(new), rows // 33)
    two = bound * (setup + wide * -(-max_length // keys)) > c["kChunkLong"] * aim
    # the device's
    total = sum(u * x for u, x in zip(units, cost))
    splits = lambda t: [min(max(1, math.ceil(x / t - 1e-3)), most) if u else 0 for u, x in zip(units, cost)]  # noqa: E731

    def fit(t, target):
        for k in range(4):
            items = sum(s * u for s, u in zip(splits(t), units))
            if items <= max(target, sum(units)):
                return t
            if k < 3:
                t = max(t + 1, math.ceil(t * items / target))
        return -t
    one, half = abs(fit(max(least, math.ceil(total / aim)), aim)), fit(max(least, math.ceil(total / (2 * aim))), 2 * aim)
    two = two and 0 < half and 2 * half + c["kChunkRound"] < one
    return two, units, splits(half if two else one)


@pytest.mark.parametrize("dtype,new,lengths", [("float16", [1600], [10000]), ("bfloat16", [1600], [10000]),
                                               ("float16", [1300, 100, 20, 1], [9000, 3000, 60, 500])])
def test_second_round_of_items(device, oracle, dtype, new, lengths):
    """Units in more items than workgroups that the chip holds: each item leaves its partial in a slot of its own, the rest of the
    workspace as it was, and the outputs are attention's. The last case's sequences are cut into six, into two and not at all."""
    import torch
    from bgtq import batched
    print(dtype, new, lengths, flush=True)
    dim, G, rng = 128, 16, np.random.RandomState(7)
    columns, resident = (256, 1) if dtype == "float16" else (128, 2)  # chunk_wide_waves, chunk_wide_residents
    aim = resident * torch.cuda.get_device_properties(0).multi_processor_count
    pool, table = _written(device, "B", "q8", dim, 1, 64, lengths, rng, 5)
    two, units, splits = _plan(new, lengths, G, columns, aim, 64 * table.shape[1])
    slots = sum(u * s for u, s in zip(units, splits) if s > 1)
    assert two and aim < slots <= 2 * aim
    if len(new) > 1:
        assert min(s for s in splits if s) == 1 and len(set(splits)) == 4
    q = _rows(sum(new), G, dim, dtype, 2, 3).cuda()
    workspace = torch.zeros(1 << 29, dtype=torch.uint8, device="cuda")
    out = _call(pool, q, new, lengths, table, workspace=workspace)
    torch.cuda.synchronize()
    counters = batched._lib.PAGED_PREFILL_COUNTER_BYTES
    part = workspace[counters:counters + 2 * aim * columns * (dim + 2) * 4].view(torch.float32).view(2 * aim, -1)
    used = (part[:, dim * columns:] != 0).any(1).cpu()
    assert bool(used[:slots].all()) and not bool(used[slots:].any()) and not bool(workspace[:counters].any())
    _check(pool, oracle, q, out, new, lengths, table)
    assert torch.equal(out, _call(pool, q, new, lengths, table, workspace=workspace)), "two calls give the same bits"
    pool.destroy()
