"""Block tables and slot maps on the GPU (ops.cache_slots) against the plain form request by
request (oracle/paged.py): whole numbers, so every output has to be equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
BOUNDS = 9  # KTA_ERR_DEVICE_BOUNDS


def _case(ctx, new, block, spare=3, wide=2, seed=0, pool=None):
    """Tables with the held blocks entered and the free list behind them, in a random order."""
    g = np.random.default_rng(seed)
    held = [-(-max(c, 0) // block) for c in ctx]
    need = [max(-(-max(c + n, 0) // block), h) for c, n, h in zip(ctx, new, held)]
    ids = g.permutation(sum(need) + spare).tolist()
    tables = np.full((len(ctx), max(need) + wide), -7, dtype=np.int32)
    for b, h in enumerate(held):
        tables[b, :h] = ids[:h]
        del ids[:h]
    free = np.array(ids if pool is None else ids[:pool], dtype=np.int32)
    return tables, free


def _run(dev, ctx, new, tables, free, block, rows, **out):
    from kta_b200 import ops

    t = torch.from_numpy(tables).to(dev)
    got = ops.cache_slots(torch.tensor(ctx, dtype=torch.int32, device=dev),
                          torch.tensor(new, dtype=torch.int32, device=dev), t,
                          torch.from_numpy(free).to(dev), block, rows, **out)
    torch.cuda.synchronize()
    return (t, *got)


def _check(dev, ctx, new, tables, free, block, rows):
    want = paged.cache_slots(ctx, new, tables, free, block, rows)
    got = _run(dev, ctx, new, tables, free, block, rows)
    for w, g, name in zip(want, got, ("tables", "slots", "positions", "offsets", "used")):
        assert np.array_equal(np.asarray(w).reshape(-1), g.cpu().numpy().reshape(-1)), name


def _status():
    from kta_b200 import lib

    return lib.device_status(clear=True)


@pytest.mark.parametrize("ctx,new,block,pad", [
    ([0], [1], 16, 0),                                   # the first token of the only request
    ([15], [1], 16, 3), ([16], [1], 16, 0), ([17], [1], 16, 1),
    ([0, 0, 0], [0, 5, 0], 4, 2),                        # requests without new tokens around one
    ([7, 0, 33], [0, 0, 0], 8, 5),                       # no new token at all
    ([3, 31, 0, 64, 1], [30, 1, 65, 64, 0], 32, 10),     # blocks begun, full, and several at once
    ([5, 9], [20, 11], 1, 0), ([5, 9], [20, 11], 7, 0),  # blocks of one, and of no power of two
])
def test_small(cuda_device, ctx, new, block, pad):
    tables, free = _case(ctx, new, block)
    _check(cuda_device, ctx, new, tables, free, block, max(1, sum(new) + pad))
    assert _status()[0] == 0


@pytest.mark.parametrize("bsz,hi,new_hi,block", [(33, 100, 9, 16), (257, 5000, 16, 64),
                                                 (2048, 300, 3, 16), (64, 0, 4095, 16),
                                                 (1, 70000, 60000, 128)])
def test_ragged(cuda_device, bsz, hi, new_hi, block):
    g = np.random.default_rng(bsz)
    ctx = g.integers(0, hi + 1, bsz).tolist()
    new = g.integers(0, new_hi + 1, bsz).tolist()
    tables, free = _case(ctx, new, block)
    _check(cuda_device, ctx, new, tables, free, block, sum(new) + 77)
    assert _status()[0] == 0


def test_what_does_not_fit_is_cut_off_and_recorded(cuda_device):
    # the free list ends: later blocks are -1 and their tokens have no slot
    ctx, new = [10, 0, 30], [20, 40, 7]
    tables, free = _case(ctx, new, 8, pool=4)
    _check(cuda_device, ctx, new, tables, free, 8, 70)
    assert _status()[0] == BOUNDS
    # an empty free list, and none needed
    tables, free = _case([3, 4], [2, 1], 8, pool=0)
    _check(cuda_device, [3, 4], [2, 1], tables, free, 8, 3)
    assert _status()[0] == 0
    # more tokens than rows: offsets end at the last row
    tables, free = _case(ctx, new, 8)
    _check(cuda_device, ctx, new, tables, free, 8, 33)
    assert _status()[0] == BOUNDS
    # negative lengths and one past the table's row count as no new tokens
    for ctx, new in (([5, -1, 9], [1, 2, 3]), ([5, 4, 9], [1, -2, 3]), ([5, 4, 9], [1, 1000, 3]),
                     ([5, 2**31 - 1, 9], [1, 2**31 - 1, 3])):
        tables = np.full((3, 4), -7, dtype=np.int32)
        tables[0, 0], tables[2, :2] = 11, (12, 13)
        _check(cuda_device, ctx, new, tables, np.arange(20, 40, dtype=np.int32), 8, 8)
        assert _status()[0] == BOUNDS
    assert _status()[0] == 0


def test_strided_tables_given_outputs_and_replay(cuda_device):
    from kta_b200 import ops

    dev = cuda_device
    ctx, new, block, rows = [9, 0, 40, 16], [3, 17, 1, 16], 8, 48
    tables, free = _case(ctx, new, block)
    want = paged.cache_slots(ctx, new, tables, free, block, rows)
    wide = torch.full((4, tables.shape[1] + 5), 99, dtype=torch.int32, device=dev)
    view = wide[:, :tables.shape[1]]
    view.copy_(torch.from_numpy(tables))
    c, n = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (ctx, new))
    f = torch.from_numpy(free).to(dev)
    out = dict(slots=torch.empty(rows, dtype=torch.int64, device=dev),
               positions=torch.empty(rows, dtype=torch.int32, device=dev),
               offsets=torch.empty(5, dtype=torch.int32, device=dev),
               used=torch.empty(1, dtype=torch.int32, device=dev))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.cache_slots(c, n, view, f, block, rows, **out)  # another stream than the tensors' own
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_slots(c, n, view, f, block, rows, **out)
    for _ in range(2):  # new lengths in the same memory, then the first ones again
        c.zero_()
        graph.replay()
        c.copy_(torch.tensor(ctx, dtype=torch.int32))
        view.copy_(torch.from_numpy(tables))
        graph.replay()
    torch.cuda.synchronize()
    got = (view, out["slots"], out["positions"], out["offsets"], out["used"])
    for w, g in zip(want, got):
        assert np.array_equal(np.asarray(w).reshape(-1), g.cpu().numpy().reshape(-1))
    assert (wide[:, tables.shape[1]:] == 99).all()
