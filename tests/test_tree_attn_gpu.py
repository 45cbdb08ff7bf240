"""Attention of drafted tokens over a paged cache on the GPU (ops.tree_attn) against the float64
form row by row (oracle/paged.py).

Tolerance of O, from the arithmetic. With s the scaled score of a key, its fp32 value is off by
D 2^-24 (sum |q||k|) scale from the products' sum, and the exponent s log2 e - m by a rounding of
2 |s| 2^-24 and of the scale's product; 2^x has 2 ulp: d32 = D 2^-24 dot + 6 |s| 2^-24 + 2^-22
relative, on a weight and again on the sum. Each weight is rounded to the storage type (half a
step, and for f16 half a subnormal step 2^-25 where weights are relative to a maximum no larger
than the true one), the products are summed in fp32 over n keys (n 2^-24), and O is rounded once:
  |O - want| <= (eps/2 + 2 d32 + n 2^-24) sum p|v| + 2^-25 sum |v| / l + eps/2 (|O| + the same).
LSE: d32 (times log's slope 1) + n 2^-24, fp32 rounding of the result."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


class Case:
    """A paged cache whose unwritten places hold NaN, with blocks in a random order."""

    def __init__(self, ctx, new, hq, hkv, d, block, dtype, parents="random", seed=0, spare=2, wide=0,
                 gap=0):
        g = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.ctx, self.new, self.hq, self.hkv, self.d = ctx, new, hq, hkv, d
        self.block, self.dtype = block, dtype
        need = [-(-(c + n) // block) for c, n in zip(ctx, new)]
        self.blocks = sum(need) + spare
        ids = g.permutation(self.blocks).tolist()
        self.tables = np.full((len(ctx), max(max(need), 1) + wide), -1, dtype=np.int32)
        self.kc = torch.full((self.blocks, block, hkv, d), float("nan")).to(dtype)
        self.vc = torch.full_like(self.kc, float("nan"))
        self.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.offsets[-1]) + gap
        self.q = torch.randn((max(self.rows, 1), hq, d), generator=gen).to(dtype)
        bits = []
        for b, (c, n, m) in enumerate(zip(ctx, new, need)):
            self.tables[b, :m] = ids[:m]
            del ids[:m]
            for cache in (self.kc, self.vc):
                flat = torch.randn((c + n, hkv, d), generator=gen).to(dtype)
                for j in range(m):
                    part = flat[j * block:(j + 1) * block]
                    cache[self.tables[b, j], :part.shape[0]] = part
            if parents == "random":
                bits += paged.tree_bits([int(g.integers(-1, i)) if i else -1 for i in range(n)])
        self.bits = np.array(bits + [0] * gap, dtype=np.int64) if parents == "random" else None

    def run(self, dev, max_new=None, **kw):
        from kta_b200 import ops

        self.dev = [t.to(dev) for t in (self.q, self.kc, self.vc, torch.from_numpy(self.tables),
                                        torch.tensor(self.ctx, dtype=torch.int32),
                                        torch.from_numpy(self.offsets))]
        tree = None if self.bits is None else torch.from_numpy(self.bits).to(dev)
        got = ops.tree_attn(*self.dev, max_new or max(max(self.new), 1), tree, **kw)
        torch.cuda.synchronize()
        return got

    def check(self, out, lse, scale=None, skip=()):
        scale = self.d ** -0.5 if scale is None else scale
        eps = torch.finfo(self.dtype).eps / 2
        group = self.hq // self.hkv
        out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        q, kc, vc = (t.double().numpy() for t in (self.q, self.kc, self.vc))
        for b, (c, n) in enumerate(zip(self.ctx, self.new)):
            a = self.offsets[b]
            if b in skip or n == 0:
                continue
            bits = None if self.bits is None else self.bits[a:a + n]
            sight = paged.seen(c, n, bits)
            ids = self.tables[b, :-(-(c + n) // self.block)]
            k = kc[ids].reshape(-1, self.hkv, self.d)[:c + n]
            v = vc[ids].reshape(-1, self.hkv, self.d)[:c + n]
            for h in range(self.hq):
                o, z, pv, tiny, smax, dot = paged.attention(q[a:a + n, h], k[:, h // group],
                                                            v[:, h // group], sight, scale)
                far, far_lse = paged.attention_bounds(sight, eps, 2.0 ** -25 if self.dtype == F16 else 0.0,
                                                      o, z, pv, tiny, smax, dot)
                err = np.abs(out[a:a + n, h] - o)
                assert (err <= far).all(), (b, h, float((err / far).max()), float(err.max()))
                none = ~sight.any(1)
                assert np.array_equal(lse[a:a + n, h][none], z[none])
                off = np.abs(lse[a:a + n, h][~none] - z[~none])
                assert (off <= far_lse[~none]).all(), (b, h, float(off.max()))


def _status():
    from kta_b200 import lib

    return lib.device_status(clear=True)[0]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("ctx,new,hq,hkv,d,block", [
    ([0], [1], 1, 1, 128, 16),                                  # one key, one row
    ([5], [3], 4, 2, 128, 16),
    ([126, 127, 128, 129, 0], [1, 1, 1, 1, 1], 8, 2, 128, 16),  # single tokens at a tile's edge
    ([120, 100, 250], [8, 30, 7], 8, 2, 64, 32),                # drafts across two tiles
    ([33, 0, 400], [64, 64, 5], 4, 4, 128, 64),                 # 64 drafts, one head to a group
    ([300, 17, 90], [9, 2, 13], 35, 5, 128, 8),                 # groups of seven, blocks of eight
    ([511, 1000], [33, 40], 16, 1, 128, 128),                   # groups of 16: several row tiles
    ([700, 129], [26, 64], 10, 2, 64, 256),                     # groups of five, blocks of 256
    ([0, 3000, 0], [0, 6, 0], 4, 1, 128, 16),                   # requests without rows around one
    ([300, 17, 90], [2, 1, 2], 35, 5, 128, 8),                  # few rows: blocks of 8, 128 and 256
    ([511, 1000, 40], [4, 3, 5], 16, 4, 128, 128),
    ([700, 129, 255], [8, 4, 12], 10, 2, 64, 256),
    ([200, 77], [8, 7], 16, 2, 128, 8),
])
def test_against_the_formula(cuda_device, ctx, new, hq, hkv, d, block, dtype):
    c = Case(ctx, new, hq, hkv, d, block, dtype)
    c.check(*c.run(cuda_device))
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_chain_without_a_tree_and_other_scale(cuda_device, dtype):
    c = Case([70, 200, 0], [64, 5, 9], 8, 4, 128, 16, dtype, parents=None)
    c.check(*c.run(cuda_device, scale=0.3), scale=0.3)
    # a wider max_new than any request has
    c.check(*c.run(cuda_device, max_new=64))
    assert _status() == 0


@pytest.mark.parametrize("ctx,new,hq,hkv", [
    ([9000], [4], 8, 1),                       # one KV head over every SM: many parts
    ([20000, 3], [8, 8], 8, 2),
    (list(range(0, 2000, 31)), [3] * 65, 4, 2),  # more units than ranges, cut anywhere
    ([1500] * 3, [64] * 3, 64, 4),             # groups of 16: eight row tiles share each range
])
def test_split_ranges(cuda_device, ctx, new, hq, hkv):
    c = Case(ctx, new, hq, hkv, 128, 16, BF16, seed=1)
    out, lse = c.run(cuda_device)
    c.check(out, lse)
    again = c.run(cuda_device)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])  # no order of arrival in it
    assert _status() == 0


@pytest.mark.parametrize("hq,most,max_new", [(16, 3, 3), (64, 16, 16), (128, 16, 16)])
def test_long_lists_weigh_their_requests(cuda_device, hq, most, max_new):
    """Sixteen tiles and more to a CTA: units count more than their tiles. One row tile the one way
    round and the other, and two row tiles of which most requests have one."""
    g = np.random.default_rng(hq)
    # ragged, with some of the shortest between them
    ctx = (g.integers(2200, 2900, 20) * (np.arange(20) % 7 != 3)).tolist()
    new = g.integers(1, 4, 20).tolist()
    new[5], new[12] = most, 0
    c = Case(ctx, new, hq, 8, 64, 64, BF16, seed=2)
    out, lse = c.run(cuda_device, max_new=max_new)
    c.check(out, lse)
    again = c.run(cuda_device, max_new=max_new)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    assert _status() == 0


def test_rows_that_see_nothing_and_rows_of_no_request(cuda_device):
    c = Case([0, 40], [5, 5], 8, 2, 128, 16, BF16, gap=4)
    c.bits[1] = 0          # nothing at all
    c.bits[3] = ~31        # bits past the request's own tokens do not count
    c.bits[7] = 0          # the context alone
    out = torch.full((14, 8, 128), 9.0, dtype=BF16, device=cuda_device)
    lse = torch.full((14, 8), 9.0, device=cuda_device)
    c.run(cuda_device, out=out, lse=lse)
    c.check(out, lse)
    assert (out[[1, 3]] == 0).all() and (lse[[1, 3]] == -float("inf")).all()
    assert (out[10:] == 9).all() and (lse[10:] == 9).all()
    assert _status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("ctx", [0, 100, 127])
@pytest.mark.parametrize("max_new", [7, 64])  # one kernel and the other
def test_values_that_a_row_does_not_see_do_not_reach_it(cuda_device, max_new, ctx, dtype):
    """Infinities and NaN in drafted K and V: rows that do not see the token stay exact, rows that
    do have what the formula gives."""
    c = Case([ctx, 30], [7, 3], 4, 2, 128, 16, dtype, seed=3)
    c.bits[:7] = paged.tree_bits([-1, 0, 0, 1, 2, -1, 5])

    def slot(b, p):
        return int(c.tables[b, p // 16]), p % 16

    for cache, tok, value in ((c.kc, 1, float("nan")), (c.vc, 2, float("nan")),
                              (c.vc, 5, float("inf"))):
        block, place = slot(0, ctx + tok)
        cache[block, place, 0, 3:9] = value
    out, lse = c.run(cuda_device, max_new=max_new)
    # KV head 0: token 1 (and 3 through it) has a NaN key, 2 (and 4) a NaN value, 5 (and 6) an
    # infinite one in dimensions 3..8
    o = out[:7, :2].double().cpu()
    assert torch.isnan(o[[1, 3]]).all()
    assert torch.isnan(o[[2, 4], :, 3:9]).all() and torch.isinf(o[[5, 6], :, 3:9]).all()
    c.kc[torch.isnan(c.kc)] = 0
    c.vc[~torch.isfinite(c.vc)] = 0
    clean_out, clean_lse = c.run(cuda_device, max_new=max_new)
    c.check(clean_out, clean_lse)
    for row, ok in ((0, slice(None)), (2, [0, 1, 2, 9, 127]), (4, [0, 2, 10]), (5, [1, 9]), (6, [0])):
        assert torch.equal(out[row, :2][:, ok], clean_out[row, :2][:, ok])
    assert torch.equal(out[:, 2:], clean_out[:, 2:]) and torch.equal(out[7:], clean_out[7:])
    assert _status() == 0


@pytest.mark.parametrize("max_new", [5, 64])
def test_queries_that_are_not_finite_stay_in_their_rows(cuda_device, max_new):
    c = Case([500, 90], [5, 3], 4, 2, 128, 16, BF16, seed=8)
    want, want_lse = c.run(cuda_device, max_new=max_new)
    c.check(want, want_lse)
    keep = c.q.clone()
    c.q[1, 2] = float("nan")
    c.q[3, 0, 5] = float("inf")
    c.q[6] = -float("inf")
    out, lse = c.run(cuda_device, max_new=max_new)
    same = torch.ones(8, 4, dtype=torch.bool)
    same[1, 2] = same[3, 0] = same[6] = False
    c.q = keep
    assert torch.equal(out.cpu()[same], want.cpu()[same])
    assert torch.equal(lse.cpu()[same], want_lse.cpu()[same])
    assert torch.isnan(out.cpu()[1, 2]).all() and torch.isnan(out.cpu()[3, 0]).all()
    assert _status() == 0


def test_most_requests(cuda_device):
    g = np.random.default_rng(9)
    c = Case(g.integers(0, 40, 2048).tolist(), g.integers(0, 3, 2048).tolist(), 2, 1, 64, 8, F16, seed=9)
    out, lse = c.run(cuda_device)
    c.check(out, lse)
    assert _status() == 0


@pytest.mark.parametrize("max_new", [6, 32])
def test_large_scores(cuda_device, max_new):
    """Scores up to some hundreds: the running maximum has to move, and O with it."""
    for dtype in (F16, BF16):
        c = Case([900, 600], [6, 6], 8, 2, 128, 16, dtype, seed=4)
        c.q *= 8
        grow = torch.linspace(0.1, 3.0, c.blocks)[torch.randperm(c.blocks)].to(dtype)
        c.kc *= grow[:, None, None, None]
        c.check(*c.run(cuda_device, max_new=max_new))


@pytest.mark.parametrize("hq", [8, 32])
def test_out_of_range_requests_and_blocks(cuda_device, hq):
    dev = cuda_device
    good = Case([40, 300, 7], [4, 4, 4], hq, 2, 128, 16, BF16, wide=1)
    good.run(dev)
    assert _status() == 0
    q, kc, vc, tables, ctx, offsets = good.dev
    from kta_b200 import ops

    tree = torch.from_numpy(good.bits).to(dev)

    def run(ctx=ctx, offsets=offsets, tables=tables, max_new=4):
        got = ops.tree_attn(q, kc, vc, tables, ctx, offsets, max_new, tree)
        torch.cuda.synchronize()
        return got

    room = tables.shape[1] * 16
    for bad in (-1, room - 3, 2**31 - 1):
        moved = ctx.clone()
        moved[1] = bad
        out, lse = run(ctx=moved)
        good.check(out, lse, skip=(1,))
        assert (out[4:8] == 0).all() and (lse[4:8] == -float("inf")).all()
        assert _status() == 9
    # more drafted tokens than max_new: every request is refused
    out, lse = run(max_new=3)
    assert (out == 0).all() and (lse == -float("inf")).all() and _status() == 9
    # rows past the tensor, and before it
    for i, value in ((3, 13), (3, 2**31 - 1), (0, -2)):
        moved = offsets.clone()
        moved[i] = value
        out, lse = run(offsets=moved)
        good.check(out, lse, skip=(2,) if i == 3 else (0,))
        assert _status() == 9
    # a block id past the cache reads as zeros: finite, and nothing else moves
    for value in (-1, good.blocks, 2**31 - 1, -2**31):
        moved = tables.clone()
        moved[1, 3] = value
        out, lse = run(tables=moved)
        good.check(out, lse, skip=(1,))
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        assert _status() == 9
    good.check(*run())
    assert _status() == 0


def test_strided_q_streams_workspaces_and_replay(cuda_device):
    from kta_b200 import ops

    dev = cuda_device
    c = Case([200, 64, 1000], [5, 8, 1], 8, 2, 128, 32, BF16, seed=6)
    out, lse = c.run(dev)
    c.check(out, lse)
    q, kc, vc, tables, ctx, offsets = c.dev
    tree = torch.from_numpy(c.bits).to(dev)
    fused = torch.zeros((c.rows, 12, 128), dtype=BF16, device=dev)
    fused[:, :8] = q
    wide = torch.full((3, tables.shape[1] + 3), -5, dtype=torch.int32, device=dev)
    wide[:, :tables.shape[1]] = tables
    need = ops.tree_attn_workspace_bytes(8, 8, 2, 128)
    pool = [torch.full((need,), 255, dtype=torch.uint8, device=dev) for _ in range(2)]
    args = (fused[:, :8], kc, vc, wide[:, :tables.shape[1]], ctx, offsets, 8, tree)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, ws in zip(streams, pool):  # at the same time, a workspace each
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([ops.tree_attn(*args, workspace=ws) for _ in range(3)][-1])
    torch.cuda.synchronize()
    for o, z in got:
        assert torch.equal(o, out) and torch.equal(z, lse)
    o, z = torch.empty_like(out), torch.empty_like(lse)
    graphs = []
    for ws in pool:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ops.tree_attn(*args, out=o, lse=z, workspace=ws)
    keep = ctx.clone()
    ctx.fill_(10)
    graphs[0].replay()
    ctx.copy_(keep)
    graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(o, out) and torch.equal(z, lse)
    with pytest.raises(ValueError):
        ops.tree_attn(*args, out=o[:, :4])


def test_offsets_past_32_bits(cuda_device):
    """Blocks behind 2^31 elements of the caches."""
    dev = cuda_device
    c = Case([300, 70], [6, 3], 8, 8, 128, 16, BF16, seed=7)
    blocks = 2**31 // (16 * 8 * 128) + c.blocks + 1
    q, kc, vc, tables, ctx, offsets = [t.to(dev) for t in (
        c.q, c.kc, c.vc, torch.from_numpy(c.tables), torch.tensor(c.ctx, dtype=torch.int32),
        torch.from_numpy(c.offsets))]
    from kta_b200 import ops

    big_k = torch.empty((blocks, 16, 8, 128), dtype=BF16, device=dev)
    big_v = torch.empty_like(big_k)
    big_k[-c.blocks:], big_v[-c.blocks:] = kc, vc
    shifted = torch.where(tables >= 0, tables + (blocks - c.blocks), tables)
    out, lse = ops.tree_attn(q, big_k, big_v, shifted, ctx, offsets, 6, torch.from_numpy(c.bits).to(dev))
    c.check(out, lse)
    # and the write: K and V of new tokens to slots there
    freqs, _ = ops.rope_freqs(128, device=dev)
    k = torch.randn((5, 8, 128), device=dev).to(BF16)
    slots = (blocks - 1) * 16 + torch.arange(5, device=dev)
    pos = torch.zeros(5, dtype=torch.int32, device=dev)
    ops.rope_cache(q[:5], k, -k, pos, slots, freqs, big_k, big_v)
    assert torch.equal(big_k[-1, :5], k) and torch.equal(big_v[-1, :5], -k)
    assert _status() == 0


@pytest.mark.parametrize("value", [-1, "past", 2**31 - 1, -2**31])
@pytest.mark.parametrize("block,which", [(16, 3), (16, -1), (128, 1), (256, 0), (256, -1)])
@pytest.mark.parametrize("max_new", [4, 64])  # one kernel and the other
def test_a_block_out_of_range_reads_as_zeros(cuda_device, max_new, block, which, value):
    """Of the context and of the drafted tokens, and one that is two boxes: the formula with zeros for its
    K and V, in every row; stale tiles or another block's values would show."""
    from kta_b200 import ops

    c = Case([40, 900, 7], [4, 4, 4], 8, 2, 128, block, BF16, wide=1, seed=12)
    c.run(cuda_device, max_new=max_new)
    assert _status() == 0
    q, kc, vc, tables, ctx, offsets = c.dev
    last = -(-904 // block) - 1
    at = last if which < 0 else which
    moved = tables.clone()
    moved[1, at] = c.blocks if value == "past" else value
    c.kc[c.tables[1, at]] = 0
    c.vc[c.tables[1, at]] = 0
    out, lse = ops.tree_attn(q, kc, vc, moved, ctx, offsets, max_new, torch.from_numpy(c.bits).to(cuda_device))
    c.check(out, lse)
    assert _status() == 9


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("max_new", [6, 32])
def test_large_scores_in_a_known_order(cuda_device, max_new, dtype):
    """Blocks whose scores grow up to some hundreds, in rising, falling and mixed order."""
    for order in ("up", "down", "mixed"):
        c = Case([900, 600], [6, 6], 8, 2, 128, 16, dtype, seed=4)
        c.q *= 8
        grow = torch.linspace(0.1, 3.0, 57)
        grow = {"up": grow, "down": grow.flip(0),
                "mixed": grow[torch.randperm(57, generator=torch.Generator().manual_seed(5))]}[order].to(dtype)
        for row in c.tables:
            held = torch.from_numpy(row[row >= 0]).long()
            c.kc[held] *= grow[:len(held), None, None, None]
        c.check(*c.run(cuda_device, max_new=max_new))
        assert _status() == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("max_new", [2, 6, 64])  # 8, 24 and 128 query rows
@pytest.mark.parametrize("at", [3, 250, 399])
def test_infinite_values_in_the_context(cuda_device, at, max_new, dtype):
    """Every row sees them: one gives its infinity, two of different signs NaN, NaN itself; the other
    dimensions are as they were, in requests that one CTA has and in ones that several share."""
    for ctx in ([400, 30], [400, 60000]):
        c = Case(ctx, [2, 2], 8, 2, 128, 16, dtype, seed=15)
        c.q *= 0.25  # no weight is lost below the smallest number
        want, want_lse = c.run(cuda_device, max_new=max_new)
        c.check(want, want_lse)
        block, place = c.tables[0, at // 16], at % 16
        c.vc[block, place, 1, 5] = float("inf")
        c.vc[block, place, 1, 6] = -float("inf")
        c.vc[block, place, 1, 7] = float("nan")
        c.vc[block, place, 1, 8] = float("inf")
        c.vc[c.tables[0, 1], 1, 1, 8] = -float("inf")
        out, lse = c.run(cuda_device, max_new=max_new)
        o = out[:2, 4:].cpu()
        assert (o[..., 5] == float("inf")).all() and (o[..., 6] == -float("inf")).all()
        assert torch.isnan(o[..., 7:9]).all()
        keep = [i for i in range(128) if not 5 <= i < 9]
        assert torch.equal(o[..., keep], want[:2, 4:].cpu()[..., keep])
        assert torch.equal(out[:2, :4], want[:2, :4]) and torch.equal(out[2:], want[2:])
        assert torch.equal(lse, want_lse)
        assert _status() == 0


@pytest.mark.parametrize("max_new", [2, 7, 64])  # 8, 28 and 128 query rows
@pytest.mark.parametrize("d", [64, 128])
def test_a_mean_of_the_largest_numbers_is_finite(cuda_device, d, max_new):
    """A weighted mean is never beyond its values: where every V is f16's largest number (clipped
    activations), O is that, and not infinite because the weights were rounded. Here all but one of a
    row's weights are 0.5003 of the first one's: f16 has 0.50049, 4e-4 more, and 65504 (1 + 2^-12) is
    rounded to infinity."""
    scale = -np.log(0.5003)
    c = Case([31, 0, 40, 3000], [2, 2, 1, 2], 8, 2, d, 16, F16, seed=16)
    c.q.zero_()
    c.q[..., 0] = 1
    top = torch.finfo(F16).max
    sign = 1 - 2.0 * (torch.arange(d) % 3 == 0)
    for b, (n, m) in enumerate(zip(c.ctx, c.new)):
        for p in range(n + m):
            c.kc[c.tables[b, p // 16], p % 16] = 0
            c.kc[c.tables[b, p // 16], p % 16, :, 0] = -1.0 if p else 0.0
            c.vc[c.tables[b, p // 16], p % 16] = (top * sign).to(F16)
    out, lse = c.run(cuda_device, max_new=max_new, scale=scale)
    assert torch.isfinite(out).all()
    c.check(out, lse, scale=scale)
    # what is infinite stays so
    c.vc[c.tables[3, 2], 5, 1, 7] = float("inf")
    out, _ = c.run(cuda_device, max_new=max_new, scale=scale)
    assert (out[5:, 4:, 7] == float("inf")).all() and torch.isfinite(out[5:, :4]).all()
    assert _status() == 0
