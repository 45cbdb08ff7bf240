"""A paged cache as a server uses it: every step makes its slots (ops.cache_slots), turns Q and K and
writes K and V (ops.rope_cache) and reads the cache (ops.tree_attn); launched and as a replayed graph.

The slots are whole numbers: equal. V is a copy: equal. Cached K is the rotation's, within the bounds
of test_rope_gpu; O is held against float64 attention over what the cache holds, rotated Q as the
kernel gave it, within the bounds of oracle/paged.py (one rounding of each to the storage type)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
BLOCK, ROWS, MOST = 16, 100, 24


class Server:
    """Requests with random weights' worth of Q, K and V; the host knows lengths, never the blocks."""

    def __init__(self, dev, dtype, hq, hkv, d, batch, seed):
        from kta_b200 import ops

        self.dev, self.dtype, self.hq, self.hkv, self.d = dev, dtype, hq, hkv, d
        self.g = np.random.default_rng(seed)
        self.gen = torch.Generator().manual_seed(seed)
        self.freqs, _ = ops.rope_freqs(d, device=dev)
        self.pool = torch.from_numpy(self.g.permutation(200).astype(np.int32)).to(dev)
        self.kc = torch.full((200, BLOCK, hkv, d), float("nan"), dtype=dtype, device=dev)
        self.vc = torch.full_like(self.kc, float("nan"))
        self.tables = torch.full((batch, 24), -1, dtype=torch.int32, device=dev)
        self.ctx, self.new = (torch.zeros(batch, dtype=torch.int32, device=dev) for _ in range(2))
        self.fused = torch.zeros((ROWS, hq + 2 * hkv, d), dtype=dtype, device=dev)
        self.tree = torch.zeros(ROWS, dtype=torch.int64, device=dev)
        self.free = self.pool[:64].clone()
        self.taken = 0
        self.k = [np.zeros((0, hkv, d)) for _ in range(batch)]  # before rotation, by position
        self.v = [np.zeros((0, hkv, d)) for _ in range(batch)]
        self.at = [0] * batch

    def step(self):
        from kta_b200 import ops

        slots, pos, offsets, used = ops.cache_slots(self.ctx, self.new, self.tables, self.free, BLOCK, ROWS)
        q, k, v = self.fused.split([self.hq, self.hkv, self.hkv], 1)
        turned = ops.rope_cache(q, k, v, pos, slots, self.freqs, self.kc, self.vc)
        out = torch.full_like(turned, 7.0)
        lse = torch.full((ROWS, self.hq), 7.0, device=self.dev)
        ops.tree_attn(turned, self.kc, self.vc, self.tables, self.ctx, offsets, MOST, self.tree, out=out,
                      lse=lse)
        return slots, pos, offsets, used, turned, out, lse

    def feed(self, ctx, new):
        """The step's inputs, in the memory that a captured graph reads."""
        self.fused.copy_(torch.randn(self.fused.shape, generator=self.gen).to(self.dtype))
        bits = []
        for n in new:
            parents = [int(self.g.integers(-1, i)) if i else -1 for i in range(n)]
            bits += paged.tree_bits(parents)
        self.tree.copy_(torch.tensor(bits + [0] * (ROWS - len(bits)), dtype=torch.int64))
        self.ctx.copy_(torch.tensor(ctx, dtype=torch.int32))
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        self.free.copy_(self.pool[self.taken:self.taken + 64])
        return bits

    def check(self, ctx, new, bits, result):
        slots, pos, offsets, used, turned, out, lse = (t.cpu() for t in result)
        total, before = sum(new), self.taken
        held = [-(-c // BLOCK) for c in ctx]
        assert int(used) == sum(-(-(c + n) // BLOCK) - h for c, n, h in zip(ctx, new, held))
        self.taken += int(used)
        assert offsets.tolist() == [0, *np.cumsum(new)]
        assert (slots[total:] == -1).all() and (out[total:] == 7).all() and (lse[total:] == 7).all()
        fused, tables = self.fused.double().cpu().numpy(), self.tables.cpu().numpy()
        assert before + int(used) == len({i for b, (c, n) in enumerate(zip(ctx, new))
                                          for i in tables[b, :-(-(c + n) // BLOCK)].tolist()})
        kc, vc = self.kc.double().cpu().numpy(), self.vc.double().cpu().numpy()
        eps = torch.finfo(self.dtype).eps / 2
        freqs, group = self.freqs.tolist(), self.hq // self.hkv
        for b, (c, n) in enumerate(zip(ctx, new)):
            a, L = int(offsets[b]), c + n
            if n == 0:
                continue
            self.k[b] = np.concatenate([self.k[b][:c], fused[a:a + n, self.hq:self.hq + self.hkv]])
            self.v[b] = np.concatenate([self.v[b][:c], fused[a:a + n, self.hq + self.hkv:]])
            assert pos[a:a + n].tolist() == list(range(c, L))
            ids = tables[b, :-(-L // BLOCK)]
            k, v = (x[ids].reshape(-1, self.hkv, self.d)[:L] for x in (kc, vc))
            assert np.array_equal(v, self.v[b])
            q = fused[a:a + n, :self.hq]
            for got, x, at in ((k, self.k[b], range(L)), (turned[a:a + n].double().numpy(), q, range(c, L))):
                half = self.d // 2
                pair = np.abs(x[..., :half]) + np.abs(x[..., half:])
                fp32 = 6e-7 * np.concatenate([pair, pair], -1)
                want = paged.rope(x, at, freqs, False)
                assert (np.abs(got - want) <= fp32 + eps * (np.abs(want) + fp32) + 2.0 ** -25).all()
            sight = paged.seen(c, n, bits[a:a + n])
            for h in range(self.hq):
                parts = paged.attention(turned[a:a + n, h].double().numpy(), k[:, h // group],
                                        v[:, h // group], sight, self.d ** -0.5)
                sub = 2.0 ** -25 if self.dtype == torch.float16 else 0.0
                far, far_lse = paged.attention_bounds(sight, eps, sub, *parts)
                assert (np.abs(out[a:a + n, h].double().numpy() - parts[0]) <= far).all(), (b, h)
                assert (np.abs(lse[a:a + n, h].double().numpy() - parts[1]) <= far_lse).all(), (b, h)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype,hq,hkv,d", [(torch.bfloat16, 8, 2, 128), (torch.float16, 12, 4, 64)])
def test_steps_of_a_server(cuda_device, dtype, hq, hkv, d, captured):
    from kta_b200 import lib

    batch = 5
    s = Server(cuda_device, dtype, hq, hkv, d, batch, seed=hq)
    ctx = [0] * batch
    # a first prompt, its rest, draft trees of which some tokens are kept, single tokens, and steps in
    # which a request rests; what was rejected is overwritten
    plan = [([24, 7, 1, 20, 0], None), ([24, 0, 5, 24, 16], None), ([8, 8, 8, 8, 8], [1, 3, 8, 0, 5]),
            ([1, 1, 1, 1, 1], None), ([0, 0, 0, 0, 1], None), ([16, 24, 2, 1, 9], [16, 0, 1, 1, 2]),
            ([1, 0, 1, 0, 1], None)]
    graph = None
    if captured:
        s.feed(ctx, plan[0][0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = s.step()
    for new, kept in plan:
        bits = s.feed(ctx, new)
        if captured:
            graph.replay()
        else:
            result = s.step()
        torch.cuda.synchronize()
        s.check(ctx, new, bits, result)
        ctx = [c + (n if kept is None else kept[i]) for i, (c, n) in enumerate(zip(ctx, new))]
        # blocks that only rejected tokens used stay with their request: the next step takes new ones
        # for the same places, so give those back first, as a server does
        if kept is not None:
            tables = s.tables.cpu()
            back = []
            for b, (c, n) in enumerate(zip(ctx, new)):
                start = c - kept[b]
                back += tables[b, -(-c // BLOCK):-(-(start + n) // BLOCK)].tolist()
            if back:
                s.taken -= len(back)
                s.pool[s.taken:s.taken + len(back)] = torch.tensor(back, dtype=torch.int32)
    assert lib.device_status(clear=True)[0] == 0


def test_two_streams_at_once(cuda_device):
    """Two servers' steps at the same time, each on its own stream: as one after the other."""
    made = []
    for pair in (False, True):
        servers = [Server(cuda_device, torch.bfloat16, 8, 2, 128, 5, seed=i) for i in range(2)]
        for s in servers:
            s.feed([0] * 5, [20, 3, 24, 1, 9])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() if pair else torch.cuda.current_stream() for _ in servers]
        results = [[], []]
        for _ in range(3):
            for s, stream, r in zip(servers, streams, results):
                with torch.cuda.stream(stream):
                    r.append(s.step())
        torch.cuda.synchronize()
        made.append([[t.cpu() for t in r[-1]] for r in results])
    for one, two in zip(*made):
        for a, b in zip(one, two):
            assert torch.equal(a, b)


def _after(free, used, tables, ctx, new, kept):
    """What a server does between steps, on the device: ids that were taken leave the free list, those of
    blocks behind the tokens it keeps return to it, and no list or length passes through the host."""
    column = torch.arange(tables.shape[1], device=tables.device)
    back = (column >= -(-kept // BLOCK)[:, None]) & (column < -(-(ctx + new) // BLOCK)[:, None])
    rest = (torch.arange(len(free), device=free.device) >= used) & (free >= 0)
    live, ids = torch.cat([rest, back.flatten()]), torch.cat([free, tables.flatten()])
    order = torch.argsort(live.logical_not().byte(), stable=True)[:len(free)]  # the live ones first
    free.copy_(torch.where(live, ids, -1)[order])
    ctx.copy_(kept)


@pytest.mark.parametrize("captured", [False, True])
def test_a_pool_that_only_the_device_knows(cuda_device, captured):
    """Steps with rejected drafts, the free list kept on the device and the whole of it replayed as one
    graph: no block has two owners, none is lost, and every kept token's V is where the table says."""
    from kta_b200 import lib, ops

    dev, batch, blocks, heads, d = cuda_device, 6, 40, 2, 64
    g = np.random.default_rng(3)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    free = i32(g.permutation(blocks).tolist())
    tables = torch.full((batch, 12), -1, dtype=torch.int32, device=dev)
    ctx, new, kept = (torch.zeros(batch, dtype=torch.int32, device=dev) for _ in range(3))
    kc = torch.zeros((blocks, BLOCK, heads, d), dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    freqs, _ = ops.rope_freqs(d, device=dev)
    x = torch.zeros((ROWS, 3 * heads, d), dtype=torch.bfloat16, device=dev)

    def step():
        slots, pos, offsets, used = ops.cache_slots(ctx, new, tables, free, BLOCK, ROWS)
        q, k, v = x.split(heads, 1)
        q = ops.rope_cache(q, k, v, pos, slots, freqs, kc, vc)
        out, _ = ops.tree_attn(q, kc, vc, tables, ctx, offsets, MOST)
        _after(free, used, tables, ctx, new, kept)
        return offsets, out

    if captured:
        for _ in range(2):
            step()  # no new tokens: nothing moves
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = step()
    held = [np.zeros((0, heads, d)) for _ in range(batch)]
    for i in range(12):
        n = g.integers(0, 17, batch) if i else np.array([16, 1, 15, 17, 0, 24])
        keep = np.array([int(g.integers(0, m + 1)) for m in n])
        if i % 4 == 3:  # a request ends: all of its blocks return
            keep[i % batch] = -len(held[i % batch])
        x.copy_(torch.from_numpy(g.standard_normal(x.shape)).to(torch.bfloat16))
        new.copy_(i32(n.tolist()))
        kept.copy_(i32([len(h) + int(m) for h, m in zip(held, keep)]))
        if captured:
            graph.replay()
        else:
            result = step()
        torch.cuda.synchronize()
        v, offsets = x[:, 2 * heads:].double().cpu().numpy(), result[0].tolist()
        assert offsets == [0, *np.cumsum(n).tolist()]
        table, pool, cache = tables.tolist(), free.tolist(), vc.double().cpu().numpy()
        owned = []
        for b in range(batch):
            held[b] = np.concatenate([held[b], v[offsets[b]:offsets[b + 1]]])[:len(held[b]) + keep[b]]
            ids = table[b][:-(-len(held[b]) // BLOCK)]
            assert np.array_equal(cache[ids].reshape(-1, heads, d)[:len(held[b])], held[b])
            owned += ids
        assert sorted(owned + [f for f in pool if f >= 0]) == list(range(blocks))
        assert pool[len(pool) - len(owned):] == [-1] * len(owned)
    assert lib.device_status(clear=True)[0] == 0
