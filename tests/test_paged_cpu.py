"""Refusals of the paged-cache entries without a GPU: argument checks of the C ABI before any
device work, and of the tensor wrappers; frequencies; the float64 forms against each other."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from kta_b200 import lib, ops
from oracle import paged

A, ODD2, ODD4, ODD8 = 0x10000, 0x10002, 0x10004, 0x10008
INVALID, UNSUPPORTED, ALIGN, WORKSPACE, NO_DEVICE = 1, 2, 3, 7, 6
NO_GPU = not torch.cuda.is_available()


def test_cache_slots_argument_checks():
    f = lib.load().kta_cache_slots

    def call(ptr=(), B=4, blocks=16, stride=16, free=8, block=16, rows=64):
        p = [A] * 8
        for i, v in dict(ptr).items():
            p[i] = v
        return f(*p, B, blocks, stride, free, block, rows, None)

    for i in (0, 1, 2, 4, 5, 6, 7):
        assert call({i: None}) == INVALID
    assert call({3: None}) == INVALID               # a free list of eight without memory
    for kw in (dict(B=0), dict(blocks=0), dict(block=0), dict(rows=0), dict(free=-1),
               dict(stride=15)):
        assert call(**kw) == INVALID, kw
    for kw in (dict(B=2049), dict(block=1 << 21), dict(blocks=1 << 28, stride=1 << 28),
               dict(rows=(1 << 30) + 1), dict(free=1 << 31)):
        assert call(**kw) == UNSUPPORTED, kw
    for i in (0, 1, 2, 3, 5, 6, 7):
        assert call({i: ODD2}) == ALIGN
    assert call({4: ODD4}) == ALIGN
    if NO_GPU:
        assert call() == NO_DEVICE
        assert call({3: None}, free=0) == NO_DEVICE
        assert call(B=1, stride=0) == NO_DEVICE


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_rope_argument_checks(dt):
    f = getattr(lib.load(), f"kta_rope_{dt}")

    def call(x=A, pos=A, size=4, freqs=A, y=A, n=8, h=4, d=128, rot=64, xs=(512, 128),
             ys=(512, 128), scale=1.0):
        return f(x, pos, size, freqs, y, n, h, d, rot, *xs, *ys, 0, 0, scale, None)

    for kw in (dict(x=None), dict(pos=None), dict(freqs=None), dict(y=None), dict(n=0), dict(h=0),
               dict(d=0), dict(rot=0), dict(rot=144), dict(size=2), dict(scale=math.inf),
               dict(scale=math.nan), dict(xs=(-512, 128)), dict(xs=(512, -128)),
               dict(ys=(512, 64)), dict(ys=(64, 128)), dict(ys=(256, 128)), dict(ys=(0, 128)),
               dict(ys=(512, 0))):
        assert call(**kw) == INVALID, kw
    for kw in (dict(d=1040, rot=16, xs=(4160, 1040), ys=(4160, 1040)), dict(n=(1 << 30) + 1)):
        assert call(**kw) == UNSUPPORTED, kw
    for kw in (dict(d=120, rot=16), dict(rot=24), dict(x=ODD8), dict(y=ODD8), dict(pos=ODD2),
               dict(pos=ODD4, size=8), dict(freqs=ODD4), dict(xs=(516, 128)), dict(ys=(516, 132))):
        assert call(**kw) == ALIGN, kw
    if NO_GPU:
        for kw in (dict(), dict(xs=(0, 0)), dict(ys=(128, 1024)), dict(pos=ODD4), dict(n=1, ys=(0, 128)),
                   dict(h=1, ys=(128, 0))):
            assert call(**kw) == NO_DEVICE, kw


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_rope_cache_argument_checks(dt):
    f = getattr(lib.load(), f"kta_rope_cache_{dt}")

    def call(ptr=(), size=4, n=8, hq=8, hkv=2, d=128, rot=128, strides=None, num_slots=64, scale=1.0):
        p = [A] * 9  # Q, K, V, positions, slots, freqs, Qo, Kc, Vc
        for i, v in dict(ptr).items():
            p[i] = v
        s = strides or (1024, 128, 256, 128, 256, 128, 1024, 128)
        return f(*p[:4], size, *p[4:], n, hq, hkv, d, rot, (ctypes.c_int64 * 8)(*s), num_slots, 0, scale,
                 None)

    for i in range(9):
        assert call({i: None}) == INVALID, i
    for kw in (dict(n=0), dict(hq=0), dict(hkv=0), dict(num_slots=0), dict(rot=256),
               dict(scale=math.inf), dict(strides=(1024, 128, 256, -8, 256, 128, 1024, 128)),
               dict(strides=(1024, 128, 256, 128, 256, 128, 512, 128))):
        assert call(**kw) == INVALID, kw
    for i in (0, 1, 2, 6, 7, 8):
        assert call({i: ODD8}) == ALIGN, i
    assert call({4: ODD4}) == ALIGN and call({5: ODD4}) == ALIGN
    assert call(strides=(1024, 128, 260, 128, 256, 128, 1024, 128)) == ALIGN
    if NO_GPU:
        assert call() == NO_DEVICE
        assert call(strides=(1536, 128) * 4) == NO_DEVICE  # slices of a fused tensor


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_tree_attn_argument_checks(dt):
    L = lib.load()
    f = getattr(L, f"kta_tree_attn_{dt}")
    full = L.kta_tree_attn_workspace_bytes(64, 32, 8, 128)
    assert full > 0
    for bad in ((0, 32, 8, 128), (65, 32, 8, 128), (8, 33, 8, 128), (8, 34, 2, 128), (8, 8, 8, 96)):
        assert L.kta_tree_attn_workspace_bytes(*bad) == 0

    def call(ptr=(), n=32, B=4, hq=32, hkv=8, d=128, q=4096, blocks=100, block=16, width=50, stride=50,
             new=8, scale=0.1, ws=A, size=full):
        p = [A] * 9  # Q, Kc, Vc, tables, ctx, offsets, tree, O, LSE
        p[7] = A + (1 << 20)
        for i, v in dict(ptr).items():
            p[i] = v
        return f(*p, n, B, hq, hkv, d, q, blocks, block, width, stride, new, scale, ws, size, None)

    for i in (0, 1, 2, 3, 4, 5, 7, 8):
        assert call({i: None}) == INVALID, i
    for kw in (dict(n=0), dict(B=0), dict(hq=0), dict(hkv=0), dict(d=0), dict(blocks=0), dict(block=0),
               dict(width=0), dict(new=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
               dict(stride=49), dict(q=4088)):
        assert call(**kw) == INVALID, kw
    for kw in (dict(new=65), dict(d=96), dict(hq=30), dict(hq=136), dict(block=4), dict(block=48),
               dict(block=512), dict(B=2049), dict(width=1 << 27, stride=1 << 27),
               dict(blocks=1 << 24)):
        assert call(**kw) == UNSUPPORTED, kw
    for kw in (dict(ptr={0: ODD8}), dict(ptr={1: ODD8}), dict(ptr={2: ODD8}), dict(ptr={7: A + (1 << 20) + 8}),
               dict(ptr={7: A + (1 << 20) + 16}),
               dict(ptr={3: ODD2}), dict(ptr={4: ODD2}), dict(ptr={5: ODD2}), dict(ptr={6: ODD4}),
               dict(ptr={8: ODD2}), dict(q=4100)):
        assert call(**kw) == ALIGN, kw
    # Q is 32 rows of 8192 bytes, or as many 16384 bytes apart
    high, size = A + (1 << 20), 32 * 8192
    for at in (high, high + size - 32, high - size + 32):
        assert call({0: high, 7: at}) == INVALID
    assert call({0: high, 7: high + size}, q=8192) == INVALID
    need = L.kta_tree_attn_workspace_bytes(8, 32, 8, 128)
    assert call(ws=None) == WORKSPACE and call(size=need - 1) == WORKSPACE and call(ws=ODD8) == WORKSPACE
    if NO_GPU:
        assert call(size=need) == NO_DEVICE and call({6: None}) == NO_DEVICE
        assert call(B=1, stride=0) == NO_DEVICE
        assert call({0: high, 7: high + size}) == call({0: high, 7: high - size}) == NO_DEVICE


def test_wrappers_refuse_wrong_tensors():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    pos, freqs = torch.zeros(4, dtype=torch.int32), torch.zeros(16, dtype=torch.float64)
    slots = torch.zeros(4, dtype=torch.int64)
    cache = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    for args in ((x.float(), pos, freqs), (x[0], pos, freqs), (x, pos[:3], freqs), (x, pos.float(), freqs),
                 (x, pos, freqs.float()), (x.transpose(1, 2), pos, freqs), (x, pos[:, None], freqs),
                 (x, pos, freqs)):  # the last one: tensors of the host
        with pytest.raises(ValueError):
            ops.rope(*args)
    with pytest.raises(ValueError):
        ops.rope(x, pos, freqs, out=x[:, :1])
    good = dict(q=x, k=x, v=x, positions=pos, slots=slots, freqs=freqs, k_cache=cache, v_cache=cache)
    for change in (dict(k=x[:, :1]), dict(v=x[:, :1]), dict(k=x.half()), dict(slots=pos),
                   dict(slots=slots[:2]), dict(k_cache=cache.half()), dict(v_cache=cache[:2]),
                   dict(k_cache=cache[..., :32]), dict(k_cache=cache.transpose(0, 1)), dict()):
        with pytest.raises(ValueError):
            ops.rope_cache(**{**good, **change})
    lens, tab = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 5, dtype=torch.int32)
    offs, tree = torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)
    attn = dict(q=x, k_cache=cache, v_cache=cache, block_tables=tab, context_lens=lens, offsets=offs,
                max_new=2, tree=tree)
    for change in (dict(q=x.float()), dict(q=x[:, :, :32]), dict(block_tables=tab.long()),
                   dict(block_tables=tab[:1]), dict(block_tables=tab.t()), dict(context_lens=lens.long()),
                   dict(offsets=offs[:2]), dict()):
        with pytest.raises(ValueError):
            ops.tree_attn(**{**attn, **change})
    for args in ((lens, lens[:1], tab, lens, 16, 4), (lens, lens, tab.t(), lens, 16, 4),
                 (lens.long(), lens, tab, lens, 16, 4), (lens, lens, tab, lens, 16, 4)):
        with pytest.raises(ValueError):
            ops.cache_slots(*args)


def test_rope_freqs():
    f, scale = ops.rope_freqs(64, 10000.0, device="cpu")
    assert scale == 1.0 and f.dtype == torch.float64
    want = [10000.0 ** (-2 * i / 64) for i in range(32)]
    assert np.allclose(f.numpy(), want, rtol=1e-14)
    lin, _ = ops.rope_freqs(64, scaling="linear", factor=4.0, device="cpu")
    assert np.allclose(lin.numpy(), np.array(want) / 4, rtol=1e-14)
    ntk, _ = ops.rope_freqs(64, scaling="ntk", factor=4.0, device="cpu")
    assert math.isclose(ntk[0], 1.0) and math.isclose(ntk[-1], want[-1] / 4, rel_tol=1e-12)
    for kind in ("bands", "yarn"):
        g, s = ops.rope_freqs(64, scaling=kind, factor=8.0, device="cpu")
        assert math.isclose(g[0], want[0]) and math.isclose(g[-1], want[-1] / 8, rel_tol=1e-12)
        assert all(a >= b for a, b in zip(g.tolist(), g.tolist()[1:]))
        turns = 4096 * np.array(want) / (2 * math.pi)
        assert np.allclose(g.numpy()[turns > 40], np.array(want)[turns > 40])
        assert np.allclose(g.numpy()[turns < 0.7], np.array(want)[turns < 0.7] / 8)
        assert math.isclose(s, 1 + 0.1 * math.log(8) if kind == "yarn" else 1.0)
    for bad in (dict(rot=3), dict(rot=0), dict(rot=64, factor=0.5), dict(rot=64, scaling="other"),
                dict(rot=2, scaling="ntk"), dict(rot=64, low_turns=4, high_turns=2)):
        with pytest.raises(ValueError):
            ops.rope_freqs(device="cpu", **bad)


def _yarn(rot, base, factor, original_len, low_turns=1.0, high_turns=32.0):
    """The ramp pair by pair: pair index x makes original_len base^(-2 x / rot) / (2 pi) turns, solved for
    x at both bounds; whole indices outward, in 0 .. rot - 1 (the upper one may lie past the last pair)."""
    def index(turns):
        return rot / 2 * math.log(original_len / (2 * math.pi * turns), base)

    low, high = max(math.floor(index(high_turns)), 0), min(math.ceil(index(low_turns)), rot - 1)
    out = []
    for i in range(rot // 2):
        divided = min(max((i - low) / (high - low), 0.0), 1.0)
        out.append(base ** (-2 * i / rot) * (1 - divided + divided / factor))
    return out


@pytest.mark.parametrize("rot,base,original_len,bounds,last", [
    (64, 10000.0, 4096, (10, 23), 0.25),               # both bounds among the pairs
    (64, 10000.0, 131072, (22, 35), 0.25 + 0.75 * 4 / 13),   # the upper one past the last pair, 31
    (128, 10000.0, 131072, (45, 70), 0.25 + 0.75 * 7 / 25),  # ... 63
    (16, 10000.0, 32768, (4, 8), 0.25 + 0.75 * 1 / 4),       # ... 7
    (64, 100.0, 1 << 30, (107, 63), 1.0),              # even the lower one: every frequency is kept
])
def test_yarn_ramp_between_its_bounds(rot, base, original_len, bounds, last):
    """The bounds by hand: rot / 2 * log_base(original_len / (2 pi turns))."""
    freqs, _ = ops.rope_freqs(rot, base, scaling="yarn", factor=4.0, original_len=original_len, device="cpu")
    plain = base ** (-2.0 * (rot // 2 - 1) / rot)
    assert math.isclose(freqs[-1], plain * last, rel_tol=1e-12)
    low, high = bounds
    if low < high:
        assert np.allclose(freqs.numpy(), _yarn(rot, base, 4.0, original_len), rtol=1e-12, atol=0)
        if low + 1 < rot // 2:
            assert freqs[low] == base ** (-2.0 * low / rot) and freqs[low + 1] < base ** (-2.0 * (low + 1) / rot)


def test_yarn_needs_frequencies_that_fall():
    for base in (1.0, 0.5):  # every pair turns as fast as the first, or faster: no index has the turns
        with pytest.raises(ValueError):
            ops.rope_freqs(64, base, scaling="yarn", factor=2.0, device="cpu")


def test_float64_forms():
    """The oracle on cases that can be told by hand."""
    assert paged.tree_bits([-1, 0, 0, 1]) == [1, 3, 5, 11]
    assert paged.tree_bits([-1] * 64)[63] == -(1 << 63)
    assert paged.seen(2, 2, [1, 2]).tolist() == [[1, 1, 1, 0], [1, 1, 0, 1]]
    t, s, p, o, u = paged.cache_slots([3, 0], [2, 1], [[5, -1], [-1, -1]], [8, 9, 4], 4, 4)
    assert t.tolist() == [[5, 8], [9, -1]] and s.tolist() == [23, 32, 36, -1]
    assert p.tolist() == [3, 4, 0, 0] and o.tolist() == [0, 2, 3] and u == 2
    x = np.array([[[1.0, 0.0, 2.0, 0.0]]])
    y = paged.rope(x, [1], [math.pi / 2, math.pi], True)
    assert np.allclose(y, [[[0, 1, -2, 0]]])
    y = paged.rope(x, [1], [math.pi / 2, math.pi], False)
    assert np.allclose(y, [[[-2, 0, 1, 0]]])
    q, k = np.zeros((1, 2)), np.ones((3, 2))
    out, lse, *_ = paged.attention(q, k, np.arange(6.0).reshape(3, 2), np.array([[True, True, False]]), 1.0)
    assert np.allclose(out, [[1, 2]]) and math.isclose(lse[0], math.log(2))


def test_rope_oracle_at_far_positions():
    """Against libm's sine and cosine, which reduce any argument; position * frequency is exact here."""
    for f, n in ((1.0, 2**40 + 3), (1.0, -2**53 + 1), (0.75, 2**50 + 1), (1.0 + 2.0 ** -20, 2**31 - 1),
                 (96.0, 2**46 + 5), (-3.0, 2**51 - 1)):
        y = paged.rope(np.array([[[1.0, 0.0]]]), [n], [f], True)[0, 0]
        assert np.allclose(y, [math.cos(n * f), math.sin(n * f)], rtol=0, atol=4e-16), (f, n)


def test_rope_of_a_tensor_that_needs_a_gradient_refuses_out():
    """An output given by the caller has no history: the gradient would be lost without a word."""
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, requires_grad=True)
    pos, freqs = torch.zeros(4, dtype=torch.int32), torch.zeros(16, dtype=torch.float64)
    for args, out in (((x, pos, freqs), torch.zeros(4, 2, 64, dtype=torch.bfloat16)), ((x, pos, freqs), x),
                      ((x.detach(), pos, freqs.clone().requires_grad_()), None)):
        with pytest.raises(ValueError, match="gradient"):
            ops.rope(*args, out=out)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_tree_attn_scale_in_its_own_units(dt):
    """The kernel's scores are in powers of two: a scale whose scale * log2(e) is infinite makes NaN of
    every masked key (-inf + inf), so it is refused like an infinite one."""
    L = lib.load()
    need = L.kta_tree_attn_workspace_bytes(1, 8, 2, 64)
    largest = 3.4028235e38

    def call(scale):
        return getattr(L, f"kta_tree_attn_{dt}")(A, A, A, A, A, A, None, A + (1 << 20), A, 1, 1, 8, 2, 64, 512,
                                                 4, 16, 2, 2, 1, scale, A, need, None)

    for scale in (largest, largest / 1.4, math.inf, math.nan, 0.0, -0.0):
        assert call(scale) == INVALID, scale
    if NO_GPU:
        assert call(largest / 1.5) == call(1e-30) == NO_DEVICE
