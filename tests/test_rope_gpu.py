"""Rotary positions on the GPU (ops.rope, ops.rope_cache) against the float64 form.

Tolerance, from the arithmetic: the angle is exact to 2^-25 of a half turn (1e-7 rad), cos and
sin to 2 ulp, scale and the two products and the sum one rounding each (2^-24): 6e-7 of
scale (|a| + |b|) in fp32, then half a step of the storage type (and half a subnormal step)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _close(got, x, want, scale, rot, interleaved, dtype):
    """got against the float64 result `want` of rotating x."""
    mag = np.abs(x)
    pair = np.zeros_like(mag)
    if interleaved:
        pair[..., 0:rot:2] = pair[..., 1:rot:2] = mag[..., 0:rot:2] + mag[..., 1:rot:2]
    else:
        pair[..., :rot // 2] = pair[..., rot // 2:rot] = mag[..., :rot // 2] + mag[..., rot // 2:rot]
    fp32 = 6e-7 * abs(scale) * pair
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half
    err = np.abs(got.double().cpu().numpy() - want)
    bad = err > fp32 + half * (np.abs(want) + fp32) + tiny
    assert not bad.any(), f"{int(bad.sum())} off, worst {err.max():.3e}"
    assert np.array_equal(got.double().cpu().numpy()[..., rot:], x[..., rot:])


def _x(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,h,d,rot", [(1, 1, 16, 16), (1, 32, 128, 128), (7, 5, 64, 32),
                                       (63, 3, 80, 48), (130, 8, 128, 64), (1201, 2, 128, 128),
                                       (301, 7, 256, 256), (2, 1, 1024, 1008)])
def test_forward_and_gradient(cuda_device, n, h, d, rot, interleaved, dtype):
    from kta_b200 import ops

    x = _x((n, h, d), dtype)
    freqs, _ = ops.rope_freqs(rot, device="cpu")
    pos = torch.randint(0, 5000, (n,), generator=torch.Generator().manual_seed(1))
    for inverse, scale, pt in ((False, 1.0, torch.int32), (True, 1.25, torch.int64)):
        got = ops.rope(x.to(cuda_device), pos.to(pt).to(cuda_device), freqs.to(cuda_device),
                       interleaved=interleaved, inverse=inverse, scale=scale)
        torch.cuda.synchronize()
        want = paged.rope(x.double().numpy(), pos.tolist(), freqs.tolist(), interleaved, inverse, scale)
        _close(got, x.double().numpy(), want, scale, rot, interleaved, dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,h,d,rot", [(5000, 8, 128, 128), (20001, 2, 128, 96), (2400, 20, 256, 64),
                                       (40000, 1, 64, 64)])
def test_more_than_a_wave(cuda_device, n, h, d, rot, interleaved):
    """Several items to a thread, and several tokens to a CTA; in place, what does not turn stays."""
    from kta_b200 import ops

    x = _x((n, h, d), torch.bfloat16, 3)
    freqs, _ = ops.rope_freqs(rot, device="cpu")
    pos = torch.randint(0, 100000, (n,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    dev, at, turn = x.to(cuda_device), pos.to(cuda_device), freqs.to(cuda_device)
    got = ops.rope(dev, at, turn, interleaved=interleaved, scale=0.75)
    want = paged.rope(x.double().numpy(), pos.tolist(), freqs.tolist(), interleaved, False, 0.75)
    _close(got, x.double().numpy(), want, 0.75, rot, interleaved, torch.bfloat16)
    assert ops.rope(dev, at, turn, interleaved=interleaved, scale=0.75, out=dev) is dev
    assert torch.equal(dev, got)


def test_far_and_negative_positions(cuda_device):
    from kta_b200 import ops

    freqs, scale = ops.rope_freqs(128, 500000.0, scaling="yarn", factor=32.0, device="cpu")
    pos = [0, 1, -1, 999_999, 16_777_217, 2**31 - 1, -2**31, 2**40 + 3, -2**40]
    x = _x((len(pos), 4, 128), torch.float16)
    got = ops.rope(x.to(cuda_device), torch.tensor(pos).to(cuda_device), freqs.to(cuda_device),
                   scale=scale)
    torch.cuda.synchronize()
    # the 64-bit fraction of a turn is off by 2^-64 / 2 + 2^-53 relative of the frequency: times
    # 2^40 under 2e-4 rad; exact to fp32 for the positions below 2^31 (1e-6 rad at 2^31)
    want = paged.rope(x.double().numpy(), pos, freqs.tolist(), False, False, scale)
    _close(got[:5], x[:5].double().numpy(), want[:5], scale, 128, False, torch.float16)
    err = np.abs(got.double().cpu().numpy() - want)
    assert err.max() < 2e-3 + 2e-4 * 2 * np.abs(x.double().numpy()).max() * scale


def test_gradient_is_the_transpose_and_matches_differences(cuda_device):
    """<g, R x> = <R^T g, x>, and R is linear: (R(x + h) - R(x)) = R h."""
    from kta_b200 import ops

    dev = cuda_device
    freqs, _ = ops.rope_freqs(64, device=dev)
    pos = torch.arange(100, 137, device=dev, dtype=torch.int32)
    for inter in (False, True):
        x, g = _x((37, 3, 64), torch.float16, 2).to(dev), _x((37, 3, 64), torch.float16, 3).to(dev)
        y = ops.rope(x, pos, freqs, interleaved=inter, scale=1.5).double()
        gx = ops.rope(g, pos, freqs, interleaved=inter, inverse=True, scale=1.5).double()
        a, b = (g.double() * y).sum(-1), (gx * x.double()).sum(-1)
        # each side is a sum of 64 products with one rounding of half a step: Cauchy-Schwarz
        bound = 2.0 ** -11 * 1.5 * (g.double().norm(dim=-1) * x.double().norm(dim=-1)) * 2 + 1e-5
        assert ((a - b).abs() <= bound).all()
        basis = torch.zeros_like(x)
        basis[..., 5] = 1.0  # a difference of one coordinate: a column of R
        col = ops.rope(basis, pos, freqs, interleaved=inter, scale=1.5).double()
        dot = (g.double() * col).sum(-1)
        assert ((dot - gx[..., 5]).abs() <= 2.0 ** -11 * (gx[..., 5].abs() + 2 * 1.5 * 2 *
                                                          g.double().abs().amax(-1)) + 1e-5).all()


def test_views_in_place_streams_and_replay(cuda_device):
    from kta_b200 import ops

    dev = cuda_device
    freqs, _ = ops.rope_freqs(96, device=dev)
    n, h, d = 50, 6, 128
    fused = _x((n, h + 4, d), torch.bfloat16, 5).to(dev)
    pos = torch.arange(n, device=dev, dtype=torch.int32) * 3
    x = fused[:, 2:2 + h]
    want = paged.rope(x.double().cpu().numpy(), pos.tolist(), freqs.tolist(), True)
    plain = ops.rope(x, pos, freqs, interleaved=True)
    _close(plain, x.double().cpu().numpy(), want, 1.0, 96, True, torch.bfloat16)
    # head-major output, and one row broadcast over all heads
    out = torch.full((h, n, d), 7.0, dtype=torch.bfloat16, device=dev)
    ops.rope(x, pos, freqs, interleaved=True, out=out.transpose(0, 1))
    assert torch.equal(out.transpose(0, 1), plain)
    one = ops.rope(x[:, :1].expand(n, 3, d), pos, freqs, interleaved=True)
    assert torch.equal(one, plain[:, :1].expand(n, 3, d))
    # in place, in a slice: nothing around it moves
    keep = fused.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.rope(x, pos, freqs, interleaved=True, out=x)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(fused[:, 2:2 + h], plain)
    assert torch.equal(fused[:, :2], keep[:, :2]) and torch.equal(fused[:, 2 + h:], keep[:, 2 + h:])
    src = keep[:, 2:2 + h].contiguous()
    dst = torch.empty_like(src)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rope(src, pos, freqs, interleaved=True, out=dst)
    pos.add_(1)
    graph.replay()
    pos.sub_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dst, plain)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hkv,d,rot,bs", [(1, 1, 1, 16, 16, 16), (9, 8, 2, 128, 128, 16),
                                               (65, 5, 5, 64, 32, 8), (700, 32, 8, 128, 64, 64),
                                               (3001, 8, 4, 128, 96, 32), (1000, 32, 8, 128, 128, 16)])
def test_rope_cache(cuda_device, n, hq, hkv, d, rot, bs, interleaved, dtype):
    from kta_b200 import lib, ops

    dev = cuda_device
    fused = _x((n, hq + 2 * hkv, d), dtype, 8).to(dev)
    q, k, v = fused.split([hq, hkv, hkv], 1)
    freqs, _ = ops.rope_freqs(rot, device=dev)
    blocks = -(-n // bs) + 2
    g = torch.Generator().manual_seed(4)
    slots = torch.randperm(blocks * bs, generator=g)[:n].to(dev)
    pos = torch.randint(0, 9000, (n,), generator=g, dtype=torch.int32).to(dev)
    slots[n // 2] = -1  # a padded row
    kc = torch.full((blocks, bs, hkv, d), 3.0, dtype=dtype, device=dev)
    vc = torch.full_like(kc, 5.0)
    out = ops.rope_cache(q, k, v, pos, slots, freqs, kc, vc, interleaved=interleaved, scale=1.125)
    turned = ops.rope(k, pos, freqs, interleaved=interleaved, scale=1.125)
    assert torch.equal(out, ops.rope(q, pos, freqs, interleaved=interleaved, scale=1.125))
    want_k, want_v = torch.full_like(kc, 3.0), torch.full_like(vc, 5.0)
    on = slots >= 0
    want_k.flatten(0, 1)[slots[on]] = turned[on]
    want_v.flatten(0, 1)[slots[on]] = v[on]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    assert lib.device_status(clear=True)[0] == 0
    # in place for Q; a slot past the cache is skipped and recorded
    slots[0] = blocks * bs
    kc2, vc2 = torch.full_like(kc, 3.0), torch.full_like(vc, 5.0)
    ops.rope_cache(q, k, v, pos, slots, freqs, kc2, vc2, interleaved=interleaved, scale=1.125, out=q)
    assert torch.equal(q, out)
    on[0] = False
    want_k.fill_(3.0).flatten(0, 1)[slots[on]] = turned[on]
    assert torch.equal(kc2, want_k)
    assert lib.device_status(clear=True)[0] == 9


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("freqs", ["model", "turning"])
def test_positions_past_32_bits(cuda_device, freqs, interleaved):
    """A frequency's fraction of a turn is off by 2^-64, so an angle by |position| 2^-64 turns and the
    reduced angle's rounding to fp32 (the 1e-7 rad in _close's 6e-7): tight at 2^40, 3e-3 rad at 2^53. In
    both forms of the kernel (a token's heads over several CTAs, and several tokens to a CTA)."""
    from kta_b200 import ops

    dev = cuda_device
    if freqs == "model":
        f, _ = ops.rope_freqs(64, 500000.0, device="cpu")
    else:  # more than a turn to a position, and negative ones
        f = torch.linspace(-40.0, 90.0, 32, dtype=torch.float64)
    far = [2**31 - 1, -2**31, 2**32 + 1, 2**40 + 3, -2**40 - 77, 2**47 + 12345, 2**53 - 1, -2**53]
    for n, h in ((len(far), 32), (5000, 1)):
        pos = (far * n)[:n]
        x = _x((n, h, 64), torch.float16, 11)
        got = ops.rope(x.to(dev), torch.tensor(pos, dtype=torch.int64).to(dev), f.to(dev),
                       interleaved=interleaved).double().cpu().numpy()
        x = x.double().numpy()
        want = paged.rope(x, pos, f.tolist(), interleaved)
        turned = paged.rope(np.abs(x), [0] * n, f.tolist(), interleaved)  # |x|, and its pair's other one
        other = (turned.reshape(n, h, 32, 2)[..., ::-1].reshape(n, h, 64) if interleaved
                 else np.roll(turned, 32, -1))
        angle = 6e-7 + 2 * np.pi * 2.0 ** -64 * np.abs(np.array(pos, dtype=np.float64))[:, None, None]
        fp32 = angle * (turned + other)
        half = torch.finfo(torch.float16).eps / 2
        tiny = torch.finfo(torch.float16).smallest_normal * half
        assert (np.abs(got - want) <= fp32 + half * (np.abs(want) + fp32) + tiny).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (True, True)])
def test_autograd(cuda_device, interleaved, inverse, dtype):
    """The gradient of a loss over the output reaches the input: the formula's (the transpose, in float64),
    for dense, broadcast and strided gradients, through views, and twice."""
    from kta_b200 import ops

    dev = cuda_device
    freqs, _ = ops.rope_freqs(96, device=dev)
    pos = torch.arange(7, 7 + 33, device=dev)
    turn = dict(interleaved=interleaved, inverse=inverse, scale=1.25)

    def want(g):
        return paged.rope(g.double().cpu().numpy(), pos.tolist(), freqs.tolist(), interleaved, not inverse, 1.25)

    fused = _x((33, 5, 128), dtype, 20).to(dev).requires_grad_()
    x = fused[:, 1:4]
    y = ops.rope(x, pos, freqs, **turn)
    assert y.requires_grad and torch.equal(y, ops.rope(x.detach(), pos, freqs, **turn))
    wide = _x((33, 3, 256), dtype, 21).to(dev)
    for g in (wide[..., :128].contiguous(), wide[..., :128], wide[..., 4:132], wide[:, :, ::2],
              wide[:1, :1, :1].expand(33, 3, 128)):
        got, = torch.autograd.grad(y, fused, g, retain_graph=True)
        _close(got[:, 1:4], g.double().cpu().numpy(), want(g), 1.25, 96, interleaved, dtype)
        assert (got[:, 0] == 0).all() and (got[:, 4] == 0).all()
    # linear: the gradient's own gradient, with respect to g, is the output of that direction
    g = wide[..., :128].clone().requires_grad_()
    first, = torch.autograd.grad(y, fused, g, create_graph=True)
    h = _x((33, 5, 128), dtype, 22).to(dev)
    second, = torch.autograd.grad(first, g, h)
    assert torch.equal(second, ops.rope(h[:, 1:4], pos, freqs, **turn))
    # one row for all heads: the heads' gradients are added up by autograd
    one = _x((33, 1, 128), dtype, 23).to(dev).requires_grad_()
    g = wide[:, :, :128].contiguous()
    got, = torch.autograd.grad(ops.rope(one.expand(33, 3, 128), pos, freqs, **turn), one, g)
    each = ops.rope(g, pos, freqs, interleaved=interleaved, inverse=not inverse, scale=1.25)
    assert torch.equal(got, each.sum(1, keepdim=True))
    with torch.no_grad():
        assert not ops.rope(fused, pos, freqs, **turn).requires_grad
        ops.rope(fused, pos, freqs, out=torch.empty_like(fused), **turn)


def test_autograd_on_another_stream_and_captured(cuda_device):
    from kta_b200 import ops

    dev = cuda_device
    freqs, _ = ops.rope_freqs(64, device=dev)
    pos = torch.arange(40, device=dev)
    x = _x((40, 4, 64), torch.bfloat16, 30).to(dev)
    g = _x((40, 4, 64), torch.bfloat16, 31).to(dev)
    want = ops.rope(g, pos, freqs, inverse=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    leaf = x.clone().requires_grad_()
    with torch.cuda.stream(stream):
        for _ in range(2):  # as torch asks for before a capture
            got, = torch.autograd.grad(ops.rope(leaf, pos, freqs), leaf, g)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(ops.rope(leaf, pos, freqs), leaf, g)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
