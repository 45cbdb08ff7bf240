"""Tensors that the binding (csrc/binding.cpp) cannot take are errors, never the end of the process."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_tensors_without_memory_are_refused(cuda_device):
    """A sparse block table of one column passes every check of sizes, and a tracer's tensors pass all; only
    their pointers are missing."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from kta_b200 import ops

    dev = cuda_device
    one = torch.ones(1, dtype=torch.int32, device=dev)
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    with pytest.raises((RuntimeError, ValueError)):
        ops.cache_slots(one, one, table.to_sparse(), one, 16, 1)
    x = torch.ones((2, 1, 64), dtype=torch.float16, device=dev)
    freqs, _ = ops.rope_freqs(64, device=dev)
    pos = torch.arange(2, device=dev)
    with FakeTensorMode() as mode, pytest.raises((RuntimeError, ValueError)):
        ops.rope(*(mode.from_tensor(t) for t in (x, pos, freqs)))
    got = ops.cache_slots(one, one, table, one, 16, 1)  # and the binding goes on
    assert [t.tolist() for t in got] == [[1], [1], [0, 1], [0]]
    assert torch.equal(ops.rope(x, pos * 0, freqs), x)


def test_what_is_written_in_place_counts_as_changed(cuda_device):
    """Autograd keeps inputs for its backward pass and looks at their version: a tensor that a call wrote
    since is an error there, never a wrong gradient. Tensors of inference mode have no version."""
    from kta_b200 import ops

    dev = cuda_device
    one = torch.ones(1, dtype=torch.int32, device=dev)
    freqs, _ = ops.rope_freqs(64, device=dev)
    pos = torch.zeros(1, dtype=torch.int32, device=dev)
    slots = torch.zeros(1, dtype=torch.int64, device=dev)

    def made():
        t = {n: torch.ones((1, h, 64), dtype=torch.float16, device=dev) for n, h in (("x", 2), ("kv", 1), ("o", 2))}
        t.update({n: torch.ones((1, 16, 1, 64), dtype=torch.float16, device=dev) for n in ("kc", "vc")})
        t.update(lse=torch.ones((1, 2), device=dev), table=torch.zeros((1, 1), dtype=torch.int32, device=dev),
                 at=torch.zeros(1, dtype=torch.int32, device=dev))
        return t

    calls = {
        "x": lambda t: ops.rope(t["x"], pos, freqs, out=t["x"]),
        "at": lambda t: ops.cache_slots(one, one, t["table"], one, 16, 1, positions=t["at"]),
        "table": lambda t: ops.cache_slots(one, one, t["table"], one, 16, 1),
        "kc": lambda t: ops.rope_cache(t["x"], t["kv"], t["kv"], pos, slots, freqs, t["kc"], t["vc"]),
        "vc": lambda t: ops.rope_cache(t["x"], t["kv"], t["kv"], pos, slots, freqs, t["kc"], t["vc"]),
        "o": lambda t: ops.rope_cache(t["x"], t["kv"], t["kv"], pos, slots, freqs, t["kc"], t["vc"], out=t["o"]),
        "lse": lambda t: ops.tree_attn(t["x"], t["kc"], t["vc"], t["table"], pos, torch.cat([pos, one]), 1,
                                       out=t["o"], lse=t["lse"]),
    }
    for name, call in calls.items():
        t = made()
        before = {n: v._version for n, v in t.items()}
        w = torch.ones((), device=dev, requires_grad=True)
        y = w * t[name]  # its backward pass needs t[name]
        call(t)
        assert t[name]._version > before[name], name
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.float().sum().backward()
        with torch.inference_mode():
            t = made()
        call(t)
    t = made()
    before = {n: v._version for n, v in t.items()}
    calls["o"](t)
    calls["lse"](t)
    assert t["x"]._version == before["x"] and t["kv"]._version == before["kv"]  # only read
