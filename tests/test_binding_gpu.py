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
