"""CPU: which tensors the ops copy before the kernels read them with 16-byte
vectors."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_vectors_cannot_read_are_copied(dtype):
    from asrback_amd.attention import _aligned

    per = 16 // torch.empty((), dtype=dtype).element_size()
    buffer = torch.arange(4096, dtype=torch.float32).to(dtype)
    assert buffer.data_ptr() % 16 == 0
    for t in (
        buffer[:257].view(1, 257)[:, :256],             # one row of odd stride: contiguous to torch
        buffer[3:259].view(1, 256),                     # contiguous, at an odd offset
        buffer[1:513].view(2, 1, 4, 64),
        buffer[:4 * 65].view(4, 65)[:, :64],
        buffer[:512].view(8, 64).t(),
        buffer[:130].view(1, 2, 65)[:, :1, :64],
    ):
        copy = _aligned(t)
        assert copy.data_ptr() != t.data_ptr() and torch.equal(copy, t)
        assert copy.data_ptr() % 16 == 0 and copy.stride(-1) == 1
        assert all(stride % per == 0 for stride in copy.stride()[:-1])
    for t in (buffer[:512].view(2, 256), buffer[:512].view(2, 256)[:, per:per + 64], buffer[per:per + 64].view(1, 64)):
        assert _aligned(t) is t
