"""Calls of the trained operators that their documentation allows at its edges: layouts of
one position, candidates next to zero, the largest batches, gates far below zero."""

from __future__ import annotations

import pytest
import torch

import test_gpu_recurrence_training as recurrence_tests
from koemi_amd import recurrent


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width", [1, 33, 50, 256])
@pytest.mark.parametrize("layout", ["turned", "no stride", "one column", "odd stride", "far stride"])
def test_one_position_of_any_row_stride(layout, width, dtype):
    """The row stride of a single position means nothing: each gives a contiguous tensor's bits."""
    batch, columns = 1 if layout == "one column" else 3, 2 * width
    z, _, initial, d_states, d_final = recurrence_tests.draw((batch, 1, width), dtype, width, None)
    flat = z.reshape(batch, columns)
    other = {"turned": lambda: flat[..., None].contiguous().transpose(1, 2),
             "no stride": lambda: torch.as_strided(flat, z.shape, (columns, 0, 1)),
             "one column": lambda: flat.reshape(columns, 1).T[None],
             "odd stride": lambda: torch.as_strided(flat, z.shape, (columns, width + 1, 1)),
             "far stride": lambda: torch.as_strided(flat, z.shape, (columns, (1 << 30) + 3, 1))}[layout]()
    assert other.shape == z.shape and other.is_contiguous() and (width == 1 or other.stride(1) != columns)

    def run(z):
        z, h0 = z.detach().requires_grad_(), initial.clone().requires_grad_()
        out = recurrent.gated_recurrence(z, None, h0)
        return (*out, *torch.autograd.grad(out, (z, h0), (d_states, d_final)))

    for got, want in zip(run(other), run(z)):
        assert torch.equal(got, want)
    recurrence_tests.check(other, None, initial, d_states, d_final)
