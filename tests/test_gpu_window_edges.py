"""Calls of the windowed attention and its cache at the edges of what they take.

Large calls that keep the precision of small ones, against float64 with the bounds of
test_gpu_window_attention.py and of test_gpu_window_cache.py.
"""

from __future__ import annotations

import math

import pytest
import torch

import test_gpu_window_attention as attention
from koemi_amd import window as W


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width, window, sinks", [(32, 100, 3), (64, 60, 4), (64, 61, 4), (64, 100, 0), (128, 90, 2)])
def test_calls_of_many_rows_and_keys_keep_the_types_precision(device, width, window, sinks, dtype, monkeypatch):
    """2^17 rows of heads: off by their own rounding and little more, whatever the call's size and its visible keys.

    Between two products a probability or a derivative is held in two values of its type, so it is off by
    H^2 of itself, H half a step: the elements' bounds are those of ``reference`` with H^2 in H's place, and
    D's too (the output is kept with what it was rounded off by). One value alone would be off by H. Over many
    elements, a rounding's error is spread over H either way for values from 1 to 2: at most H / sqrt(3)
    of the norm; the rest adds less than 1% of H.
    """

    q, k, v, _, d_out = attention.make((64, 128, 16, 4, width), dtype, 7, None)
    half = attention.HALF_STEP[dtype]
    with monkeypatch.context() as patch:
        patch.setitem(attention.HALF_STEP, dtype, half * half)
        want, bounds = attention.reference(q, k, v, None, window, sinks, 1.0 / math.sqrt(width), d_out)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = W.window_attention(*leaves, window=window, sinks=sinks)
    grads = torch.autograd.grad(out, leaves, d_out)
    for name, got, w, b in zip(("out", "d_queries", "d_keys", "d_values"), (out, *grads), want, bounds):
        attention.close(got, w, b, name)
        off = ((got.detach().double() - w).norm() / w.norm()).item()
        assert off <= half * (1 / math.sqrt(3) + 0.01), (name, off)
