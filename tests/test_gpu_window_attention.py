"""Attention over a window and the first positions (window.window_attention) against float64.

The reference masks a full score matrix in float64 and forms the gradients from the
formulas; a second test forms them by differences. Bounds count roundings, at half a step
H of the inputs' type (2^-24, 2^-11, 2^-8): a probability is off by H where it is rounded
between the products, by the score's error (D products of size |q||k| summed in fp32, and
the exponential, under 2^-20 of the largest) where it is formed. With a row's values A =
sum_j p_ij |v_j| the output's error is at most (H + E) A and its own rounding, E = 2^-18 (1 +
the largest |score|). Gradients likewise, each product with its absolute values: the bound
takes the formulas with every factor's size in place of the factor.
"""

from __future__ import annotations

import math

import pytest
import torch

from koemi_amd import window as W
from koemi_amd.think import CudaThinkValidationError

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# below a type's range: half of its smallest step
SMALLEST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def seen_by(length, total, window, sinks, valid, device):
    i = torch.arange(total - length, total, device=device)[:, None]
    j = torch.arange(total, device=device)[None]
    see = (j <= i) & ((i - j < window) | (j < sinks))
    if valid is None:
        return see[None]
    return see[None] & valid[:, None, :] & valid[:, total - length:, None]


def clean(t, keep):
    return t.detach().double() if keep is None else torch.where(keep[..., None, None], t.detach().double(), 0.0)


def reference(q, k, v, valid, window, sinks, scale, d_out=None):
    """float64 output, its gradients, and the bounds of each before their own rounding."""

    (batch, length, heads, width), (total, groups) = q.shape, k.shape[1:3]
    shared, half = heads // groups, HALF_STEP[q.dtype]
    kept = None if valid is None else valid[:, total - length:]
    q64 = clean(q, kept).permute(0, 2, 1, 3).contiguous()
    k64, v64 = (clean(t, valid).permute(0, 2, 1, 3).repeat_interleave(shared, dim=1).contiguous() for t in (k, v))
    see = seen_by(length, total, window, sinks, valid, q.device)[:, None]
    s = torch.matmul(q64, k64.transpose(2, 3).contiguous()) * scale
    size = torch.matmul(q64.abs(), k64.abs().transpose(2, 3).contiguous()) * scale
    size = torch.where(see, size, torch.zeros_like(size)).amax(dim=-1, keepdim=True) if total else size.sum(-1, keepdim=True)
    p = torch.softmax(s.masked_fill(~see, float("-inf")), dim=-1)
    p = torch.where(see.any(dim=-1, keepdim=True), p, torch.zeros_like(p))
    rough = 2.0 ** -18 * (1.0 + size)  # of a probability, before it is rounded
    out = torch.matmul(p, v64)
    out_bound = torch.matmul((half + 2 * rough) * p, v64.abs())
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    if d_out is None:
        return back(out), back(out_bound)
    up = clean(d_out, kept).permute(0, 2, 1, 3).contiguous()
    dp = torch.matmul(up, v64.transpose(2, 3).contiguous())
    dp_size = torch.matmul(up.abs(), v64.abs().transpose(2, 3).contiguous())
    delta = (up * out).sum(dim=-1, keepdim=True)
    # D comes from the rounded output
    delta_off = (up.abs() * (half * out.abs() + out_bound + SMALLEST[q.dtype])).sum(dim=-1, keepdim=True)
    ds = p * (dp - delta)
    ds_off = p * ((half + 2 * rough) * (dp - delta).abs() + 2.0 ** -20 * dp_size + delta_off + 2.0 ** -20 * (up * out).abs().sum(dim=-1, keepdim=True))
    if q.dtype == torch.float16:  # what fp16 has no digits for next to a column's largest, held near 2^10 (or lifted by 2^8)
        ds_off = ds_off + torch.where(see, 2.0 ** -33, 0.0) * ds.abs().amax(dim=(-1, -2), keepdim=True)
        p_off = (half + 2 * rough) * p + torch.where(see, 2.0 ** -33, 0.0)
    else:
        p_off = (half + 2 * rough) * p
    gather = lambda t: t.reshape(batch, groups, shared, total, width).sum(dim=2).permute(0, 2, 1, 3)  # noqa: E731
    T = lambda t: t.transpose(2, 3).contiguous()  # noqa: E731
    grads = (back(torch.matmul(ds, k64)) * scale, gather(torch.matmul(T(ds), q64)) * scale, gather(torch.matmul(T(p), up)))
    bounds = (back(torch.matmul(ds_off, k64.abs())) * scale, gather(torch.matmul(T(ds_off), q64.abs())) * scale,
              gather(torch.matmul(T(p_off), up.abs())))
    # fp32 sums of a gradient's terms
    sums = (back(torch.matmul(ds.abs(), k64.abs())) * scale, gather(torch.matmul(T(ds.abs()), q64.abs())) * scale,
            gather(torch.matmul(T(p), up.abs())))
    bounds = tuple(b + 2.0 ** -19 * t for b, t in zip(bounds, sums))
    return (back(out), *grads), (back(out_bound), *bounds)


def close(got, want, bound, what):
    assert torch.isfinite(got).all(), what
    allowed = bound + HALF_STEP[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    off = (got.detach().double() - want).abs()
    worst = (off - allowed).max().item() if off.numel() else 0.0
    assert worst <= 0.0, (what, worst, off.max().item())


def make(shape, dtype, seed, mask, total=None, junk=True):
    batch, length, heads, groups, width = shape
    total = length if total is None else total
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn((batch, length, heads, width), device="cuda", generator=gen).to(dtype)
    k = torch.randn((batch, total, groups, width), device="cuda", generator=gen).to(dtype)
    v = torch.randn((batch, total, groups, width), device="cuda", generator=gen).to(dtype)
    d_out = torch.randn((batch, length, heads, width), device="cuda", generator=gen).to(dtype)
    valid = None
    if mask == "random":
        valid = torch.rand((batch, total), device="cuda", generator=gen) < 0.7
    elif mask == "none":
        valid = torch.zeros((batch, total), dtype=torch.bool, device="cuda")
    elif mask == "tail":
        valid = torch.arange(total, device="cuda")[None] < torch.randint(0, total + 1, (batch, 1), device="cuda", generator=gen)
    elif mask == "head":  # the sinks among the masked ones
        valid = torch.arange(total, device="cuda")[None] >= torch.randint(0, total + 1, (batch, 1), device="cuda", generator=gen)
    if valid is not None and junk:  # what a masked position holds does not matter
        odd = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min], device="cuda", dtype=dtype)
        fill = lambda t, keep: torch.where(keep[..., None, None], t, odd[torch.randint(0, 4, t.shape, device="cuda", generator=gen)])  # noqa: E731
        kept = valid[:, total - length:]
        q, d_out, k, v = fill(q, kept), fill(d_out, kept), fill(k, valid), fill(v, valid)
    return q, k, v, valid, d_out


def check(q, k, v, valid, d_out, window, sinks, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = W.window_attention(*leaves, valid, window=window, sinks=sinks, scale=scale)
    assert out.dtype == q.dtype and out.shape == q.shape
    grads = torch.autograd.grad(out, leaves, d_out)
    want, bounds = reference(q, k, v, valid, window, sinks, scale or 1.0 / math.sqrt(q.shape[-1]), d_out)
    for name, got, w, b in zip(("out", "d_queries", "d_keys", "d_values"), (out, *grads), want, bounds):
        close(got, w, b, name)
    with torch.no_grad():
        again = W.window_attention(q, k, v, valid, window=window, sinks=sinks, scale=scale)
    assert torch.equal(again, out)


SHAPES = [  # batch, length, heads, groups, width, window, sinks, mask
    (1, 1, 1, 1, 8, 1, 0, None),
    (2, 7, 2, 1, 16, 3, 1, "random"),
    (1, 33, 4, 4, 32, 33, 0, None),
    (2, 64, 4, 2, 64, 16, 4, "tail"),
    (1, 129, 8, 1, 64, 40, 4, "random"),
    (2, 200, 6, 2, 80, 100, 3, "tail"),
    (1, 257, 3, 1, 128, 64, 130, None),
    (2, 300, 4, 4, 128, 1, 2, "random"),
    (1, 400, 4, 2, 96, 1000, 5, "head"),
    (1, 150, 5, 5, 100, 31, 1, "tail"),
    (1, 140, 2, 1, 192, 50, 4, None),
    (2, 130, 4, 2, 256, 70, 2, "tail"),
    (1, 70, 2, 1, 251, 30, 3, "random"),
    (3, 90, 7, 1, 33, 20, 200, "none"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch, length, heads, groups, width, window, sinks, mask", SHAPES)
def test_against_float64(device, batch, length, heads, groups, width, window, sinks, mask, dtype):
    args = make((batch, length, heads, groups, width), dtype, 11 + length, mask)
    check(*args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("length, total, window, sinks, mask", [
    (1, 200, 64, 4, None), (5, 3000, 2048, 4, "tail"), (64, 1500, 4000, 0, "random"), (100, 101, 30, 2, None), (17, 600, 100, 150, "tail")])
def test_keys_carried_before_the_queries(device, length, total, window, sinks, mask, dtype):
    args = make((2, length, 4, 2, 64), dtype, length, mask, total=total)
    check(*args, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("length, total, window, sinks, mask", [
    (1, 1, 5, 2, None), (77, 77, 1, 0, None), (130, 160, 1, 0, "random"), (3, 3, 9, 0, "single"), (400, 400, 1, 0, "tail")])
def test_one_visible_key_has_no_gradient_through_its_score(device, length, total, window, sinks, mask, dtype):
    q, k, v, valid, d_out = make((2, length, 4, 2, 48), dtype, 5, None if mask == "single" else mask, total=total)
    if mask == "single":
        valid = torch.arange(total, device=device)[None].expand(2, -1) == 1
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = W.window_attention(*leaves, valid, window=window, sinks=sinks)
    d_q, d_k, d_v = torch.autograd.grad(out, leaves, d_out)
    assert not d_q.any() and not d_k.any()
    check(q, k, v, valid, d_out, window, sinks)
