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


def together(leaves, out, d_out, wanted):
    return torch.autograd.grad(out, [t for t, w in zip(leaves, wanted) if w], d_out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["fused", "heads first", "shared keys", "odd start", "odd columns", "reversed columns", "one row for all"])
def test_any_strides(device, layout, dtype):
    """Views of one projection, transposed and broadcast inputs, starts and strides off 16 bytes: as contiguous copies."""

    gen = torch.Generator(device="cuda").manual_seed(2)
    draw = lambda *shape: torch.randn(shape, device=device, generator=gen).to(dtype)  # noqa: E731
    B, L, H, G, D = 2, 90, 4, 2, 64
    if layout == "fused":
        wide = draw(B, L, (H + 2 * G) * D)
        q, k, v = (t.unflatten(-1, (-1, D)) for t in wide.split([H * D, G * D, G * D], dim=-1))
    elif layout == "heads first":
        q, k, v = draw(B, H, L, D).transpose(1, 2), draw(B, G, L, D).transpose(1, 2), draw(B, G, L, D).transpose(1, 2)
    elif layout == "shared keys":
        q, k, v = draw(B, L, H, D), draw(B, L, 1, D).expand(-1, -1, H, -1), draw(1, L, 1, D).expand(B, -1, H, -1)
    elif layout == "odd start":
        q, k, v = draw(B, L, H, D), draw(B * L * G * D + 1)[1:].view(B, L, G, D), draw(B, L, G, D)
    elif layout == "odd columns":
        q, k, v = draw(B, L, H, D + 3)[..., 1:D + 1], draw(B, L, G, D), draw(B, L, G, D + 1)[..., :D]
    elif layout == "reversed columns":
        q, k, v = draw(B, L, H, D), draw(B, L, D, G).transpose(2, 3), draw(B, L, G, 2 * D)[..., ::2]
    else:
        q, k, v = draw(B, 1, 1, D).expand(-1, L, H, -1), draw(B, L, G, D), draw(1, L, G, D).expand(B, -1, -1, -1)
    d_out = draw(B, 1, 1, D).expand(-1, L, H, -1)
    straight = [t.contiguous().detach().requires_grad_() for t in (q, k, v)]
    want = W.window_attention(*straight, window=20, sinks=2)
    want_grads = torch.autograd.grad(want, straight, d_out.contiguous())
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    got = W.window_attention(*leaves, window=20, sinks=2)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, d_out), want_grads):
        assert torch.equal(a, b)
    check(q.contiguous(), k.contiguous(), v.contiguous(), None, d_out.contiguous(), 20, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("wanted", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_gradients_of_some_inputs(device, wanted):
    q, k, v, valid, d_out = make((2, 100, 4, 2, 64), torch.bfloat16, 9, "tail")
    every = [t.detach().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(W.window_attention(*every, valid, window=30, sinks=3), every, d_out)
    leaves = [t.detach().requires_grad_(w) for t, w in zip((q, k, v), wanted)]
    got = together(leaves, W.window_attention(*leaves, valid, window=30, sinks=3), d_out, wanted)
    for a, b in zip(got, [t for t, w in zip(want, wanted) if w]):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_is_not_finite_reaches_only_those_who_see_it(device, value, dtype):
    """NaN and infinities at valid positions: rows that do not see them, and the gradients of keys that their rows do
    not see, are what they are without them, within the bounds of any order of their sums."""

    window, sinks, length, at = 40, 2, 200, 90
    q, k, v, _, d_out = make((1, length, 4, 2, 64), dtype, 3, None)
    want, bounds = reference(q, k, v, None, window, sinks, 0.125, d_out)

    def unmoved(got, n, rows, name):
        close(got[:, rows], want[n][:, rows], bounds[n][:, rows], (name, n))

    i = torch.arange(length, device=device)
    sees = (i >= at) & (i - at < window)          # queries that see position `at`
    seen = ((i <= at) & (at - i < window)) | (i < sinks)  # keys that the query there sees
    for name in ("keys", "values", "queries", "d_out"):
        t = {"queries": q.clone(), "keys": k.clone(), "values": v.clone(), "d_out": d_out.clone()}
        t[name][0, at, :, 5] = value
        leaves = [t[n].requires_grad_() for n in ("queries", "keys", "values")]
        out = W.window_attention(*leaves, window=window, sinks=sinks)
        grads = torch.autograd.grad(out, leaves, t["d_out"])
        hit = sees if name in ("keys", "values") else (i == at) & (name == "queries")
        unmoved(out, 0, ~hit, name)
        assert not hit.any() or not torch.isfinite(out[0, hit]).all(), name
        rows = sees if name in ("keys", "values") else i == at
        unmoved(grads[0], 1, ~rows, name)
        # keys seen by any row that holds something not finite
        reached = seen if name in ("queries", "d_out") else (i > at - window) & (i < at + window) | (i < sinks)
        unmoved(grads[1], 2, ~reached, name)
        unmoved(grads[2], 3, ~reached, name)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -24, 2.0 ** -16, 1.0, 2.0 ** 10])
def test_half_precision_gradients_of_any_size(device, size):
    """fp16 derivatives far below and above one keep their digits between the products: the gradients are those of d_out =
    1 times size, as far as fp16 holds them."""

    q, k, v, valid, d_out = make((1, 200, 2, 1, 64), torch.float16, 21, "tail")
    d_out = (d_out.float() * size).half()
    check(q, k, v, valid, d_out, 64, 2)


@pytest.mark.gpu
def test_gradients_against_differences(device):
    """Central differences of the float32 output along random directions: with steps h of 2^-6 the cubic term is below 2^-11 of
    the slope's size here (scores move by under 1/2), rounding (2^-20 of the output's sum of sizes, over h) below 2^-12."""

    q, k, v, valid, d_out = make((2, 60, 4, 2, 32), torch.float32, 4, "tail", junk=False)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(W.window_attention(*leaves, valid, window=17, sinks=2), leaves, d_out)
    gen = torch.Generator(device="cuda").manual_seed(8)
    h = 2.0 ** -6
    for n in range(3):
        along = torch.randn(leaves[n].shape, device=device, generator=gen)
        ends = []
        for sign in (1.0, -1.0):
            moved = [t.detach() + (sign * h * along if m == n else 0.0) for m, t in enumerate(leaves)]
            ends.append(W.window_attention(*moved, valid, window=17, sinks=2).double())
        slope = ((ends[0] - ends[1]) * d_out.double()).sum() / (2 * h)
        want = (grads[n].double() * along.double()).sum()
        size = (grads[n].double() * along.double()).norm()
        assert abs(slope - want) <= 2.0 ** -5 * size, (n, slope.item(), want.item(), size.item())


@pytest.mark.gpu
def test_the_same_bits_every_time_and_on_two_streams(device):
    args = [make((2, 700, 8, 2, 64), torch.bfloat16, seed, "tail") for seed in (1, 2)]

    def step(q, k, v, valid, d_out):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = W.window_attention(*leaves, valid, window=100, sinks=4)
        return (out, *torch.autograd.grad(out, leaves, d_out))

    want = [step(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(3):
        got = []
        for a, s in zip(args, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step(*a))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_captured_forward_and_backward(device):
    """A training step in a graph: replays with new inputs, with eager work between them, equal eager steps."""

    q, k, v, valid, d_out = make((2, 300, 4, 2, 64), torch.bfloat16, 1, "tail")
    static = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    up, mask = d_out.clone(), valid.clone()

    def step(leaves, m, d):
        out = W.window_attention(*leaves, m, window=60, sinks=4)
        return (out.detach(), *torch.autograd.grad(out, leaves, d))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, mask, up)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static, mask, up)
    for seed in range(4):
        new = make((2, 300, 4, 2, 64), torch.bfloat16, 30 + seed, "random")
        with torch.no_grad():
            for s, t in zip((*static, mask, up), new):
                s.copy_(t)
        graph.replay()
        leaves = [t.detach().requires_grad_() for t in new[:3]]
        want = step(leaves, new[3], new[4])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), seed


@pytest.mark.gpu
def test_past_2_31_elements(device):
    """A key tensor of more than 2^31 elements: the last queries, whose window and sinks are its ends."""

    total, groups, width, window, sinks, length = 270000, 64, 128, 96, 3, 70
    assert total * groups * width > 1 << 31
    near = window + length
    q, k, v, _, d_out = make((1, length, groups, groups, width), torch.bfloat16, 6, None, total=near + sinks)
    big = [torch.full((1, total, groups, width), float("nan"), device=device, dtype=torch.bfloat16) for _ in range(2)]
    for full, part in zip(big, (k, v)):
        full[:, :sinks], full[:, total - near:] = part[:, :sinks], part[:, sinks:]
    leaves = [t.requires_grad_() for t in (q, *big)]
    out = W.window_attention(*leaves, window=window, sinks=sinks)
    d_q, d_k, d_v = torch.autograd.grad(out, leaves, d_out)
    # in a short call the same pairs are seen: the sinks far behind the window are the first keys
    want, bounds = reference(q, k, v, None, window, sinks, 1.0 / math.sqrt(width), d_out)
    close(out, want[0], bounds[0], "out")
    close(d_q, want[1], bounds[1], "d_queries")
    for got, w, b, name in ((d_k, want[2], bounds[2], "d_keys"), (d_v, want[3], bounds[3], "d_values")):
        close(got[:, :sinks], w[:, :sinks], b[:, :sinks], name)
        close(got[:, total - near:], w[:, sinks:], b[:, sinks:], name)
        assert not got[:, sinks:total - near].any()


@pytest.mark.gpu
@pytest.mark.parametrize("batch, length, total", [(0, 5, 5), (2, 0, 0), (2, 0, 9)])
def test_nothing_to_do(device, batch, length, total):
    q = torch.zeros(batch, length, 4, 32, device=device, requires_grad=True)
    k, v = (torch.zeros(batch, total, 2, 32, device=device, requires_grad=True) for _ in range(2))
    out = W.window_attention(q, k, v, window=3, sinks=1)
    grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert out.shape == q.shape and all(g.shape == t.shape and not g.any() for g, t in zip(grads, (q, k, v)))


@pytest.mark.gpu
def test_windows_and_sinks_past_the_length_and_other_scales(device):
    q, k, v, valid, d_out = make((2, 120, 4, 2, 64), torch.bfloat16, 14, "random")
    whole = W.window_attention(q, k, v, valid, window=120)
    for window, sinks in ((1 << 40, 0), (1, 1 << 40), (7, 120)):
        close(W.window_attention(q, k, v, valid, window=window, sinks=sinks),
              *reference(q, k, v, valid, min(window, 1 << 30), min(sinks, 1 << 30), 0.125), (window, sinks))
    assert torch.equal(W.window_attention(q, k, v, valid, window=1 << 40, scale=0.125), whole)
    check(q, k, v, valid, d_out, 50, 3, scale=1.0)
    check(q, k, v, valid, d_out, 50, 3, scale=2.0 ** -20)


REFUSED = [
    (dict(q=(2, 5, 4)), "shape"), (dict(k=(2, 5, 2, 16)), "same shape"), (dict(q=(2, 6, 4, 8)), "no fewer keys"),
    (dict(k=(2, 5, 3, 8), v=(2, 5, 3, 8)), "divide"), (dict(q=(2, 5, 4, 300), k=(2, 5, 2, 300), v=(2, 5, 2, 300)), "wide"),
    (dict(dtype=torch.float64), "float32, float16 or bfloat16"), (dict(window=0), "window must be a positive integer"),
    (dict(window=True), "window must be a positive integer"), (dict(window=2.0), "window must be a positive integer"),
    (dict(sinks=-1), "sinks must be a non-negative integer"), (dict(scale=0.0), "scale must be"), (dict(scale=True), "scale must be"),
    (dict(scale=float("inf")), "scale must be"), (dict(scale=float("nan")), "scale must be"), (dict(), "must be on CUDA"),
]


@pytest.mark.parametrize("change, message", REFUSED)
def test_refusals(change, message):
    shapes = {"q": (2, 5, 4, 8), "k": (2, 5, 2, 8), "v": (2, 5, 2, 8)} | {n: s for n, s in change.items() if n in "qkv"}
    q, k, v = (torch.zeros(shapes[n], dtype=change.get("dtype", torch.float32)) for n in "qkv")
    numbers = {"window": 4} | {n: x for n, x in change.items() if n in ("window", "sinks", "scale")}
    with pytest.raises(CudaThinkValidationError, match=message):
        W.window_attention(q, k, v, **numbers)


def test_refusals_of_mixed_inputs():
    q, k = torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 2, 8)
    with pytest.raises(CudaThinkValidationError, match="torch.Tensor"):
        W.window_attention(q, k, None, window=3)
    with pytest.raises(CudaThinkValidationError, match="share a dtype"):
        W.window_attention(q, k, k.half(), window=3)


@pytest.mark.gpu
def test_masks_that_are_refused(device):
    q, k = torch.zeros(2, 5, 4, 8, device=device), torch.zeros(2, 6, 2, 8, device=device)
    for mask in (torch.ones(2, 5, dtype=torch.bool, device=device), torch.ones(2, 6, device=device), torch.ones(2, 6, dtype=torch.bool)):
        with pytest.raises(CudaThinkValidationError, match="valid_mask"):
            W.window_attention(q, k, k, mask, window=3)


def test_the_library_refuses_what_its_kernels_cannot_take():
    """Checked on the host, before any launch: addresses and strides off 16 bytes, sizes past the indices."""

    import ctypes

    from koemi_amd import _native

    strides = (ctypes.c_int64 * 9)(*[64 * 4, 64, 16] * 3)

    def call(q=16, stride=strides, batch=1, length=4, total=4, heads=4, groups=4, width=16, window=2, sinks=0, scale=1.0, out=16):
        return lambda: _native.call("koemi_window_attention_forward", q, 16, 16, None, stride, out, None, None, batch, length, total,
                                    heads, groups, width, window, sinks, scale, _native.F32, None, 0, None)

    odd = (ctypes.c_int64 * 9)(*[64 * 4, 64, 17] * 3)
    far = (ctypes.c_int64 * 9)(*[1 << 30, 1 << 23, 16] * 3)
    for bad, message in ((call(q=20), "aligned"), (call(stride=odd), "aligned"), (call(stride=far), "2\\^24 bytes"), (call(width=18), "pieces"),
                         (call(width=320), "256"), (call(heads=3), "divide"), (call(window=0), "window"), (call(scale=-1.0), "scale"),
                         (call(total=3), "no fewer keys"), (call(length=1 << 30, total=1 << 30), "2\\^29"), (call(out=None), "null pointer")):
        with pytest.raises(_native.NativeCallError, match=message):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width, mask", [(32, "random"), (64, "tail"), (64, None), (96, "tail"), (128, None), (160, "random"), (256, "tail")])
def test_many_rows(device, width, mask, dtype):
    """Calls of many rows: probabilities in one plane, 128 keys a workgroup."""

    args = make((160, 130, 4, 1, width), dtype, width, mask)
    check(*args, 40, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_rows(device, dtype):
    """Whole tiles between the window's ends, sinks with many rows past their window."""

    args = make((2, 2300, 16, 4, 64), dtype, 2, "tail")
    check(*args, 700, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width, mask", [(32, "tail"), (64, "random"), (96, None), (128, "tail"), (160, None), (256, "random")])
def test_many_rows_that_see_many_keys(device, width, mask, dtype):
    """More keys than those that keep two planes of probabilities."""

    args = make((160, 130, 4, 1, width), dtype, width + 1, mask)
    check(*args, 100, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window, sinks", [(1, 1), (3, 1), (2, 4), (21, 6)])
def test_few_visible_keys_keep_the_types_precision(device, window, sinks, dtype):
    """Many rows of few keys are off by their own rounding and little more.

    A rounding's error is spread over H = half a step of 1 either way for values from 1 to 2, so a
    result's error is at most H / sqrt(3) of its norm over many elements, were all at their
    binade's start; at 2^-16 of a row's largest size, two planes add less than 1% of H. One
    plane adds an error of about the same size again, and more through D.
    """

    q, k, v, _, d_out = make((64, 128, 16, 4, 32), dtype, 3, None)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = W.window_attention(*leaves, window=window, sinks=sinks)
    grads = torch.autograd.grad(out, leaves, d_out)
    want, _ = reference(q, k, v, None, window, sinks, 1.0 / math.sqrt(32), d_out)
    for name, got, w in zip(("out", "d_queries", "d_keys", "d_values"), (out, *grads), want):
        off = ((got.detach().double() - w).norm() / w.norm()).item()
        assert off <= HALF_STEP[dtype] * (1 / math.sqrt(3) + 0.01), (name, off)
