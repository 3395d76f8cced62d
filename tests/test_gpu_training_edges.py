"""Calls of the trained operators that their documentation allows at its edges: layouts of
one position, candidates next to zero, the largest batches, gates far below zero."""

from __future__ import annotations

import pytest
import torch

import test_gpu_experts_training as experts_tests
import test_gpu_recurrence_training as recurrence_tests
from koemi_amd import _native, moe, recurrent


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [0.3, 0.1, 1e-2, 1e-3, 1e-4, 1e-5])
def test_candidates_next_to_zero_keep_their_precision(scale, dtype):
    """One position from zero: h = k u, dr = -g u (1 - 2^-7) s (1 - s), dc = g k (1 - u^2), each relative to itself.

    In units of 2^-24 for |r| <= 1: the exponential's argument is rounded (1) and it and the reciprocal are off by 2
    each, so 1 - s and k by at most 10 with their products and s (1 - s) by 16; tanh takes 8 more (c <= 0.3: a product
    of its argument and a polynomial within 3, or 1 - 2^(-2 c log2 e) within 8), products and sums 4: 32 units, 2^-19.
    """
    batch, width = 64, 96
    gen = torch.Generator(device="cuda").manual_seed(17)
    r = torch.rand((batch, 1, width), device="cuda", generator=gen) * 2.0 - 1.0
    c = (torch.rand((batch, 1, width), device="cuda", generator=gen) * 0.9 + 0.1) * scale
    z = torch.cat([r, c * torch.sign(r)], dim=-1).to(dtype).requires_grad_()
    states, final = recurrent.gated_recurrence(z)
    d_final = torch.randn((batch, width), device="cuda", generator=gen)
    (d_z,) = torch.autograd.grad(final, z, d_final)
    z64 = z.detach().double()[:, 0].requires_grad_()
    s, u = torch.sigmoid(z64[:, :width]), torch.tanh(z64[:, width:])
    want = (1.0 - (recurrence_tests.MIN_RETENTION + recurrence_tests.SPAN * s)) * u
    (d_want,) = torch.autograd.grad(want, z64, d_final.double())
    recurrence_tests.close(final, want, 2.0 ** -19 * want.detach().abs(), "final")
    recurrence_tests.close(states[:, 0], want, 2.0 ** -19 * want.detach().abs(), "states")
    recurrence_tests.close(d_z[:, 0], d_want, 2.0 ** -19 * d_want.abs(), "d_z")


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-2, 1e-4, 1e-6])
@pytest.mark.parametrize("length", [40, 4100])
def test_sequences_of_candidates_next_to_zero(length, scale):
    """The bound of the recurrence's own tests without its absolute part: EPS of what the states add up to."""
    z, valid, _, d_states, _ = recurrence_tests.draw((2, length, 70), torch.float32, 23, "random")
    z[..., 70:] *= scale
    z.requires_grad_()
    states, _ = recurrent.gated_recurrence(z, valid)
    want, _, d_want, _, _, d_bound, _ = recurrence_tests.reference(z, valid, None, d_states, None)
    with torch.no_grad():
        z64 = torch.where(valid[..., None], z.detach().double(), 0.0)
        a, b = recurrence_tests.gates(z64, valid)
        none = torch.zeros_like(b[:, 0])
        size = recurrence_tests.scan(a, b.abs(), none)
        bound = 4 * recurrence_tests.EPS * recurrence_tests.scan(a, size, none)
    recurrence_tests.close(states, want, bound, "states")
    (d_z,) = torch.autograd.grad(states, z, d_states)
    recurrence_tests.close(d_z, d_want, d_bound, "d_z")


@pytest.mark.gpu
@pytest.mark.parametrize("width,batch", [(33, (1 << 23) - 8), (65, ((1 << 23) - 8) // 2), (130, ((1 << 23) - 8) // 3)])
def test_the_largest_batches_that_are_accepted(width, batch):
    """Widths just above whole strips, where narrow strips would be more than a launch takes."""
    small, _, initial, d_states, d_final = recurrence_tests.draw((400, 1, width), torch.bfloat16, width, None)
    at = torch.cat([torch.arange(200, device="cuda"), torch.arange(batch - 200, batch, device="cuda")])
    z = torch.zeros((batch, 1, 2 * width), device="cuda", dtype=torch.bfloat16)
    h0, up = torch.zeros((batch, width), device="cuda"), torch.zeros((batch, width), device="cuda")
    z[at], h0[at], up[at] = small, initial, d_final
    z.requires_grad_()
    h0.requires_grad_()
    states, final = recurrent.gated_recurrence(z, None, h0)
    d_z, d_h0 = torch.autograd.grad(final, (z, h0), up)
    want = recurrence_tests.reference(small, None, initial, None, d_final)
    recurrence_tests.close(states[at], want[0], want[4], "states")
    recurrence_tests.close(final[at], want[1], want[4][:, -1], "final")
    recurrence_tests.close(d_z[at], want[2], want[5], "d_z")
    recurrence_tests.close(d_h0[at], want[3], want[6], "d_initial")
    for t in (states, final, d_z, d_h0):
        assert not t[200:-200].any()


FAR = (-3e38, -1e30, -1e4, -200.0, -110.0, -89.0, -60.0, -20.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,width,hidden", [(6, 20, 24), (40, 64, 64), (300, 64, 64)])
def test_gates_far_below_zero_vanish(tokens, width, hidden, dtype):
    """g = b_g alone (W_g = 0), each row of FAR in turn: silu(g) and its slope go to 0, however far below zero g lies.

    The sigmoid of g is within 1.3 |g| + 8 units of 2^-24 of itself, 2^-17 of it down to -87 where it passes 2^-126, and
    may be 0 below: 110 x 2^-126 of silu covers that. Products of K terms in float32 add (K + 64) 2^-24 of their terms'
    sizes twice, and the bf16 tiles' rows between products 2^-8."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)

    def normal(*shape):
        return (torch.randn(shape, device="cuda", generator=gen) * 0.25).to(dtype)

    g = torch.tensor(FAR, device="cuda").repeat(hidden // len(FAR)).to(dtype)
    case = {"context": normal(tokens, width), "assignments": torch.zeros((tokens, 1), device="cuda", dtype=torch.int64),
            "pair_weights": torch.ones((tokens, 1), device="cuda"), "valid": torch.ones(tokens, device="cuda", dtype=torch.bool),
            "gate_weights": torch.zeros((1, hidden, width), device="cuda", dtype=dtype), "gate_biases": g[None],
            "value_weights": normal(1, hidden, width), "value_biases": normal(1, hidden),
            "output_weights": normal(1, width, hidden), "output_biases": torch.zeros((1, width), device="cuda", dtype=dtype)}
    d_out = normal(tokens, width)
    case, leaves, names = experts_tests.leaves_of(case)
    y = experts_tests.call(case)
    grads = dict(zip(names, torch.autograd.grad(y, leaves, d_out)))
    with torch.no_grad():
        plain = experts_tests.call(case)
        x, wv, bv, wo = (case[n].detach().double().squeeze(0) for n in ("context", "value_weights", "value_biases", "output_weights"))
        g, d = g.double(), d_out.double()
        between = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
        s, tiny, units = torch.sigmoid(g), 110 * 2.0 ** -126, 2.0 ** -17 + between + (max(width, hidden, tokens) + 64) * 2.0 ** -23
        silu, slope = g * s, s * (1.0 + g * torch.sigmoid(-g))
        v, v_size = x @ wv.T + bv, x.abs() @ wv.abs().T + bv.abs()
        up, up_size = d @ wo, d.abs() @ wo.abs()

        def like(got, want, size, what):
            experts_tests.close(got, want, size, what)

        h_size = (silu.abs() * units + tiny) * v_size
        like(y, (silu * v) @ wo.T, h_size @ wo.abs().T, "out")
        like(plain, (silu * v) @ wo.T, h_size @ wo.abs().T, "out without gradients")
        like(grads["gate_biases"], (up * v * slope).sum(0), (up_size * v_size * (slope.abs() * units + tiny)).sum(0), "d gate_biases")
        like(grads["value_biases"], (up * silu).sum(0), (up_size * (silu.abs() * units + tiny)).sum(0), "d value_biases")
        like(grads["pair_weights"], (up * silu * v).sum(1), (up_size * h_size).sum(1), "d pair_weights")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [20, 400])
def test_fp16_terms_at_the_worst_rounding(tokens):
    """h = W_o = 1 + 2^-8 in every term: halfway between two bf16 values, so both second planes are 2^-8 and their
    dropped product is 2^-16 of each term, all of one sign. The third plane would add 2^-17 at most, sums of 96 terms
    in float32 (96 + 64) 2^-24; b_o takes most of the sum away, so that the output's own half step shows it."""
    width, hidden = 40, 96
    one = 1.0 + 2.0 ** -8
    half = torch.float16

    def full(value, *shape):
        return torch.full(shape, value, device="cuda", dtype=half)

    b_o = full(-hidden * one * one, 1, width)
    case = {"context": full(1.0, tokens, width), "assignments": torch.zeros((tokens, 1), device="cuda", dtype=torch.int64),
            "pair_weights": torch.ones((tokens, 1), device="cuda"), "valid": torch.ones(tokens, device="cuda", dtype=torch.bool),
            "gate_weights": full(0.0, 1, hidden, width), "gate_biases": full(32.0, 1, hidden),  # silu(32) = 32 in float32
            "value_weights": full(0.0, 1, hidden, width), "value_biases": full(one / 32.0, 1, hidden),
            "output_weights": full(one, 1, width, hidden), "output_biases": b_o}
    want = (hidden * one * one + b_o.double()).expand(tokens, width)
    terms = hidden * one * one
    bound = torch.full_like(want, (2.0 ** -16 + 2.0 ** -17 + (hidden + 64) * 2.0 ** -24) * terms)
    with torch.no_grad():
        experts_tests.close(experts_tests.call(case), want, bound, "out")
    trained, _, _ = experts_tests.leaves_of(case)
    experts_tests.close(experts_tests.call(trained), want, bound, "out with what the gradients need")


def test_routes_of_2_32_choices_are_refused():
    """Their counts would pass 32 bits."""
    for name, pointers in (("koemi_moe_route_balanced_forward", 7), ("koemi_moe_route_balanced_backward", 8)):
        tail = (None, 0, None) if name.endswith("forward") else (None,)
        with pytest.raises(_native.NativeCallError, match="2\\^32"):
            _native.call(name, None, _native.dtype_code(torch.bfloat16), 2, *([None] * pointers), 1 << 31, 2, 2, *tail)


@pytest.mark.gpu
def test_routes_of_2_32_choices_are_refused_by_the_front():
    logits = torch.zeros((1, 2), device="cuda", dtype=torch.bfloat16).expand(1 << 31, 2)
    valid = torch.ones(1, device="cuda", dtype=torch.bool).expand(1 << 31)
    with pytest.raises(moe.CudaMoeValidationError, match="2\\^32"):
        moe.route_topk_balanced(logits, valid, top_k=2)


@pytest.mark.gpu
@pytest.mark.parametrize("validate", [False, True])
def test_experts_of_more_tiles_than_a_launch_takes_are_refused_at_once(validate):
    def t(*shape, dtype=torch.float16):
        return torch.zeros(shape, device="cuda", dtype=dtype)

    tokens, width, hidden = 1 << 24, 512, 8192
    matrix = t(4, hidden, width)
    args = [t(1, width).expand(tokens, width), torch.arange(2, device="cuda").expand(tokens, 2), None,
            t(1, dtype=torch.bool).expand(tokens), matrix, t(4, hidden), matrix, t(4, hidden), matrix.transpose(1, 2), t(4, width)]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(moe.CudaMoeValidationError, match="2\\^24"):
        moe.expert_mixture(*args, validate=validate)
    assert torch.cuda.max_memory_allocated() == before


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [5, 10, 11, 17, 26, 31, 33, 62])
def test_mass_of_equal_probabilities(experts):
    """p = 1 / E in every token, one token for each lane group of a workgroup: p is off by one unit of 2^-24 with its
    reciprocal, the eight sums of k equal values by (k + 1) / 2 (step i rounds i p of k p), and joining equal sums is
    exact. k = 1 / 8 of the 128 groups of two lanes, 64 of four and 32 of eight."""
    tokens = 256 // (2 if experts <= 8 else 4 if experts <= 16 else 8)
    logits, valid = torch.zeros((tokens, experts), device="cuda"), torch.ones(tokens, device="cuda", dtype=torch.bool)
    _, _, statistics = moe.route_topk_balanced(logits, valid, top_k=1)
    off = (statistics.probability_mass.double() * experts / tokens - 1.0).abs().max().item()
    assert off <= ((tokens / 8 + 1) / 2 + 2) * 2.0 ** -24, off * 2.0 ** 24
