"""The trained route (moe.route_topk_balanced) against float64.

Bounds count roundings of 2^-24: a probability's exponent is z - max (rounded once:
|z - max| units of its size), the exponential, a sum of at most 1024 terms in lanes of
16 and a tree, and a division; a mass adds tokens in a chain of at most 1024 links.
Choices and counts are equal.
"""

from __future__ import annotations

import pytest
import torch

from koemi_amd import moe

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def reference(logits, valid, top_k, d_weights, d_mass, d_loss):
    experts = logits.shape[-1]
    z = logits.detach().double().reshape(-1, experts)
    ok = valid.reshape(-1) & (z > float("-inf")).any(dim=-1)
    z = torch.where(ok[:, None], z, torch.zeros_like(z)).requires_grad_()
    p = torch.softmax(z, dim=-1) * ok[:, None]
    rank = torch.sort(z.detach(), dim=-1, descending=True, stable=True)[1][:, :top_k]
    chosen = ok[:, None] & (z.detach().gather(1, rank) > float("-inf"))
    assignments = rank.masked_fill(~chosen, -1)
    weights = p.gather(1, rank) * chosen
    mass = p.sum(dim=0)
    counts = torch.bincount(rank[chosen], minlength=experts).double()
    n = ok.sum().double()
    loss = experts * (mass / n.clamp(min=1) * counts / counts.sum().clamp(min=1)).sum()
    total = 0.0
    if d_weights is not None:
        total = total + (weights * d_weights.double().reshape(weights.shape)).sum()
    if d_mass is not None:
        total = total + (mass * d_mass.double()).sum()
    if d_loss is not None:
        total = total + loss * d_loss.double()
    (d_z,) = torch.autograd.grad(total, z)
    with torch.no_grad():
        x = (z - z.amax(dim=-1, keepdim=True)).abs().clamp(max=150.0)
        p_bound = U * (40 + x) * p
        g = torch.zeros_like(p)
        if d_mass is not None:
            g += d_mass.double().abs()
        if d_loss is not None:
            g += d_loss.double().abs() * experts * counts / (n.clamp(min=1) * counts.sum().clamp(min=1))
        if d_weights is not None:
            g.scatter_add_(1, rank, d_weights.double().reshape(weights.shape).abs() * chosen)
        size = (p * g).sum(dim=-1, keepdim=True)
        spread = (p_bound * g).sum(dim=-1, keepdim=True)
        d_bound = p_bound * (g + size) + p * (spread + 16 * U * (g + size))
        mass_bound = p_bound.sum(dim=0) + 1024 * U * mass
        loss_bound = experts * (mass_bound / n.clamp(min=1) * counts / counts.sum().clamp(min=1)).sum() + 32 * U * loss
    return dict(assignments=assignments, weights=weights.detach(), mass=mass.detach(), counts=counts, n=n, loss=loss.detach(),
                d_z=torch.where(ok[:, None], d_z, torch.zeros_like(d_z)), w_bound=p_bound.gather(1, rank),
                mass_bound=mass_bound, loss_bound=loss_bound, d_bound=d_bound)


def close(got, want, bound, what):
    allowed = bound + HALF_STEP[got.dtype] * want.abs() + SMALLEST[got.dtype]
    off = (got.detach().double().reshape(want.shape) - want).abs()
    assert (off <= allowed).all(), (what, (off - allowed).max().item(), off.max().item())


def check(logits, valid, top_k, d_weights, d_mass, d_loss):
    logits = logits.detach().requires_grad_()
    assignments, weights, statistics = moe.route_topk_balanced(logits, valid, top_k=top_k)
    outs = [(o, d) for o, d in ((weights, d_weights), (statistics.probability_mass, d_mass),
                                (statistics.balance_loss, d_loss)) if d is not None]
    (d_logits,) = torch.autograd.grad([o for o, _ in outs], logits, [d for _, d in outs])
    want = reference(logits, valid, top_k, d_weights, d_mass, d_loss)
    assert assignments.shape == weights.shape == (*logits.shape[:-1], top_k) and assignments.dtype == torch.int64
    assert torch.equal(assignments.reshape(-1, top_k), want["assignments"])
    assert torch.equal(statistics.assignment_counts.double(), want["counts"])
    assert statistics.valid_count.item() == want["n"].item()
    close(weights, want["weights"], want["w_bound"], "weights")
    close(statistics.probability_mass, want["mass"], want["mass_bound"], "mass")
    close(statistics.balance_loss, want["loss"], want["loss_bound"], "loss")
    assert d_logits.shape == logits.shape and d_logits.dtype == logits.dtype
    close(d_logits, want["d_z"], want["d_bound"], "d_logits")


def draw(tokens, experts, top_k, dtype, seed, masked=False, scale=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn((tokens, experts), device="cuda", generator=gen) * scale).to(dtype)
    valid = torch.rand(tokens, device="cuda", generator=gen) < 0.8
    if masked:
        logits = logits.masked_fill(torch.rand((tokens, experts), device="cuda", generator=gen) < 0.5, float("-inf"))
    junk = torch.tensor([float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min], device="cuda", dtype=dtype)
    fill = junk[torch.randint(0, 4, logits.shape, device="cuda", generator=gen)]
    logits = torch.where(valid[:, None], logits, fill)  # what an invalid token holds does not matter
    return (logits, valid, top_k, torch.randn((tokens, top_k), device="cuda", generator=gen),
            torch.randn(experts, device="cuda", generator=gen), torch.tensor(3.0 * tokens, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("tokens,experts,top_k", [
    (1, 1, 1), (3, 2, 2), (70, 3, 1), (1, 16, 2), (300, 16, 16), (1000, 16, 2), (77, 20, 5), (129, 37, 3), (500, 64, 8),
    (65, 100, 7), (40, 128, 40), (33, 256, 4), (30, 257, 9), (21, 500, 2), (17, 512, 70), (9, 777, 3), (12, 1024, 130),
    (70000, 8, 2)])
def test_route_and_gradient(tokens, experts, top_k, dtype, masked):
    check(*draw(tokens, experts, top_k, dtype, tokens + experts, masked))


@pytest.mark.gpu
def test_shapes_strides_and_single_gradients():
    logits, valid, top_k, d_w, d_m, d_l = draw(120, 24, 3, torch.bfloat16, 4)
    shaped = logits.reshape(4, 30, 24)
    check(shaped, valid.reshape(4, 30), top_k, d_w.reshape(4, 30, 3), d_m, d_l)
    check(logits[5], valid[5], top_k, d_w[5], d_m, d_l)
    wide = torch.full((120, 31), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:, 3:27] = logits  # unaligned rows of a wider matrix
    check(wide[:, 3:27], valid, top_k, d_w, d_m, d_l)
    check(logits.t().contiguous().t(), valid, top_k, d_w, d_m, d_l)
    check(shaped.transpose(0, 1), valid.reshape(4, 30).t(), top_k, d_w.reshape(30, 4, 3), d_m, d_l)
    check(logits[:1].expand(120, 24), valid[:1].expand(120), top_k, d_w, d_m, d_l)
    for upstream in ((d_w, None, None), (None, d_m, None), (None, None, d_l)):
        check(logits, valid, top_k, *upstream)


@pytest.mark.gpu
def test_nothing_routed():
    for logits, valid in ((torch.randn(50, 6, device="cuda"), torch.zeros(50, dtype=torch.bool, device="cuda")),
                          (torch.full((50, 6), float("-inf"), device="cuda"), torch.ones(50, dtype=torch.bool, device="cuda")),
                          (torch.randn(0, 6, device="cuda"), torch.zeros(0, dtype=torch.bool, device="cuda"))):
        logits.requires_grad_()
        assignments, weights, statistics = moe.route_topk_balanced(logits, valid, top_k=2)
        assert (assignments == -1).all() and (weights == 0).all() and statistics.balance_loss.item() == 0.0
        assert (statistics.probability_mass == 0).all() and (statistics.assignment_counts == 0).all()
        (d,) = torch.autograd.grad(weights.sum() + statistics.balance_loss, logits)
        assert d.shape == logits.shape and (d == 0).all()


@pytest.mark.gpu
def test_ties_zeros_and_extremes():
    valid = torch.ones(4, dtype=torch.bool, device="cuda")
    low = torch.finfo(torch.float32).min
    logits = torch.tensor([[-0.0, 0.0, -0.0, 0.0, 0.0], [1e30, -1e30, 1e30, low, 0.0], [low, low, low, low, low],
                           [low, float("-inf"), 5.0, low, -200.0]], device="cuda")
    assignments, weights, _ = moe.route_topk_balanced(logits, valid, top_k=4)
    assert assignments.tolist() == [[0, 1, 2, 3], [0, 2, 4, 1], [0, 1, 2, 3], [2, 4, 0, 3]]
    want = torch.softmax(logits.double(), dim=-1).gather(1, assignments)
    assert ((weights.double() - want).abs() <= 40 * U * want + 2.0 ** -126).all()
    nan = logits.clone()
    nan[1, 3] = float("nan")
    nan[2, 0] = float("inf")
    assignments, weights, statistics = moe.route_topk_balanced(nan, valid, top_k=2)
    assert ((assignments >= 0) & (assignments < 5)).all()
    assert weights[1].isnan().all() and weights[2].isnan().all() and weights[0].isfinite().all() and weights[3].isfinite().all()
    assert statistics.balance_loss.isnan()


@pytest.mark.gpu
def test_finite_choices_equal_the_learned_route():
    logits, valid, *_ = draw(4000, 16, 2, torch.float32, 8)
    valid[:] = True
    logits = torch.nan_to_num(logits, nan=0.5, posinf=2.0, neginf=-2.0).clamp(-30, 30)
    a0, w0, s0 = moe.route_topk_learned(logits, valid, top_k=2, return_statistics=True)
    a1, w1, s1 = moe.route_topk_balanced(logits, valid, top_k=2)
    # the learned route picks by probability, this one by logit: they differ only where probabilities round to a tie
    same = (a0 == a1).all(dim=-1)
    assert same.float().mean().item() > 0.999
    assert ((w0 - w1).abs() <= 100 * U * w0).all()
    assert ((s0.probability_mass - s1.probability_mass).abs() <= 2048 * U * s0.probability_mass).all()


@pytest.mark.gpu
def test_merged_statistics_carry_the_gradient():
    parts = [draw(tokens, 12, 2, torch.float32, tokens)[:2] for tokens in (90, 40)]
    leaves = [z.requires_grad_() for z, _ in parts]
    statistics = moe.merge_router_statistics([moe.route_topk_balanced(z, v, top_k=2)[2] for z, (_, v) in zip(leaves, parts)])
    loss = statistics.balance_loss
    got = torch.autograd.grad(loss, leaves, torch.tensor(50.0, device="cuda"))
    both, ok = torch.cat([z.detach() for z in leaves]), torch.cat([v for _, v in parts])
    want = reference(both, ok, 2, None, None, torch.tensor(50.0, device="cuda"))
    close(loss, want["loss"], want["loss_bound"], "loss")
    close(torch.cat(got), want["d_z"], want["d_bound"], "d_logits")
    with torch.no_grad():
        assert not statistics.balance_loss.requires_grad
        close(statistics.balance_loss, want["loss"], want["loss_bound"], "loss")


@pytest.mark.gpu
def test_gradient_against_differences():
    # a central difference of step 2^-7 over logits of order one: its third-order term is near 2^-14 of the slope's
    # terms, the outputs' roundings 2^-24 / 2^-7
    gen = torch.Generator(device="cuda").manual_seed(0)
    rows = torch.stack([torch.randperm(6, device="cuda", generator=gen) for _ in range(30)]).float() / 2  # no near ties
    logits = rows.requires_grad_()
    valid = torch.ones(30, dtype=torch.bool, device="cuda")
    d_w = torch.randn((30, 2), device="cuda", generator=gen)

    def value(z):
        _, w, s = moe.route_topk_balanced(z, valid, top_k=2)
        return (w.double() * d_w.double()).sum() + 30.0 * s.balance_loss.double()

    (d,) = torch.autograd.grad(value(logits), logits)
    for _ in range(4):
        v = torch.randn(logits.shape, device="cuda", generator=gen).clamp(-2, 2)
        with torch.no_grad():
            slope = (value(logits + 2.0 ** -7 * v) - value(logits - 2.0 ** -7 * v)) * 2.0 ** 6
        want = (d.double() * v.double()).sum()
        assert abs(slope.item() - want.item()) < 5e-3 * (1 + abs(want.item()))


@pytest.mark.gpu
def test_captured_and_replayed():
    logits, valid, top_k, d_w, d_m, d_l = draw(3000, 16, 2, torch.bfloat16, 1)
    logits = logits.requires_grad_()

    def step():
        a, w, s = moe.route_topk_balanced(logits, valid, top_k=top_k)
        loss = s.balance_loss
        (d,) = torch.autograd.grad((w, s.probability_mass, loss), logits, (d_w, d_m, d_l))
        return [t.detach() for t in (a, w, s.probability_mass, s.assignment_counts, s.valid_count, loss, d)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (2, 3, 4):
        new = draw(3000, 16, 2, torch.bfloat16, seed)
        with torch.no_grad():
            logits.copy_(new[0])
            valid.copy_(new[1])
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in held]
        for got, want in zip(kept, step()):
            assert torch.equal(got, want)


def test_refusals_on_the_cpu():
    z, valid = torch.zeros(4, 8), torch.ones(4, dtype=torch.bool)
    with pytest.raises(moe.CudaMoeValidationError, match="CUDA tensor"):
        moe.route_topk_balanced(z, valid, top_k=2)
    with pytest.raises(TypeError):
        moe.route_topk_balanced(None, valid, top_k=2)


@pytest.mark.gpu
def test_refusals():
    z, valid = torch.zeros(4, 8, device="cuda"), torch.ones(4, dtype=torch.bool, device="cuda")
    for logits, mask, k in ((z.double(), valid, 2), (z, valid[:3], 2), (z, valid.int(), 2), (z, valid, 0), (z, valid, 9),
                            (z, valid, True), (z, valid.cpu(), 2), (z[:, :0], valid, 1),
                            (torch.zeros(2, 1025, device="cuda"), valid[:2], 1)):
        with pytest.raises(moe.CudaMoeValidationError):
            moe.route_topk_balanced(logits, mask, top_k=k)
