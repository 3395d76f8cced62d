"""The trained experts (moe.expert_mixture) against float64.

Every product's bound is the sum of its terms' sizes times U (K + 64) for a sum of K
terms in float32 (U = 2^-24; 64 covers the few roundings around it), and a bound made in
one product is carried through the next ones by the sizes of what multiplies it.
|silu'| <= 1.1 and |silu''| <= 0.5. Where the bf16 tiles run (width and hidden multiples
of 64), what lies between two products is bf16: R = 2^-8 of h, dg, dv and w h. Outputs add
half a step of their type.
"""

from __future__ import annotations

import pytest
import torch

from koemi_amd import _native, moe

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
NAMES = ("context", "pair_weights", "gate_weights", "gate_biases", "value_weights", "value_biases", "output_weights",
         "output_biases")


def reference(case, d_out):
    """float64 outputs and bounds: {name: (value, bound)}."""

    x, assignments, w, valid = case["context"], case["assignments"], case["pair_weights"], case["valid"]
    width, top_k = x.shape[-1], assignments.shape[-1]
    flat, ids, ok = x.detach().double().reshape(-1, width), assignments.reshape(-1, top_k).long(), valid.reshape(-1)
    experts, hidden, _ = case["gate_weights"].shape
    R = 0.0 if x.dtype == torch.float32 else \
        2.0 ** -8 if x.dtype == torch.bfloat16 and width % 64 == 0 and hidden % 64 == 0 else 2.0 ** -17
    w64 = w.detach().double().reshape(-1, top_k) if w is not None else torch.full(ids.shape, 1.0 / top_k, device=x.device).double()
    d = d_out.double().reshape(-1, width)
    zeros = torch.zeros_like
    out = {"out": zeros(flat), "context": zeros(flat), "pair_weights": zeros(w64)}
    out |= {n: zeros(case[n].detach().double()) for n in NAMES[2:]}
    bound = {n: t.clone() for n, t in out.items()}
    rows = torch.where(ok[:, None], flat, torch.zeros_like(flat))  # an invalid token's values do not matter
    ups = torch.where(ok[:, None], d, torch.zeros_like(d))
    for e in range(experts):
        t, s = ((ids == e) & ok[:, None]).nonzero(as_tuple=True)
        n = t.numel()
        if n == 0:
            continue
        wg, bg, wv, bv, wo, bo = (case[name][e].detach().double() for name in NAMES[2:])
        xe, de, we = rows[t], ups[t], w64[t, s][:, None]
        g, v = xe @ wg.T + bg, xe @ wv.T + bv
        g_b = U * (width + 64) * (xe.abs() @ wg.abs().T + bg.abs())
        v_b = U * (width + 64) * (xe.abs() @ wv.abs().T + bv.abs())
        sig = torch.sigmoid(g)
        silu, slope = g * sig, sig * (1 + g * (1 - sig))
        h = silu * v
        h_b = 1.1 * v.abs() * g_b + silu.abs() * v_b + 16 * U * h.abs()
        hr_b = h_b + R * (h.abs() + h_b)
        y = h @ wo.T + bo
        y_b = hr_b @ wo.abs().T + U * (hidden + 64) * (h.abs() @ wo.abs().T + bo.abs())
        out["out"].index_add_(0, t, we * y)
        bound["out"].index_add_(0, t, we.abs() * (y_b + (top_k + 4) * U * y.abs()))
        dh = de @ wo
        dh_b = U * (width + 64) * (de.abs() @ wo.abs())
        out["pair_weights"][t, s] = (dh * h).sum(1) + (de * bo).sum(1)
        bound["pair_weights"][t, s] = ((dh_b * h.abs() + dh.abs() * h_b).sum(1) + U * (hidden + 64) * (dh * h).abs().sum(1)
                                       + U * (width + 64) * (de * bo).abs().sum(1))
        dg, dv, wh = we * dh * v * slope, we * dh * silu, we * h
        wa = we.abs()
        size = (wa * dh.abs() * v.abs()) * 1.1
        dg_b = wa * (1.1 * dh_b * v.abs() + 1.1 * dh.abs() * v_b + 0.5 * dh.abs() * v.abs() * g_b) + 16 * U * size
        dv_b = wa * (dh_b * silu.abs() + 1.1 * dh.abs() * g_b) + 16 * U * dv.abs()
        wh_b = wa * h_b + 4 * U * wh.abs()
        dg_b, dv_b, wh_b = dg_b + R * (dg.abs() + dg_b), dv_b + R * (dv.abs() + dv_b), wh_b + R * (wh.abs() + wh_b)
        out["context"].index_add_(0, t, dg @ wg + dv @ wv)
        dx_size = dg.abs() @ wg.abs() + dv.abs() @ wv.abs()
        bound["context"].index_add_(0, t, dg_b @ wg.abs() + dv_b @ wv.abs() + U * (2 * hidden + 64 + top_k) * dx_size)
        for name, a, a_b, b in (("gate_weights", dg, dg_b, xe), ("value_weights", dv, dv_b, xe)):
            out[name][e] = a.T @ b
            bound[name][e] = a_b.T @ b.abs() + U * (n + 64) * (a.abs().T @ b.abs())
        out["output_weights"][e] = de.T @ wh
        bound["output_weights"][e] = de.abs().T @ wh_b + U * (n + 64) * (de.abs().T @ wh.abs())
        for name, a, a_b in (("gate_biases", dg, dg_b), ("value_biases", dv, dv_b), ("output_biases", we * de, 0 * de)):
            out[name][e] = a.sum(0)
            bound[name][e] = (a_b + U * (n + 64) * a.abs()).sum(0)
    return {n: (out[n], bound[n]) for n in out}


def close(got, want, bound, what):
    want, bound = want.reshape(got.shape), bound.reshape(got.shape)
    allowed = bound + HALF_STEP[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    off = (got.detach().double() - want).abs()
    assert (off <= allowed).all(), (what, (off - allowed).max().item(), off.max().item(), want.abs().max().item())


def draw(tokens, width, hidden, experts, top_k, dtype, seed, skew=False, weighted=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, device="cuda", generator=gen) * scale

    logits = normal(tokens, experts) + (torch.arange(experts, device="cuda") == 0) * (100.0 if skew else 0.0)
    weights, assignments = torch.softmax(logits, dim=-1).topk(top_k, dim=-1)
    valid = torch.rand(tokens, device="cuda", generator=gen) < 0.85
    hole = torch.rand((tokens, top_k), device="cuda", generator=gen) < 0.1
    assignments = assignments.masked_fill(hole, -1)
    x = normal(tokens, width).to(dtype)
    x = torch.where(valid[:, None], x, torch.full_like(x, float("nan")))  # an invalid token's values do not matter
    case = {"context": x, "assignments": assignments, "pair_weights": weights if weighted else None, "valid": valid,
            "gate_weights": normal(experts, hidden, width, scale=width ** -0.5), "gate_biases": normal(experts, hidden, scale=0.2),
            "value_weights": normal(experts, hidden, width, scale=width ** -0.5), "value_biases": normal(experts, hidden, scale=0.2),
            "output_weights": normal(experts, width, hidden, scale=hidden ** -0.5), "output_biases": normal(experts, width, scale=0.2)}
    for name in NAMES[2:]:
        case[name] = case[name].to(dtype)
    d_out = normal(tokens, width).to(dtype)
    return case, torch.where(valid[:, None], d_out, torch.full_like(d_out, float("inf")))


def call(case, **more):
    return moe.expert_mixture(case["context"], case["assignments"], case["pair_weights"], case["valid"],
                              *(case[n] for n in NAMES[2:]), **more)


def leaves_of(case):
    case = dict(case)
    for name in NAMES:
        if case[name] is not None:
            case[name] = case[name].detach().requires_grad_()
    return case, [case[n] for n in NAMES if case[n] is not None], [n for n in NAMES if case[n] is not None]


def check(case, d_out):
    case, leaves, names = leaves_of(case)
    y = call(case)
    grads = dict(zip(names, torch.autograd.grad(y, leaves, d_out)))
    want = reference(case, d_out)
    assert y.shape == case["context"].shape and y.dtype == case["context"].dtype
    close(y, *want["out"], "out")
    for name, got in grads.items():
        assert got.shape == case[name].shape and got.dtype == case[name].dtype
        close(got, *want[name], name)
    with torch.no_grad():
        close(call(case), *want["out"], "out without gradients")


SHAPES = [(1, 1, 1, 1, 1), (1, 64, 64, 2, 2), (3, 5, 7, 3, 2), (64, 64, 128, 4, 2), (200, 64, 192, 4, 2), (130, 128, 64, 3, 1),
          (300, 96, 40, 5, 3), (257, 130, 259, 2, 2), (500, 64, 64, 40, 2), (1000, 256, 320, 3, 2), (700, 192, 64, 1, 1),
          (33, 72, 72, 9, 9), (1500, 320, 576, 2, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_outputs_and_gradients(shape, dtype):
    check(*draw(*shape, dtype, sum(shape)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(9, 8, 16, 3, 2), (150, 200, 136, 2, 2), (600, 72, 328, 2, 2)])
def test_rows_of_whole_octets_and_weights_behind_an_offset(shape, dtype):
    """Weights read eight values at a time, and from an address that does not allow it."""
    case, d_out = draw(*shape, dtype, sum(shape))
    check(case, d_out)
    moved = dict(case)
    for name in ("gate_weights", "value_weights", "output_weights"):
        flat = torch.empty(case[name].numel() + 1, device="cuda", dtype=dtype)
        moved[name] = flat[1:].view(case[name].shape).copy_(case[name])
    check(moved, d_out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,hidden", [(64, 128), (50, 90)])
def test_one_expert_takes_all_and_equal_shares(width, hidden, dtype):
    check(*draw(700, width, hidden, 6, 1, dtype, 5, skew=True))  # five experts without pairs
    check(*draw(300, width, hidden, 6, 3, dtype, 6, weighted=False))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,hidden", [(64, 128), (50, 90)])
def test_nothing_routed_and_no_tokens(width, hidden, dtype):
    case, d_out = draw(20, width, hidden, 4, 2, dtype, 7)
    for name, value in (("valid", torch.zeros_like(case["valid"])), ("assignments", torch.full_like(case["assignments"], -1))):
        none, leaves, names = leaves_of({**case, name: value})
        y = call(none)
        assert (y == 0).all()
        for got in torch.autograd.grad(y, leaves, d_out):
            assert (got == 0).all()
    empty, leaves, names = leaves_of({**case, "context": case["context"][:0], "assignments": case["assignments"][:0],
                                      "pair_weights": case["pair_weights"][:0], "valid": case["valid"][:0]})
    y = call(empty)
    assert y.shape == (0, width)
    for leaf, got in zip(leaves, torch.autograd.grad(y.sum(), leaves)):
        assert got.shape == leaf.shape and (got == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("width,hidden", [(64, 128), (50, 90)])
def test_layouts(width, hidden):
    case, d_out = draw(120, width, hidden, 5, 2, torch.bfloat16, 8)
    shaped = {**case, "context": case["context"].reshape(4, 30, width), "assignments": case["assignments"].reshape(4, 30, 2),
              "pair_weights": case["pair_weights"].reshape(4, 30, 2), "valid": case["valid"].reshape(4, 30)}
    check(shaped, d_out.reshape(4, 30, width))
    odd = dict(case)
    odd["assignments"] = case["assignments"].int()
    wide = torch.full((120, width + 9), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:, 5:5 + width] = case["context"]
    odd["context"] = wide[:, 5:5 + width]
    odd["gate_weights"] = case["gate_weights"].transpose(1, 2).contiguous().transpose(1, 2)
    store = torch.empty(case["output_weights"].numel() + 1, device="cuda", dtype=torch.bfloat16)
    odd["output_weights"] = store[1:].view_as(case["output_weights"]).copy_(case["output_weights"])  # 2 bytes off
    odd["valid"] = torch.stack([case["valid"], ~case["valid"]], dim=1)[:, 0]
    check(odd, d_out)
    up = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(120, width)
    check(case, up)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,width,hidden", [(torch.bfloat16, 64, 128), (torch.float16, 64, 128), (torch.float32, 50, 90)])
def test_weights_of_slots_that_are_not_routed_do_not_matter(dtype, width, hidden):
    case, d_out = draw(700, width, hidden, 4, 2, dtype, 17)
    routed = (case["assignments"] >= 0) & case["valid"][:, None]
    case["pair_weights"] = torch.where(routed, case["pair_weights"], torch.full_like(case["pair_weights"], float("nan")))
    check(case, d_out)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [5, 16, 32, 64, 200])
def test_sorting_strided_ids_and_masks(tokens):
    """Each strided argument's copy lives until the sort has read it."""
    case, _ = draw(tokens, 64, 64, 6, 2, torch.bfloat16, tokens)
    ids, weights, valid = case["assignments"], case["pair_weights"], case["valid"]
    want = moe.permute_indices(ids, valid, expert_count=6, pair_weights=weights)
    strided = [torch.stack([t, t], dim=-1)[..., 0] for t in (ids, valid, weights)]
    got = moe.permute_indices(strided[0], strided[1], expert_count=6, pair_weights=strided[2])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    tokens_now, before = ids[:, 0].abs(), ids[:, 1].abs()
    want = moe.permute_hash_indices(tokens_now.contiguous(), before.contiguous(), valid, expert_count=6, top_k=2)
    got = moe.permute_hash_indices(tokens_now[:, None].expand(-1, 2).contiguous()[:, 0],
                                   before[:, None].expand(-1, 2).contiguous()[:, 0], strided[1], expert_count=6, top_k=2)
    for a, b in zip(got[:3] + got[4:], want[:3] + want[4:]):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,width,hidden", [(torch.bfloat16, 256, 512), (torch.float32, 100, 300)])
def test_nothing_is_kept_without_gradients(dtype, width, hidden):
    """Parameters that require gradients cost an evaluation no more memory than plain tensors do."""
    case, _ = draw(300, width, hidden, 4, 2, dtype, 31)
    trained, _, _ = leaves_of(case)
    peaks = []
    for which in (case, trained):
        with torch.no_grad():
            call(which)
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            start = torch.cuda.memory_allocated()
            y = call(which)
            peaks.append(torch.cuda.max_memory_allocated() - start)
            del y
    assert peaks[0] == peaks[1]


@pytest.mark.gpu
@pytest.mark.parametrize("width,hidden", [(64, 128), (50, 90)])
def test_each_gradient_alone(width, hidden):
    case, d_out = draw(150, width, hidden, 4, 2, torch.bfloat16, 9)
    full, leaves, names = leaves_of(case)
    want = torch.autograd.grad(call(full), leaves, d_out)
    for name, ref in zip(names, want):
        one = {n: (t.detach() if isinstance(t, torch.Tensor) else t) for n, t in case.items()}
        one[name] = one[name].clone().requires_grad_()
        (got,) = torch.autograd.grad(call(one), one[name], d_out)
        assert torch.equal(got, ref), name


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,dtype,width,hidden", [
    (90, torch.float32, 50, 90), (90, torch.float16, 64, 128), (90, torch.bfloat16, 50, 90), (90, torch.bfloat16, 64, 128),
    (90, torch.float32, 72, 88), (90, torch.float16, 200, 136), (900, torch.bfloat16, 64, 128), (900, torch.bfloat16, 256, 320)])
def test_non_finite_values_stay_where_they_belong(tokens, dtype, width, hidden):
    case, d_out = draw(tokens, width, hidden, 3, 1, dtype, 10)
    case["valid"][:] = True
    case["context"] = torch.nan_to_num(case["context"], nan=0.5)
    d_out = torch.nan_to_num(d_out, posinf=0.25)
    ids = case["assignments"][:, 0]
    token = (ids == 1).nonzero()[0, 0]
    case["context"][token, 3] = float("nan")
    case, leaves, names = leaves_of(case)
    y = call(case)
    grads = dict(zip(names, torch.autograd.grad(y, leaves, d_out)))
    others = torch.arange(tokens, device="cuda") != token
    assert y[token].isnan().all() and y[others].isfinite().all()
    assert grads["context"][token].isnan().all() and grads["context"][others].isfinite().all()
    for name in NAMES[2:]:
        assert grads[name][[0, 2]].isfinite().all(), name
    assert grads["gate_weights"][1].isnan().all() and grads["output_biases"][1].isfinite().all()
    # an infinite weight: infinities and NaN for its expert alone, as multiply-adds give them
    case["context"] = torch.nan_to_num(case["context"].detach(), nan=0.5)
    case["output_weights"] = case["output_weights"].detach().clone()
    case["output_weights"][2, 4, 5] = float("inf")
    y = call(case)
    bad = ids == 2
    assert (~y[bad][:, 4].isfinite()).all() and y[bad][:, 5].isfinite().all() and y[~bad].isfinite().all()


@pytest.mark.gpu
def test_gradients_against_differences():
    # float32: a difference of step 2^-6 of a sum of products of order one; third-order terms near 2^-12 of it
    case, d_out = draw(40, 24, 40, 3, 2, torch.float32, 11)
    case["context"], d_out = torch.nan_to_num(case["context"], nan=0.1), torch.nan_to_num(d_out, posinf=0.1)
    case, leaves, names = leaves_of(case)
    grads = torch.autograd.grad(call(case), leaves, d_out)
    gen = torch.Generator(device="cuda").manual_seed(2)
    for name, grad in zip(names, grads):
        v = torch.randn(grad.shape, device="cuda", generator=gen)
        v = v / v.norm()
        ends = []
        for sign in (1.0, -1.0):
            with torch.no_grad():
                moved = {**case, name: case[name] + sign * 2.0 ** -6 * v}
                ends.append((call(moved).double() * d_out.double()).sum().item())
        slope, want = (ends[0] - ends[1]) * 2.0 ** 5, (grad.double() * v.double()).sum().item()
        assert abs(slope - want) < 5e-3 * (1.0 + abs(want)), (name, slope, want)


@pytest.mark.gpu
@pytest.mark.parametrize("width,hidden", [(64, 128), (50, 90)])
def test_captured_and_replayed(width, hidden):
    case, d_out = draw(400, width, hidden, 6, 2, torch.bfloat16, 12)
    case, leaves, names = leaves_of(case)

    def step():
        y = call(case, validate=False)
        return [t.detach() for t in (y, *torch.autograd.grad(y, leaves, d_out))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (13, 14, 15):
        new, up = draw(400, width, hidden, 6, 2, torch.bfloat16, seed)
        with torch.no_grad():
            for name in (*NAMES, "assignments", "valid"):
                case[name].copy_(new[name])
            d_out.copy_(up)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in held]
        for got, want in zip(kept, step()):
            assert torch.equal(got, want)


@pytest.mark.gpu
def test_repeats_and_ids_outside_the_catalog():
    case, _ = draw(10, 64, 64, 4, 2, torch.bfloat16, 16)
    case["valid"][:] = True
    case["context"] = torch.nan_to_num(case["context"], nan=1.0)
    case["assignments"] = torch.tensor([[0, 1]] * 10, device="cuda")
    case["assignments"][2], case["assignments"][3], case["assignments"][4] = (torch.tensor(v, device="cuda") for v in ((3, 3), (7, 2), (-5, 1)))
    with pytest.raises(moe.CudaMoeValidationError):
        call(case)
    alone = {**case, "assignments": case["assignments"].clone()}
    alone["assignments"][2, 1] = alone["assignments"][3, 0] = alone["assignments"][4, 0] = -1
    assert torch.equal(call(case, validate=False), call(alone))  # they count nothing
    case["valid"][2:5] = False
    call(case)  # what an invalid token's slots say does not matter


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("ids", [(3, 3), (7, 2), (2, 4), (5, -1), (-5, 1), (-2, -1)])
def test_each_bad_choice_is_refused(ids, dtype):
    case, _ = draw(10, 64, 64, 4, 2, torch.bfloat16, 18)
    case["valid"][:], case["valid"][1] = True, False
    case["context"] = torch.nan_to_num(case["context"], nan=1.0)
    case["assignments"] = torch.tensor([[0, -1], list(ids), [-1, -1]] + [[0, 1]] * 7, device="cuda", dtype=dtype)
    call(case)
    case["valid"][1] = True
    with pytest.raises(moe.CudaMoeValidationError):
        call(case)


def test_refusals_on_the_cpu():
    t = torch.zeros
    args = [t(3, 8), t(3, 2, dtype=torch.int64), t(3, 2), torch.ones(3, dtype=torch.bool), t(4, 6, 8), t(4, 6), t(4, 6, 8), t(4, 6),
            t(4, 8, 6), t(4, 8)]
    with pytest.raises(moe.CudaMoeValidationError, match="CUDA tensor"):
        moe.expert_mixture(*args)
    with pytest.raises(TypeError):
        moe.expert_mixture(None, *args[1:])


@pytest.mark.gpu
def test_refusals():
    def t(*shape, dtype=torch.float32):
        return torch.zeros(shape, device="cuda", dtype=dtype)

    good = [t(3, 8), t(3, 2, dtype=torch.int64), t(3, 2), torch.ones(3, dtype=torch.bool, device="cuda"), t(4, 6, 8), t(4, 6),
            t(4, 6, 8), t(4, 6), t(4, 8, 6), t(4, 8)]
    good[1][:, 1] = 1
    moe.expert_mixture(*good)
    for i, bad in ((0, t(3, 8).double()), (0, t(3, 9)), (0, t(2, 8)), (0, t(3, 8).half()), (1, t(3, 2)), (1, t(3, 5, dtype=torch.int64)),
                   (1, t(2, 2, dtype=torch.int64)), (2, t(3, 3)), (2, t(3, 2).half()), (3, t(3)), (3, good[3][:2]), (4, t(4, 6)),
                   (4, t(4, 0, 8)), (5, t(4, 7)), (6, t(4, 6, 9)), (7, t(6)), (8, t(4, 6, 8)), (9, t(4, 9)), (9, t(4, 8).cpu())):
        args = list(good)
        args[i] = bad
        with pytest.raises(moe.CudaMoeValidationError):
            moe.expert_mixture(*args)
    many = list(good)  # nothing is allocated for shapes past what a launch takes
    many[:4] = good[0][:1].expand(1 << 25, 8), good[1][:1].expand(1 << 25, 2), good[2][:1].expand(1 << 25, 2), good[3][:1].expand(1 << 25)
    with pytest.raises(moe.CudaMoeValidationError, match="2\\^26"):
        moe.expert_mixture(*many)
    wide = [t(1, 1).expand(1 << 19, 1 << 15), good[1][:1].expand(1 << 19, 2), None, good[3][:1].expand(1 << 19), t(4, 6, 1).expand(4, 6, 1 << 15),
            good[5], t(4, 6, 1).expand(4, 6, 1 << 15), good[7], t(4, 1, 6).expand(4, 1 << 15, 6), t(4, 1).expand(4, 1 << 15)]
    with pytest.raises(moe.CudaMoeValidationError, match="2\\^34"):
        moe.expert_mixture(*wide)


@pytest.mark.parametrize("shape", [(1 << 26, 1, 64, 64, 4), (1 << 20, 2, 1 << 16, 64, 4), (4, 257, 64, 64, 512), (8, 2, 1 << 22, 64, 4),
                                   (8, 2, 1 << 17, 1 << 17, 4), (-1, 2, 64, 64, 4), (8, 0, 64, 64, 4), (8, 2, 64, 64, 0)])
def test_sizes_past_a_launch_are_refused(shape):
    for name, last in (("koemi_moe_experts_saved_bytes", ()), ("koemi_moe_experts_workspace_bytes", (1,))):
        assert _native.query(name, *shape, _native.dtype_code(torch.bfloat16), *last) == 0
        assert _native.query(name, 1000, 2, 64, 128, 4, _native.dtype_code(torch.bfloat16), *last) > 0
