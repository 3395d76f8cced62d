"""The trained operators past 2^31 elements, and on two streams at once.

Only the first and the last positions count (the others are masked, or carry no
gradient), so that float64 references of those alone hold for the whole call, with the
bounds of the operators' own tests.
"""

from __future__ import annotations

import pytest
import torch

import test_gpu_experts_training as experts_tests
import test_gpu_recurrence_training as recurrence_tests
import test_gpu_route_training as route_tests
from koemi_amd import moe, recurrent

ENDS = 200


def ends(length):
    return torch.cat([torch.arange(ENDS, device="cuda"), torch.arange(length - ENDS, length, device="cuda")])


@pytest.mark.gpu
def test_recurrence_of_more_than_2_31_preactivations():
    length, width = (1 << 20) + 77, 1030
    assert length * 2 * width > 1 << 31
    at = ends(length)
    small = recurrence_tests.draw((1, 2 * ENDS, width), torch.bfloat16, 3, "")
    z = torch.full((1, length, 2 * width), float("nan"), device="cuda", dtype=torch.bfloat16)
    d_states = torch.zeros((1, length, width), device="cuda", dtype=torch.bfloat16)
    valid = torch.zeros((1, length), device="cuda", dtype=torch.bool)
    z[:, at], d_states[:, at], valid[:, at] = small[0], small[3], True
    z, initial = z.requires_grad_(), small[2].clone().requires_grad_()
    states, final = recurrent.gated_recurrence(z, valid, initial)
    d_z, d_initial = torch.autograd.grad((states, final), (z, initial), (d_states, small[4]))
    want = recurrence_tests.reference(small[0], None, *small[2:])
    recurrence_tests.close(states[:, at], want[0], want[4], "states")
    recurrence_tests.close(final, want[1], want[4][:, -1], "final")
    recurrence_tests.close(d_z[:, at], want[2], want[5], "d_z")
    recurrence_tests.close(d_initial, want[3], want[6], "d_initial")
    assert (states[:, ENDS:-ENDS] == states[:, ENDS - 1:ENDS]).all() and not d_z[:, ENDS:-ENDS].any()


@pytest.mark.gpu
def test_route_of_more_than_2_31_logits():
    tokens, experts, top_k = (1 << 21) + 33, 1024, 2
    at = ends(tokens)
    small, _, _, d_weights, d_mass, d_loss = route_tests.draw(2 * ENDS, experts, top_k, torch.bfloat16, 5)
    small = torch.nan_to_num(small, nan=0.0, posinf=1.0, neginf=-1.0)
    logits = torch.full((tokens, experts), float("nan"), device="cuda", dtype=torch.bfloat16)
    valid = torch.zeros(tokens, device="cuda", dtype=torch.bool)
    up = torch.full((tokens, top_k), float("nan"), device="cuda")
    logits[at], valid[at], up[at] = small, True, d_weights
    logits.requires_grad_()
    assignments, weights, statistics = moe.route_topk_balanced(logits, valid, top_k=top_k)
    outs = (weights, statistics.probability_mass, statistics.balance_loss)
    (d_logits,) = torch.autograd.grad(outs, logits, (up, d_mass, d_loss))
    want = route_tests.reference(small, valid[at], top_k, d_weights, d_mass, d_loss)
    assert torch.equal(assignments[at], want["assignments"]) and (assignments[ENDS:-ENDS] == -1).all()
    assert statistics.valid_count.item() == 2 * ENDS
    route_tests.close(weights[at], want["weights"], want["w_bound"], "weights")
    route_tests.close(statistics.probability_mass, want["mass"], want["mass_bound"], "mass")
    route_tests.close(d_logits[at], want["d_z"], want["d_bound"], "d_logits")
    assert not d_logits[ENDS:-ENDS].any() and not weights[ENDS:-ENDS].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,width,hidden", [(torch.bfloat16, 64, 2112), (torch.float16, 16, 2104)])
def test_experts_of_more_than_2_31_hidden_values(dtype, width, hidden):
    tokens = (1 << 20) + 99
    assert tokens * hidden > 1 << 31
    at = ends(tokens)
    case, d_out = experts_tests.draw(tokens, width, hidden, 2, 1, dtype, 7)
    case["valid"][:] = True
    case["context"] = torch.nan_to_num(case["context"], nan=0.5)
    keep = torch.zeros(tokens, device="cuda", dtype=torch.bool)
    keep[at] = True
    d_out = torch.where(keep[:, None], torch.nan_to_num(d_out, posinf=0.25), torch.zeros_like(d_out))
    case, leaves, names = experts_tests.leaves_of(case)
    y = experts_tests.call(case)
    grads = dict(zip(names, torch.autograd.grad(y, leaves, d_out)))
    rows = ("context", "assignments", "pair_weights", "valid")
    want = experts_tests.reference({n: t.detach()[at] if n in rows else t for n, t in case.items()}, d_out[at])
    experts_tests.close(y[at], *want["out"], "out")
    for name, got in grads.items():
        experts_tests.close(got[at] if name in rows else got, *want[name], name)
    assert not grads["context"][~keep].any() and not grads["pair_weights"][~keep].any()


@pytest.mark.gpu
def test_two_streams_at_once():
    def case_of(seed):
        z, valid, initial, d_states, _ = recurrence_tests.draw((3, 400, 64), torch.bfloat16, seed, "random")
        case, d_out = experts_tests.draw(1200, 64, 128, 4, 2, torch.bfloat16, seed)
        logits = route_tests.draw(1200, 4, 2, torch.float32, seed)[0]
        return z, valid, initial, d_states, case, torch.nan_to_num(d_out, posinf=0.5), torch.nan_to_num(logits)

    def step(z, valid, initial, d_states, case, d_out, logits):
        z, logits = z.detach().requires_grad_(), logits.detach().requires_grad_()
        states, _ = recurrent.gated_recurrence(z, valid, initial)
        ids, weights, statistics = moe.route_topk_balanced(logits, case["valid"], top_k=2)
        case, leaves, _ = experts_tests.leaves_of({**case, "assignments": ids, "pair_weights": weights})
        y = experts_tests.call(case, validate=False)
        grads = torch.autograd.grad((states, y, statistics.balance_loss), (z, logits, *leaves),
                                    (d_states, d_out, torch.ones((), device="cuda")))
        return [t.detach() for t in (states, y, *grads)]

    cases = [case_of(41), case_of(42)]
    want = [step(*c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for c, stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                got.append(step(*c))
        torch.cuda.synchronize()
        for one, ref in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(one, ref))
