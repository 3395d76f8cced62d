"""The filtered draw (sampling.sample_tokens) against its definition in float64, row by row.

Ids have to be equal: the reference forms weights and running sums in float64, off by under 2^-40
of the whole from the kernel's whole multiples of 2^-44 (at most 2^19 of them, each off by half
a step: 2^-26 of the largest weight's sum at worst, 2^-45 sqrt(2^19) as they fall); so a row
whose u, or whose top-p border, lies nearer to a running sum than 2^-24 of the whole is left
out of the comparison, and no more than a few are. Probabilities are off by that and half a step
of float32.
"""

from __future__ import annotations

import math

import pytest
import torch

from koemi_amd import herm
from koemi_amd import sampling as S


def reference(z, u, temperature, top_k, top_p, min_p, exclude):
    """Id, distribution and how near a border a row lies, in float64."""

    z = z.double().clone()
    z[torch.isnan(z)] = -math.inf
    if exclude is not None:
        z[exclude] = -math.inf
    top = z.max()
    if top == -math.inf:
        return 0, torch.zeros_like(z), 1.0
    if top == math.inf:
        z = torch.where(z == math.inf, 0.0, -math.inf)
        top = z.max()
    near = 1.0
    if top_k is not None and top_k < z.numel():
        z = torch.where(z < z.sort(descending=True)[0][top_k - 1], -math.inf, z)
    w = torch.exp((z - top) / temperature)
    keep = w >= (min_p or 0.0)
    if top_p is not None and top_p < 1.0:
        levels, index = torch.unique(z, return_inverse=True)
        mass = torch.zeros_like(levels).index_add_(0, index, w).flip(0)
        above = mass.cumsum(0) - mass
        keep &= (above < top_p * w.sum()).flip(0)[index]
        near = min(near, ((above - top_p * w.sum()).abs().min() / w.sum()).item())
    w = torch.where(keep, w, 0.0)
    running = w.cumsum(0)
    near = min(near, ((running - float(u) * running[-1]).abs().min() / running[-1]).item()) if u else near
    return int((running > float(u) * running[-1]).to(torch.int32).argmax()), w / w.sum(), near


def check(z, u, most_skipped=0.02, **limits):
    exclude = limits.get("exclude")
    ids, probabilities = S.sample_tokens(z, u, with_probabilities=True, **limits)
    assert torch.equal(S.sample_tokens(z, u, **limits), ids)
    skipped = 0
    for r in range(z.shape[0]):
        want, p, near = reference(z[r], u[r], limits.get("temperature", 1.0), limits.get("top_k"), limits.get("top_p"),
                                  limits.get("min_p"), exclude)
        if near < 2.0 ** -24:
            skipped += 1
            continue
        assert int(ids[r]) == want, (r, int(ids[r]), want, limits)
        assert ((probabilities[r].double() - p).abs() <= 2.0 ** -24 * p + 2.0 ** -24 * p.max()).all()
        if p.sum() > 0:
            assert p[int(ids[r])] > 0
    assert skipped <= max(1, most_skipped * z.shape[0]), skipped


LIMITS = [{}, {"temperature": 0.3}, {"top_k": 1}, {"top_k": 40}, {"top_p": 0.9}, {"min_p": 0.1}, {"top_p": 1.0, "min_p": 0.0},
          {"top_k": 50, "top_p": 0.8, "min_p": 0.02, "temperature": 1.7}, {"top_p": 1e-6}, {"min_p": 1.0}, {"top_k": 10 ** 9, "top_p": 0.5}]


@pytest.mark.gpu
@pytest.mark.parametrize("limits", LIMITS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows, vocab", [(5, 1), (33, 2), (64, 257), (7, 511), (3, 2049), (4, 5000), (2, 50001)])
def test_against_float64(device, rows, vocab, dtype, limits):
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    z = (3.0 * torch.randn(rows, vocab, device=device, generator=gen)).to(dtype)
    u = torch.rand(rows, device=device, generator=gen)
    exclude = vocab // 2 if vocab > 2 and rows % 2 else None
    check(z, u, exclude=exclude, **limits)


@pytest.mark.gpu
@pytest.mark.parametrize("limits", [{}, {"top_k": 7}, {"top_p": 0.6}, {"min_p": 0.5}, {"top_k": 300, "top_p": 0.3}])
def test_equal_scores_and_odd_values(device, limits):
    """Ties in great numbers (more than a list holds), infinities, NaN, zeros of either sign, huge gaps."""

    vocab = 9000
    z = torch.zeros(8, vocab, device=device)
    z[1] = (torch.arange(vocab, device=device) % 3).float()
    z[2, ::2] = -0.0
    z[3, 17::1000] = float("inf")
    z[4] = float("-inf")
    z[4, 8999] = -3.0e38
    z[5, ::3] = float("nan")
    z[6] = torch.linspace(-3e38, 3e38, vocab, device=device)
    z[7] = float("-inf")
    u = torch.tensor([0.0, 0.4999, 0.75, 0.55, 0.999, 1.0 - 2.0 ** -24, 0.5, 0.3], device=device)
    check(z, u, **limits)
    assert int(S.sample_tokens(z, u, **limits)[7]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("limits", LIMITS)
@pytest.mark.parametrize("vocab, dtype", [(65536, torch.float32), (70001, torch.bfloat16), (1 << 19, torch.float16)])
def test_long_rows_against_float64(device, vocab, dtype, limits):
    """Rows in several workgroups. Of 2^19 running sums one lies within 2^-24 of u in a row of sixteen, of
    top-p's border in as many: of eight rows four are hardly ever left out."""

    gen = torch.Generator(device="cuda").manual_seed(vocab + 1)
    z = (3.0 * torch.randn(8, vocab, device=device, generator=gen)).to(dtype)
    check(z, torch.rand(8, device=device, generator=gen), most_skipped=0.5, exclude=vocab - 1, **limits)


@pytest.mark.gpu
@pytest.mark.parametrize("limits", [{}, {"top_k": 7}, {"top_p": 0.6}, {"min_p": 0.5}, {"top_k": 300, "top_p": 0.3}])
def test_long_rows_of_equal_scores_and_odd_values(device, limits):
    vocab = 70003
    z = torch.zeros(8, vocab, device=device)
    z[1] = (torch.arange(vocab, device=device) % 3).float()
    z[2, ::2] = -0.0
    z[3, 17::1000] = float("inf")
    z[4] = float("-inf")
    z[4, 70002] = -3.0e38
    z[5, ::3] = float("nan")
    z[6] = torch.linspace(-3e38, 3e38, vocab, device=device)
    z[7] = float("-inf")
    u = torch.tensor([0.0, 0.4999, 0.75, 0.55, 0.999, 1.0 - 2.0 ** -24, 0.5, 0.3], device=device)
    check(z, u, **limits)
    assert int(S.sample_tokens(z, u, **limits)[7]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("limits", [{}, {"top_p": 0.9, "min_p": 0.01}, {"top_k": 50, "top_p": 0.8, "temperature": 0.7}])
def test_one_workgroup_a_row_and_several_agree(device, limits):
    """129 rows take one workgroup each, fewer take several: the same bits, also on another stream."""

    gen = torch.Generator(device="cuda").manual_seed(6)
    z = (2.0 * torch.randn(129, 66000, device=device, generator=gen)).bfloat16()
    u = torch.rand(129, device=device, generator=gen)
    ids, probabilities = S.sample_tokens(z, u, with_probabilities=True, **limits)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    for rows in (1, 5, 128):
        with torch.cuda.stream(other):
            got, p = S.sample_tokens(z[:rows], u[:rows], with_probabilities=True, **limits)
        other.synchronize()
        assert torch.equal(got, ids[:rows])
        assert torch.equal(p, probabilities[:rows])


@pytest.mark.gpu
def test_long_rows_in_a_graph(device):
    gen = torch.Generator(device="cuda").manual_seed(8)
    z = torch.randn(4, 65536, device=device, generator=gen)
    u = torch.rand(4, device=device, generator=gen)
    S.sample_tokens(z, u, top_k=40, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids = S.sample_tokens(z, u, top_k=40, top_p=0.9)
    for _ in range(3):
        z.normal_(generator=gen)
        u.uniform_(generator=gen)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(S.sample_tokens(z, u, top_k=40, top_p=0.9), ids)


@pytest.mark.gpu
def test_rows_apart_and_no_rows(device):
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(6, 1003, device=device, generator=gen)
    u = torch.rand(6, device=device, generator=gen)
    part = wide[:, 1:1000]
    assert torch.equal(S.sample_tokens(part, u, top_p=0.9), S.sample_tokens(part.contiguous(), u, top_p=0.9))
    assert torch.equal(S.sample_tokens(wide.t().contiguous().t(), u, top_k=9), S.sample_tokens(wide, u, top_k=9))
    spread = torch.rand(12, device=device, generator=gen)[::2]
    assert torch.equal(S.sample_tokens(wide, spread), S.sample_tokens(wide, spread.contiguous()))
    assert S.sample_tokens(wide[:0], u[:0]).shape == (0, 1)
    first = wide[:1].expand(6, -1)  # a stride of zero
    assert torch.equal(S.sample_tokens(first, u), S.sample_tokens(first.contiguous(), u))


@pytest.mark.gpu
def test_a_policy_draws_with_them(device):
    gen = torch.Generator(device="cuda").manual_seed(4)
    logits = torch.randn(32, 257, device=device, generator=gen)
    u = torch.rand(32, device=device, generator=gen)
    sampler = S.TokenSampler(S.SamplingPolicy(temperature=0.7, top_k=60, top_p=0.8, min_p=0.01), device)
    ids, probabilities = sampler.sample_with_probabilities(logits, uniforms=u)
    want, distribution = S.sample_tokens(logits, u, temperature=0.7, top_k=60, top_p=0.8, min_p=0.01, exclude=256, with_probabilities=True)
    assert torch.equal(ids, want) and torch.equal(probabilities, distribution) and (probabilities[:, 256] == 0).all()
    assert torch.equal(sampler(logits, uniforms=u), want)
    # without the new limits: a vocabulary past what the narrow kernel takes
    wide = torch.randn(4, 5000, device=device, generator=gen)
    got = S.TokenSampler(S.SamplingPolicy(top_k=5), device)(wide, uniforms=u[:4])
    assert torch.equal(got, S.sample_tokens(wide, u[:4], top_k=5, exclude=256))


@pytest.mark.gpu
def test_a_decode_graph_draws_with_them(device):
    """Replays of the captured step, with eager work between them, against eager steps."""

    settings = herm.HermSettings(width=64, memory_features=4, local_memory_size=4, salience_memory_size=3,
                                 expert_count=4, top_k=2, layers=2, scan_chunk=8)
    params = herm.prepare_stack(herm.init_stack(settings, 5, device), settings, device)
    ids = torch.randint(0, 256, (8, 1), generator=torch.Generator().manual_seed(2)).to(device)
    policy = S.SamplingPolicy(temperature=0.9, top_p=0.7, min_p=0.01)
    decode = herm.DecodeGraph(params, settings, ids, herm.initial_states(settings, 8, device), policy=policy,
                              generator=torch.Generator(device=device).manual_seed(9))
    for step in range(5):
        logits = decode.run().clone()
        want = S.TokenSampler(policy, device)(logits[:, -1], uniforms=decode.uniforms.clone())
        torch.cuda.synchronize()
        assert torch.equal(decode.ids, want), step


@pytest.mark.parametrize("limits, message", [
    ({"temperature": 0.0}, "temperature must be positive"), ({"top_k": 0}, "top_k must be a positive integer"), ({"top_k": True}, "top_k must be a positive integer"),
    ({"top_p": 0.0}, "top_p must be a number above 0"), ({"top_p": 1.01}, "top_p must be a number"),
    ({"min_p": -0.1}, "min_p must be a number from 0"), ({"min_p": float("nan")}, "min_p must be a number")])
def test_policies_refuse(limits, message):
    with pytest.raises(ValueError, match=message):
        S.SamplingPolicy(**limits)


def test_fronts_refuse_before_anything_runs():
    u = torch.zeros(2)
    with pytest.raises(ValueError, match=r"\[batch, vocabulary\]"):
        S.sample_tokens(torch.zeros(2, 3, 4), u)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        S.sample_tokens(torch.zeros(2, 3, dtype=torch.float64), u)
    with pytest.raises(ValueError, match="CUDA"):
        S.sample_tokens(torch.zeros(2, 3), u)


@pytest.mark.gpu
@pytest.mark.parametrize("change, message", [
    ({"uniforms": torch.zeros(3)}, "uniforms must be"), ({"temperature": 1e31}, "temperature"), ({"temperature": "1"}, "temperature"),
    ({"top_k": -1}, "top_k"), ({"top_p": 0.0}, "top_p"), ({"min_p": 1.5}, "min_p"), ({"exclude": 9}, "exclude"), ({"exclude": -1}, "exclude")])
def test_calls_refuse(device, change, message):
    uniforms = change.pop("uniforms", torch.zeros(2, device=device))
    with pytest.raises(ValueError, match=message):
        S.sample_tokens(torch.zeros(2, 9, device=device), uniforms, **change)
