"""Calls of the windowed attention and its cache at the edges of what they take.

Precision that does not depend on a call's size, layouts of padded rows, infinities, values and keys of any size,
chunks behind a cache whose rows lack their sinks, and what is refused; against float64 with the bounds of
test_gpu_window_attention.py and of test_gpu_window_cache.py.
"""

from __future__ import annotations

import math

import pytest
import torch

import test_gpu_window_attention as attention
import test_gpu_window_cache as caching
from koemi_amd import window as W
from koemi_amd.think import CudaThinkValidationError


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


def positions_last(t):
    """The same values in the layout that an operator over positions hands back: neighbours along the positions."""

    return t.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)


def stray_stride(t):
    """A single position whose stride, which nothing steps by, is odd."""

    t = t.contiguous()
    return t.as_strided(t.shape, (t.stride(0), 1, t.stride(2), t.stride(3)))


@pytest.mark.parametrize("width, padded", [(10, 16), (16, 16), (3, 4)])
def test_copies_of_rows_are_contiguous(width, padded):
    t = torch.arange(2 * 7 * 3 * width, dtype=torch.float32).reshape(2, 7, 3, width)
    for rows in (t, positions_last(t), t.transpose(1, 2), t[:, :1], stray_stride(t[:, :1]), t[:1, :, :1], t[:0]):
        got = W._rows(rows, padded)
        shape = (*rows.shape[:3], padded)
        assert got.shape == shape and got.stride() == torch.empty(shape).stride()
        assert torch.equal(got[..., :width], rows) and not got[..., width:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width", [10, 64, 100])
@pytest.mark.parametrize("layout", ["gradient", "inputs", "both", "one position"])
def test_rows_whose_neighbours_lie_along_the_positions(device, layout, width, dtype):
    """The gradient that an operator over positions hands back, and such inputs, at widths on and off 16 bytes."""

    length = 1 if layout == "one position" else 90
    q, k, v, valid, d_out = attention.make((2, length, 4, 2, width), dtype, 17, "tail", total=90)
    inputs, up = [q, k, v], d_out
    if layout in ("inputs", "both"):
        inputs = [positions_last(t) for t in inputs]
    if layout in ("gradient", "both"):
        up = positions_last(up)
    if layout == "one position":
        inputs, up = [stray_stride(q), k, v], stray_stride(d_out)

    def step(tensors, up):
        leaves = [t.detach().requires_grad_() for t in tensors]
        out = W.window_attention(*leaves, valid, window=20, sinks=2)
        return (out, *torch.autograd.grad(out, leaves, up))

    want = step([t.contiguous() for t in (q, k, v)], d_out)
    assert all(torch.equal(a, b) for a, b in zip(step(inputs, up), want))
    attention.check(q, k, v, valid, d_out, 20, 2)


@pytest.mark.gpu
def test_a_convolution_over_positions_behind_heads_of_ten(device):
    """The same layout from a real graph: what follows the heads runs over channels first."""

    q, k, v, _, _ = attention.make((2, 60, 3, 1, 10), torch.float32, 4, None)
    weight = torch.randn(5, 30, 3, device=device)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = W.window_attention(*leaves, window=9, sinks=1)
    got = []
    out.register_hook(lambda g: got.append(g))
    loss = torch.nn.functional.conv1d(out.flatten(2).transpose(1, 2), weight).square().sum()
    grads = torch.autograd.grad(loss, leaves)
    want, bounds = attention.reference(q, k, v, None, 9, 1, 1.0 / math.sqrt(10), got[0])
    for g, w, b, name in zip(grads, want[1:], bounds[1:], ("d_queries", "d_keys", "d_values")):
        attention.close(g, w, b, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch, sinks", [(2, 2), (90, 2), (2, 0)])
@pytest.mark.parametrize("value", ["inf", "-inf", "nan", "overflow"])
def test_an_infinite_gradient_reaches_every_key_that_its_row_sees(device, value, batch, sinks, dtype):
    """D, the sum of d_out times out, of any size and sign: a row whose D is infinite counts like any other.

    Column 5 of the values is positive, so with d_out = +-inf there D is, too, and every ds of the row NaN. With
    overflow it is finite: the columns 5 and 6 of values are 0 or 3 (in fp16, whose largest D is far below fp32's, this
    one has no infinite D and is left out), so that D = 2^127 (out_5 + out_6) passes 2^128 in heads where out_5 + out_6 >= 2.
    Where it does not, keys of zeros have finite derivatives.
    """

    if value == "overflow" and dtype == torch.float16:
        return
    window, length, at = 40, 200, 130
    q, k, v, _, d_out = attention.make((batch, length, 4, 2, 64), dtype, 3, None)
    v[..., 5] = v[..., 5].abs() + 1.0
    i = torch.arange(length, device=device)
    if value == "overflow":
        v[..., 5:7] = 3.0 * (i % 2 == 0)[None, :, None, None]
        d_out[0, at, :, 5:7] = 2.0 ** 127
    else:
        d_out[0, at, :, 5] = float(value)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = W.window_attention(*leaves, window=window, sinks=sinks)
    d_q, d_k, d_v = torch.autograd.grad(out, leaves, d_out)
    seen = ((i <= at) & (at - i < window)) | (i < sinks)
    assert torch.isfinite(out).all() and not torch.isfinite(d_q[0, at]).any()
    reached = torch.ones(2, dtype=torch.bool, device=device)  # key heads
    if value == "overflow":
        reached = (out[0, at, :, 5].double() + out[0, at, :, 6].double() >= 2.0).view(2, 2).any(dim=1)
        assert reached.any()
    assert not torch.isfinite(d_k[0, seen][:, reached]).any()
    assert torch.isfinite(d_k[0, ~seen]).all() and torch.isfinite(d_k[1:]).all() and torch.isfinite(d_q[0, i != at]).all()
    if value != "overflow":
        assert not torch.isfinite(d_v[0, seen][..., 5]).any() and torch.isfinite(d_v[0, ~seen]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch, length, window", [(2, 200, 40), (90, 200, 150), (1, 2000, 1200)])
@pytest.mark.parametrize("value", [float("inf"), float("-inf")])
def test_an_infinity_that_a_row_sees_is_an_infinity(device, value, batch, length, window, dtype):
    """A sum with one infinite term is infinite, of the term's sign: outputs over an infinite value. The gradients of
    values under an infinite d_out are not finite. Rows and keys that see none stay within their bounds.
    Scores are small, so that no probability vanishes."""

    sinks, at = 1, 130
    q, k, v, _, d_out = attention.make((batch, length, 4, 2, 64), dtype, 5, None)
    i = torch.arange(length, device=device)
    sees = (i >= at) & (i - at < window)
    seen = ((i <= at) & (at - i < window)) | (i < sinks)
    one = slice(0, 1)
    want, bounds = attention.reference(q[one], k[one], v[one], None, window, sinks, 0.125, d_out[one])
    bad = v.clone()
    bad[0, at, :, 9] = value
    for train in (False, True):
        leaves = [t.clone().requires_grad_(train) for t in (q, k, bad)]
        out = W.window_attention(*leaves, window=window, sinks=sinks)[0]
        assert (out[sees][..., 9] == value).all()
        others = [c for c in range(64) if c != 9]
        attention.close(out[..., others], want[0][0][..., others], bounds[0][0][..., others], "out")
        attention.close(out[~sees], want[0][0][~sees], bounds[0][0][~sees], "out")
    up = d_out.clone()
    up[0, at, :, 9] = value
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    d_v = torch.autograd.grad(W.window_attention(*leaves, window=window, sinks=sinks), leaves, up)[2][0]
    assert not torch.isfinite(d_v[seen][..., 9]).any()
    attention.close(d_v[..., others], want[3][0][..., others], bounds[3][0][..., others], "d_values")
    attention.close(d_v[~seen], want[3][0][~seen], bounds[3][0][~seen], "d_values")


@pytest.mark.parametrize("which", ["queries", "keys", "values"])
def test_forward_mode_is_refused(which):
    """A tangent is not dropped: there is no forward-mode derivative. On the CPU, before anything runs."""

    tensors = {"queries": torch.zeros(2, 5, 4, 8), "keys": torch.zeros(2, 5, 2, 8), "values": torch.zeros(2, 5, 2, 8)}
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(CudaThinkValidationError, match="must be on CUDA"):  # an open level alone refuses nothing
            W.window_attention(*tensors.values(), window=3)
        tensors[which] = torch.autograd.forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(CudaThinkValidationError, match="forward-mode"):
                W.window_attention(*tensors.values(), window=3)


def held_cache(code, keys, values, window, sinks=0):
    """A cache that holds these rows [batch, n, groups, width], its plain form, and the counts."""

    batch, n, groups, width = keys.shape
    cache = W.window_cache(batch, groups, width, window=window, sinks=sinks, dtype=code, device=keys.device)
    none = torch.zeros(batch, dtype=torch.int64, device=keys.device)
    W.window_cache_write(cache, keys, values, none)
    return cache, caching.Plain(cache), none + n


def read_and_step(cache, plain, counts, queries, key, value, scale):
    """window_cache_read and _step against float64 over what the cache stands for."""

    n = int(counts[0])
    read = W.window_cache_read(cache, queries, counts, scale=scale)
    for b in range(queries.shape[0]):
        want, bound = plain.read(b, n, queries[b], scale)
        caching.close(read[b], want, bound, ("read", b))
    out = W.window_cache_step(cache, queries, key, value, counts, scale=scale)
    for b in range(queries.shape[0]):
        plain.append(b, n, key[b], value[b])
        want, bound = plain.read(b, n + 1, queries[b], scale)
        caching.close(out[b], want, bound, ("step", b))
    plain.check()


@pytest.mark.gpu
@pytest.mark.parametrize("code", caching.CODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("entries, width", [(20, 40), (700, 64), (5000, 128)])
@pytest.mark.parametrize("size", [2.0 ** -124, 1e-35, 1e-31, 1e-27, 1e-10, 1e10, 1e30, 3e37])
def test_values_of_any_size_are_read(device, size, entries, width, dtype, code):
    """Values from the smallest scale to the largest: bounds are relative to them, and their sum before it is divided passes the range."""

    gen = torch.Generator(device="cuda").manual_seed(entries)
    keys, values = (torch.randn(2, entries, 2, width, device=device, generator=gen) for _ in range(2))
    if size > 1.0:  # one sign, so that the unscaled sum is large
        values = values.abs()
    values = (values * size).clamp(max=3e38).to(dtype)
    cache, plain, counts = held_cache(code, keys.to(dtype), values, 5000)
    queries = torch.randn(2, 6, width, device=device, generator=gen).to(dtype)
    key = torch.randn(2, 2, width, device=device, generator=gen).to(dtype)
    value = (torch.randn(2, 2, width, device=device, generator=gen).abs() * size).clamp(max=3e38).to(dtype)
    read_and_step(cache, plain, counts, queries, key, value, 1.0 / math.sqrt(width))


@pytest.mark.gpu
@pytest.mark.parametrize("code", caching.CODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-31, 1.0, 1e17, 1e20, 1e37])
def test_rows_of_zeros_with_rising_scores_after_values_of_any_size(device, size, dtype, code):
    """One wave's chunks lie 256 slots apart: values first, then chunks of zero rows (whose scale is 2^-126), each of which brings a new
    largest score, and a last chunk of small values. Scores rise by 1 a chunk, so that the first values stay in the result."""

    width, chunks = 64, 8
    gen = torch.Generator(device="cuda").manual_seed(9)
    i = torch.arange(256 * chunks, device=device)
    keys = torch.zeros(1, 256 * chunks, 1, width, device=device)
    keys[0, :, 0, 0] = (i // 256).float()
    values = torch.randn(1, 256 * chunks, 1, width, device=device, generator=gen) * size
    values[0, 256:-256] = 0.0
    values[0, -256:] *= 2.0 ** -20
    queries = torch.zeros(1, 3, width, device=device)
    queries[0, :, 0] = torch.tensor([1.0, 0.5, -1.0], device=device)
    cache, plain, counts = held_cache(code, keys.to(dtype), values.to(dtype), 4096)
    read_and_step(cache, plain, counts, queries.to(dtype), keys[:, -1].to(dtype), values[:, 0].to(dtype), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("code", caching.CODES)
@pytest.mark.parametrize("seed", range(6))
def test_values_of_mixed_sizes(device, seed, code):
    """Rows whose sizes are spread over sixty binary orders of magnitude, with scores over some tens."""

    gen = torch.Generator(device="cuda").manual_seed(seed)
    entries, width = 1500, 32
    spread = torch.exp2(torch.rand(2, entries, 2, 1, device=device, generator=gen) * 60.0 - 30.0)
    keys = torch.randn(2, entries, 2, width, device=device, generator=gen)
    values = torch.randn(2, entries, 2, width, device=device, generator=gen) * spread
    cache, plain, counts = held_cache(code, keys, values, 1024, sinks=3)
    queries = torch.randn(2, 4, width, device=device, generator=gen)
    read_and_step(cache, plain, counts, queries, keys[:, 5], values[:, 7], 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("code", caching.CODES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("key_size", [2.0 ** -100, 2.0 ** -60, 2.0 ** 60, 2.0 ** 100, 2.0 ** 122])
def test_keys_of_any_size_are_scored(device, key_size, dtype, code):
    """Large keys under small queries and the reverse: scores of order one, whose factors alone pass the range."""

    width, entries = 64, 300
    gen = torch.Generator(device="cuda").manual_seed(13)
    keys = (torch.randn(2, entries, 2, width, device=device, generator=gen) * key_size).to(dtype)
    values = torch.randn(2, entries, 2, width, device=device, generator=gen).to(dtype)
    queries = (torch.randn(2, 4, width, device=device, generator=gen) / min(key_size, 2.0 ** 110)).to(dtype)
    cache, plain, counts = held_cache(code, keys, values, 512)
    scale = 0.125 * min(1.0, 2.0 ** 110 / key_size)
    read_and_step(cache, plain, counts, queries, keys[:, 3], values[:, 4], scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width, window, sinks, chunks", [
    (64, 50, 3, (70, 20, 9)),          # a first chunk longer than the window
    (64, 30, 5, (2, 1, 3, 40, 40)),    # chunks shorter than the sinks
    (128, 40, 130, (100, 90, 200)),    # sinks of more than two tiles, filled over two chunks
    (10, 20, 4, (33, 300)),
    (32, 16, 1, (900, 30)),            # many tiles between the late sinks and the window
    (64, 100, 0, (150, 20)),
    (256, 25, 70, (60, 130)),
])
def test_chunks_behind_a_cache_whatever_its_rows_hold(device, width, window, sinks, chunks, dtype):
    """Every row's chunks against float64 over its own entries in one sequence: rows that are behind with their sinks, fresh
    ones among old ones, rows that pause. The sinks are a row's first entries, in the cache or in the chunk."""

    batch, heads, groups = 4, 6, 2
    gen = torch.Generator(device="cuda").manual_seed(width + sinks)
    cache = W.window_cache(batch, groups, width, window=window, sinks=sinks, device=device)
    plain = caching.Plain(cache)
    lengths = torch.zeros(batch, dtype=torch.int64, device=device)
    scale = 1.0 / math.sqrt(width)
    for turn, length in enumerate(chunks):
        q = torch.randn(batch, length, heads, width, device=device, generator=gen).to(dtype)
        k, v = (torch.randn(batch, length, groups, width, device=device, generator=gen).to(dtype) for _ in range(2))
        counts = torch.tensor([length, max(1, length - 13), min(2, length), 0 if turn == 0 else length], device=device)
        held_k, held_v, present = W.window_cache_entries(cache, lengths, dtype=dtype)
        chunk = torch.arange(length, device=device)[None] < counts[:, None]
        out = W.window_attention(q, torch.cat([held_k, k], 1), torch.cat([held_v, v], 1), torch.cat([present, chunk], 1),
                                 window=window, sinks=sinks, lengths=lengths)
        for b in range(batch):
            n, count = int(lengths[b]), int(counts[b])
            assert not out[b, count:].any()
            if not count:
                continue
            entries = plain.held(n)
            at = [plain.slot(p) for p in entries]
            past = [plain.stands_for(name, b, at, torch.float32).to(dtype).transpose(0, 1) for name in ("keys", "values")]
            kk, vv = (torch.cat([p, new[b, :count]]).double().repeat_interleave(heads // groups, 1).transpose(0, 1)
                      for p, new in zip(past, (k, v)))
            places = torch.tensor(entries + list(range(n, n + count)), device=device)
            i, j = places[len(entries):, None], places[None]
            see = (j <= i) & ((i - j < window) | (j < sinks))
            qq = q[b, :count].double().transpose(0, 1)
            s = torch.matmul(qq, kk.transpose(1, 2).contiguous()) * scale
            size = torch.where(see, torch.matmul(qq.abs(), kk.abs().transpose(1, 2).contiguous()) * scale, 0.0).amax(dim=-1, keepdim=True)
            p = torch.softmax(s.masked_fill(~see, float("-inf")), dim=-1)
            half = attention.HALF_STEP[dtype]
            bound = torch.matmul((half * half + 2.0 ** -17 * (1.0 + size)) * p, vv.abs())
            attention.close(out[b, :count], torch.matmul(p, vv).transpose(0, 1), bound.transpose(0, 1), (length, b))
        W.window_cache_write(cache, k, v, lengths, counts)
        for b in range(batch):
            for t in range(int(counts[b])):
                plain.append(b, int(lengths[b]) + t, k[b, t], v[b, t])
        lengths = lengths + counts


@pytest.mark.gpu
def test_a_chunk_of_one_position_and_full_rows(device):
    """With all sinks held, or none to hold, `lengths` changes nothing, whatever else it says; negative ones hold nothing."""

    gen = torch.Generator(device="cuda").manual_seed(1)
    for length, window, sinks in ((1, 30, 4), (70, 30, 4), (40, 600, 2), (5, 3, 0)):
        q = torch.randn(3, length, 4, 64, device=device, generator=gen).bfloat16()
        k, v = (torch.randn(3, sinks + window + length, 2, 64, device=device, generator=gen).bfloat16() for _ in range(2))
        valid = torch.rand(3, sinks + window + length, device=device, generator=gen) < 0.8
        want = W.window_attention(q, k, v, valid, window=window, sinks=sinks)
        for held in ([sinks, sinks + 9, 1 << 40], torch.tensor([[sinks, 0], [1 << 62, 0], [sinks, 0]])[:, 0]):
            held = torch.as_tensor(held).to(device)
            assert torch.equal(W.window_attention(q, k, v, valid, window=window, sinks=sinks, lengths=held), want)
        none, less = (W.window_attention(q, k, v, valid, window=window, sinks=sinks, lengths=torch.full((3,), n, device=device)) for n in (0, -5))
        assert torch.equal(none, less)


@pytest.mark.gpu
def test_chunks_in_a_graph(device):
    """The counts are read on the device: replays with others."""

    gen = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(2, 40, 4, 64, device=device, generator=gen).bfloat16()
    k, v = (torch.randn(2, 56, 2, 64, device=device, generator=gen).bfloat16() for _ in range(2))
    valid, held = torch.ones(2, 56, dtype=torch.bool, device=device), torch.zeros(2, dtype=torch.int64, device=device)
    run = lambda: W.window_attention(q, k, v, valid, window=10, sinks=6, lengths=held)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for a, b in ((0, 3), (6, 1), (2, 100), (0, 0)):
        held.copy_(torch.tensor([a, b]))
        graph.replay()
        assert torch.equal(out, run())


def test_chunks_that_are_refused():
    q, k, n = torch.zeros(2, 5, 4, 8), torch.zeros(2, 12, 2, 8), torch.zeros(2, dtype=torch.int64)
    valid = torch.ones(2, 12, dtype=torch.bool)

    def call(lengths=n, mask=valid, sinks=3, queries=q):
        return lambda: W.window_attention(queries, k, k, mask, window=4, sinks=sinks, lengths=lengths)

    for bad, message in ((call(lengths=n.int()), "lengths must be an int64"), (call(lengths=n[:1]), "lengths must be an int64"),
                         (call(lengths=[0, 0]), "lengths must be an int64"), (call(mask=None), "with lengths"), (call(sinks=2), "with lengths"),
                         (call(queries=q.clone().requires_grad_()), "no gradients with lengths"), (call(), "must be on CUDA")):
        with pytest.raises(CudaThinkValidationError, match=message):
            bad()


def test_the_library_refuses_chunks_that_it_cannot_take():
    import ctypes

    from koemi_amd import _native

    strides = (ctypes.c_int64 * 9)(*[64 * 4, 64, 16] * 3)

    def call(valid=16, held=16, length=4, window=2, sinks=1, width=16):
        return lambda: _native.call("koemi_window_attention_chunk", 16, 16, 16, valid, strides, held, 16, 1, length, 4, 4, width, window,
                                    sinks, 1.0, _native.F32, None, 0, None)

    for bad, message in ((call(valid=None), "null pointer"), (call(held=None), "null pointer"), (call(length=-1), "not negative"),
                         (call(window=0), "window"), (call(sinks=-1), "window"), (call(window=1 << 40), "2\\^29"), (call(width=320), "256")):
        with pytest.raises(_native.NativeCallError, match=message):
            bad()


def test_a_step_without_a_key_and_a_value_is_refused():
    """A step appends; reading alone is another call."""

    cache = W.window_cache(2, 2, 8, window=4, device="cpu")
    q, n = torch.zeros(2, 4, 8), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(CudaThinkValidationError, match="keys must be a torch.Tensor"):
        W.window_cache_step(cache, q, None, None, n)
    with pytest.raises(CudaThinkValidationError, match="keys must be a torch.Tensor"):
        W.window_cache_step(cache, q, None, q[:, :2], n)


def test_sizes_past_a_launch_are_refused():
    """On the host, before any launch: a launch takes fewer than 2^32 threads. Addresses are never followed."""

    import ctypes

    from koemi_amd import _native

    six = (ctypes.c_int64 * 6)(*[8] * 6)
    nine = (ctypes.c_int64 * 9)(*[16, 8, 8] * 3)

    def write(batch, length):
        return "koemi_window_cache_write", (16, 16, 16, 16, 0, 16, 16, six, 16, None, batch, length, 1, 8, 2, 0, _native.BF16, None)

    def entries(batch, window):
        return "koemi_window_cache_entries", (16, 16, 16, 16, 0, 16, 16, 16, 16, batch, 1, 8, window, 0, _native.BF16, None)

    def step(batch, heads, width):
        return "koemi_window_cache_step", (16, 16, 16, 16, 0, 16, None, None, six, 16, None, 16, batch, heads, heads, width, 1, 0, 1.0,
                                           _native.BF16, None, 0, None)

    def draw(rows, vocab):
        return "koemi_sample_filtered", (16, _native.F32, vocab, rows, vocab, -1, 1.0, 0, 1.0, 0.0, 16, 16, None, None, 0, None)

    def sinks(batch, total, window):
        need = _native.query("koemi_window_attention_backward_workspace_bytes", batch, total, total, 1, 1, 8, window, total, _native.BF16)
        return "koemi_window_attention_backward", (16, 16, 16, None, nine, 16, None, 16, 16, 16, 16, 16, batch, total, total, 1, 1, 8,
                                                   window, total, 1.0, _native.BF16, 16, need, None)

    for name, args in (write(1 << 20, 1024), entries(1 << 20, 1024), step(1 << 23, 1, 64), step(1 << 20, 8, 64), step(1 << 22, 4, 256),
                       draw(1 << 26, 2), draw(1 << 24, 600), draw(1 << 22, 5000), sinks(1 << 15, 1 << 14, 1)):
        with pytest.raises(_native.NativeCallError, match="2\\^32 threads"):
            _native.call(name, *args)
