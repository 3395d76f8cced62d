"""The windowed attention, its cache and the draw together, as a prompt and its continuation use them.

A prompt in chunks (attention over what the cache holds and the chunk, then the chunk written), single
positions, and the ids drawn from their read, against float64 over the values that the cache
stands for; the steps captured in a graph; edges of the cache that no sequence reaches by itself.
"""

from __future__ import annotations

import math

import pytest
import torch

import test_gpu_window_attention as attention
import test_gpu_window_cache as caching
from koemi_amd import sampling
from koemi_amd import window as W
from koemi_amd.think import CudaThinkValidationError


@pytest.mark.gpu
@pytest.mark.parametrize("code", caching.CODES)
def test_a_prompt_in_chunks_and_its_continuation(device, code):
    batch, heads, groups, width, window, sinks, vocab = 2, 6, 2, 64, 50, 3, 700
    gen = torch.Generator(device="cuda").manual_seed(12)
    cache = W.window_cache(batch, groups, width, window=window, sinks=sinks, dtype=code, device=device)
    plain = caching.Plain(cache)
    lengths = torch.zeros(batch, dtype=torch.int64, device=device)
    slots = window + sinks
    for length in (40, 70, 9):
        q = caching.rows(gen, batch, length, heads, width, dtype=torch.bfloat16)
        k, v = (caching.rows(gen, batch, length, groups, width, dtype=torch.bfloat16) for _ in range(2))
        counts = torch.tensor([length, max(1, length - 13)], device=device)
        held_k, held_v, present = W.window_cache_entries(cache, lengths, dtype=torch.bfloat16)
        chunk = torch.arange(length, device=device)[None] < counts[:, None]
        out = W.window_attention(q, torch.cat([held_k, k], 1), torch.cat([held_v, v], 1), torch.cat([present, chunk], 1),
                                 window=window, sinks=sinks)
        # the same queries over each row's own entries, all in one sequence
        for b in range(batch):
            n, count = int(lengths[b]), int(counts[b])
            entries = plain.held(n)
            at = [plain.slot(p) for p in entries]
            past = [plain.stands_for(name, b, at, torch.float32).to(torch.bfloat16).transpose(0, 1)[None] for name in ("keys", "values")]
            keys, values = (torch.cat([p, new[b:b + 1, :count]], 1) for p, new in zip(past, (k, v)))
            places = torch.tensor(entries + list(range(n, n + count)), device=device)
            i, j = places[len(entries):, None], places[None]
            see = (j <= i) & ((i - j < window) | (j < sinks))
            kk, vv = (t[0].double().repeat_interleave(heads // groups, 1).transpose(0, 1) for t in (keys, values))
            s = torch.matmul(q[b, :count].double().transpose(0, 1), kk.transpose(1, 2).contiguous()) / math.sqrt(width)
            p = torch.softmax(s.masked_fill(~see, float("-inf")), dim=-1)
            want, size = torch.matmul(p, vv).transpose(0, 1), torch.matmul(p, vv.abs()).transpose(0, 1)
            big = torch.where(see, s.abs(), 0.0).amax()
            attention.close(out[b, :count], want, (2.0 ** -8 + 2.0 ** -16 * (1 + big)) * size, (length, b))
            assert not out[b, count:].any()
        W.window_cache_write(cache, k, v, lengths, counts)
        for b in range(batch):
            for t in range(int(counts[b])):
                plain.append(b, int(lengths[b]) + t, k[b, t], v[b, t])
        plain.check()
        lengths = lengths + counts
    head = torch.randn(vocab, heads * width, device=device, generator=gen) / math.sqrt(heads * width)
    for _ in range(4):
        q = caching.rows(gen, batch, heads, width, dtype=torch.bfloat16)
        k, v = (caching.rows(gen, batch, groups, width, dtype=torch.bfloat16) for _ in range(2))
        read = W.window_cache_step(cache, q, k, v, lengths)
        for b in range(batch):
            plain.append(b, int(lengths[b]), k[b], v[b])
        lengths = lengths + 1
        for b in range(batch):
            want, bound = plain.read(b, int(lengths[b]), q[b], 1.0 / math.sqrt(width))
            caching.close(read[b], want, bound, b)
        logits = torch.mm(read.reshape(batch, -1).float(), head.t())
        u = torch.rand(batch, device=device, generator=gen)
        ids, p = sampling.sample_tokens(logits, u, top_k=50, top_p=0.9, min_p=0.01, with_probabilities=True)
        assert ((p > 0).sum(dim=1) <= 50).all() and (p.gather(1, ids) > 0).all()
    plain.check()
    assert slots == cache.keys.shape[2]


@pytest.mark.gpu
@pytest.mark.parametrize("code", caching.CODES)
def test_captured_steps(device, code):
    """Write, read and draw in a graph, the counts advanced inside it; eager work between replays."""

    batch, heads, groups, width, window, sinks = 3, 4, 2, 96, 600, 2
    gen = torch.Generator(device="cuda").manual_seed(5)
    cache = W.window_cache(batch, groups, width, window=window, sinks=sinks, dtype=code, device=device)
    other = W.window_cache(batch, groups, width, window=window, sinks=sinks, dtype=code, device=device)
    lengths = torch.tensor([0, 599, 1500], device=device)
    first = [caching.rows(gen, batch, 1500, groups, width, dtype=torch.float16) for _ in range(2)]
    for c in (cache, other):
        W.window_cache_write(c, *first, torch.zeros_like(lengths), lengths)
    q = torch.zeros(batch, heads, width, device=device, dtype=torch.float16)
    k, v = (torch.zeros(batch, groups, width, device=device, dtype=torch.float16) for _ in range(2))
    u, at, active = torch.zeros(batch, device=device), lengths.clone(), torch.ones(batch, dtype=torch.bool, device=device)

    def step(c, counts):
        out = W.window_cache_step(c, q, k, v, counts, active)
        counts += active
        return out, sampling.sample_tokens(out.reshape(batch, -1), u, top_p=0.8, min_p=0.01)

    spare = [t.clone() for t in (other.keys.view(torch.uint8), other.key_scales, other.values.view(torch.uint8), other.value_scales)]
    warm = W.WindowCache(spare[0].view(code), spare[1], spare[2].view(code), spare[3], width=width, window=window, sinks=sinks)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, lengths.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(cache, at)
    eager = lengths.clone()
    for turn in range(5):
        for t in (q, k, v):
            t.copy_(caching.rows(gen, *t.shape, dtype=torch.float16))
        u.uniform_(generator=gen)
        active.copy_(torch.rand(batch, device=device, generator=gen) < 0.7)
        graph.replay()
        want = step(other, eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), turn
        assert torch.equal(at, eager) and torch.equal(cache.keys.view(torch.uint8), other.keys.view(torch.uint8))
        assert torch.equal(cache.value_scales, other.value_scales)


@pytest.mark.gpu
@pytest.mark.parametrize("code", caching.CODES)
def test_rows_that_are_not_finite_or_tiny_or_zero(device, code):
    groups, width, window = 2, 40, 8
    cache = W.window_cache(1, groups, width, window=window, dtype=code, device=device)
    plain = caching.Plain(cache)
    keys = torch.zeros(1, 8, groups, width, device=device)
    keys[0, 0, 0, 3], keys[0, 1, 1, 39], keys[0, 2, 0, 0] = float("nan"), float("inf"), float("-inf")
    keys[0, 3], keys[0, 4, :, 7], keys[0, 5], keys[0, 6] = 3e38, 2.0 ** -149, 1e-40, -5e-39
    values = keys.flip(1).clone()
    lengths = torch.zeros(1, dtype=torch.int64, device=device)
    W.window_cache_write(cache, keys, values, lengths)
    for t in range(8):
        plain.append(0, t, keys[0, t], values[0, t])
    plain.check()
    got, _, present = W.window_cache_entries(cache, lengths + 8, dtype=torch.float32)
    assert present.all() and torch.isnan(got[0, 0, 0]).all() and torch.isfinite(got[0, 0, 1]).all() and not got[0, 7].any()
    # a read that sees an entry of NaN is NaN in the heads that see it, and only there
    q = torch.randn(1, 4, width, device=device)
    read = W.window_cache_read(cache, q, lengths + 1)
    assert torch.isnan(read[0, :2]).all()
    one = W.window_cache(1, groups, width, window=window, dtype=code, device=device)
    W.window_cache_write(one, torch.zeros_like(keys), torch.zeros_like(keys), lengths)
    assert not W.window_cache_read(one, q, lengths + 8).any()


@pytest.mark.gpu
@pytest.mark.parametrize("code", caching.CODES)
def test_what_no_entry_holds_does_not_matter(device, code):
    """Buffers of a program's own, full of anything: slots without an entry are neither read nor written."""

    batch, groups, width, window, sinks = 3, 2, 72, 300, 4
    gen = torch.Generator(device="cuda").manual_seed(2)
    shape = (batch, groups, window + sinks)
    junk = lambda: torch.full((*shape, 96), 0x7f, device=device, dtype=torch.uint8).view(code)  # noqa: E731
    nan = lambda: torch.full(shape, float("nan"), device=device)  # noqa: E731
    cache = W.WindowCache(junk(), nan(), junk(), nan(), width=width, window=window, sinks=sinks)
    clean = W.window_cache(batch, groups, width, window=window, sinks=sinks, dtype=code, device=device)
    keys, values = (caching.rows(gen, batch, 50, groups, width, dtype=torch.bfloat16) for _ in range(2))
    keys[1, 20:], values[2] = float("nan"), float("inf")
    lengths, counts = torch.tensor([0, 2, -1], device=device), torch.tensor([99, 20, 50], device=device)
    start = torch.zeros(batch, dtype=torch.int64, device=device)
    for c in (cache, clean):
        W.window_cache_write(c, keys[:, :2].nan_to_num(0, 0, 0), values[:, :2].nan_to_num(0, 0, 0), start, torch.tensor([0, 2, 0], device=device))
        W.window_cache_write(c, keys, values, lengths, counts)
    held = torch.tensor([50, 22, 0], device=device)
    for c in (cache, clean):
        W.window_cache_write(c, keys, values, held, torch.tensor([0, -3, 0], device=device))
    q = torch.randn(batch, 4, width, device=device, dtype=torch.bfloat16)
    for n in (held, torch.tensor([50, 22, -7], device=device)):
        a, b = W.window_cache_read(cache, q, n), W.window_cache_read(clean, q, n)
        assert torch.equal(a, b) and torch.isfinite(a).all() and not a[2].any()
    for a, b in zip(W.window_cache_entries(cache, held, dtype=torch.float32), W.window_cache_entries(clean, held, dtype=torch.float32)):
        assert torch.equal(a, b)
    assert (cache.keys.view(torch.uint8)[0, :, 50:] == 0x7f).all() and torch.isnan(cache.key_scales[2]).all()
    # inactive rows and negative lengths: left as they are
    before = cache.keys.view(torch.uint8).clone()
    off = torch.tensor([False, True, True], device=device)
    out = W.window_cache_step(cache, q, q[:, :2].contiguous(), q[:, 2:], torch.tensor([50, -1, -9], device=device), off)
    assert not out.any() and torch.equal(cache.keys.view(torch.uint8), before)


@pytest.mark.gpu
def test_rows_of_any_strides(device):
    batch, heads, groups, width, window = 2, 4, 2, 64, 20
    gen = torch.Generator(device="cuda").manual_seed(6)
    wide = torch.randn(batch, 9, (heads + 2 * groups) * width, device=device, generator=gen).to(torch.bfloat16)
    q, k, v = (t.unflatten(-1, (-1, width)) for t in wide.split([heads * width, groups * width, groups * width], dim=-1))
    flipped = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (k, v)]
    caches = [W.window_cache(batch, groups, width, window=window, device=device) for _ in range(3)]
    lengths = torch.zeros(batch, dtype=torch.int64, device=device)
    W.window_cache_write(caches[0], k.contiguous(), v.contiguous(), lengths)
    W.window_cache_write(caches[1], k, v, lengths)
    W.window_cache_write(caches[2], *flipped, lengths)
    n = lengths + 9
    outs = [W.window_cache_step(caches[0], q[:, 8].contiguous(), k[:, 3].contiguous(), v[:, 3].contiguous(), n),
            W.window_cache_step(caches[1], q[:, 8], k[:, 3], v[:, 3], torch.stack([n, n], 1)[:, 0]),
            W.window_cache_step(caches[2], q[:, 8], flipped[0][:, 3], flipped[1][:, 3], n)]
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    assert all(torch.equal(caches[0].keys, c.keys) and torch.equal(caches[0].value_scales, c.value_scales) for c in caches[1:])


@pytest.mark.gpu
def test_cache_past_2_31_bytes(device):
    """The last rows of a cache whose codes pass 2^31 bytes."""

    batch, groups, width, window = 70, 8, 128, 33000
    assert batch * groups * window * width > 1 << 31
    cache = W.window_cache(batch, groups, width, window=window, device=device)
    gen = torch.Generator(device="cuda").manual_seed(1)
    keys, values = (torch.randn(batch, 40, groups, width, device=device, generator=gen, dtype=torch.bfloat16) for _ in range(2))
    lengths = torch.full((batch,), (1 << 33) + 5, dtype=torch.int64, device=device)
    W.window_cache_write(cache, keys, values, lengths)
    n = int(lengths[0]) + 40
    at = [(p % window) for p in range(n - 40, n)]
    codes, scales = caching.quantised(keys[-1], torch.int8)
    assert torch.equal(cache.keys.view(torch.uint8)[-1][:, at].transpose(0, 1), codes)
    assert torch.equal(cache.key_scales[-1][:, at].t(), scales)
    # entries never written hold zeros: they weigh as a score of 0 and add nothing
    q = torch.randn(batch, 8, width, device=device, generator=gen)
    out = W.window_cache_read(cache, q, lengths + 40)
    k = cache.keys[-1][:, at].double() * cache.key_scales[-1][:, at][..., None]
    v = cache.values[-1][:, at].double() * cache.value_scales[-1][:, at][..., None]
    e = torch.exp(torch.matmul(k, q[-1].double()[:, :, None])[..., 0] / math.sqrt(width))
    want = torch.matmul((e / (e.sum(-1, keepdim=True) + window - 40))[:, None], v)[:, 0]
    size = torch.matmul((e / (e.sum(-1, keepdim=True) + window - 40))[:, None], v.abs())[:, 0]
    caching.close(out[-1], want, 2.0 ** -14 * size, "read")  # 2 (2^-19 (1 + 8) + 2^-21), scores below 8


@pytest.mark.parametrize("numbers, message", [
    ({"window": 0}, "window must be a positive integer"), ({"sinks": -1}, "sinks must be a non-negative integer"), ({"width": 0}, "width must be"),
    ({"width": 257}, "wide"), ({"dtype": torch.uint8}, "int8 or float8_e4m3fn"), ({"window": True}, "window must be")])
def test_caches_that_are_refused(numbers, message):
    with pytest.raises(CudaThinkValidationError, match=message):
        W.window_cache(2, 2, **({"width": 8, "window": 4, "device": "cpu"} | numbers))


def test_calls_that_are_refused():
    """On the CPU: every refusal comes before anything runs."""

    cache = W.window_cache(2, 2, 8, window=4, sinks=1, device="cpu")
    rows, q, n = torch.zeros(2, 3, 2, 8), torch.zeros(2, 4, 8), torch.zeros(2, dtype=torch.int64)
    one = rows[:, 0]
    calls = [
        (lambda: W.window_cache_write(None, rows, rows, n), "WindowCache"),
        (lambda: W.window_cache_write(cache, rows[:, :, :1], rows, n), "shape"),
        (lambda: W.window_cache_write(cache, rows[0], rows, n), "shape"),
        (lambda: W.window_cache_write(cache, rows, rows.half(), n), "one type"),
        (lambda: W.window_cache_write(cache, rows.double(), rows.double(), n), "float32, float16"),
        (lambda: W.window_cache_write(cache, rows, rows, n.int()), "lengths must be an int64"),
        (lambda: W.window_cache_write(cache, rows, rows, n, n[:1]), "counts must be an int64"),
        (lambda: W.window_cache_write(cache, rows, rows, n), "on CUDA"),
        (lambda: W.window_cache_entries(cache, n, dtype=torch.int8), "dtype must be"),
        (lambda: W.window_cache_entries(cache, n, dtype=torch.float32), "on CUDA"),
        (lambda: W.window_cache_step(cache, q[:, :3], one, one, n), "divide"),
        (lambda: W.window_cache_step(cache, q[..., :4], one, one, n), "shape"),
        (lambda: W.window_cache_step(cache, q, one, None, n), "values must be a torch.Tensor"),
        (lambda: W.window_cache_step(cache, q, one.half(), one, n), "one type"),
        (lambda: W.window_cache_step(cache, q, one, one, n, n), "active must be a bool"),
        (lambda: W.window_cache_step(cache, q, one, one, n, scale=-1.0), "scale must be"),
        (lambda: W.window_cache_read(cache, q, n), "on CUDA"),
        (lambda: W.WindowCache(cache.keys[:, :, 1:], cache.key_scales, cache.values, cache.value_scales, width=8, window=4, sinks=1), "codes must be"),
        (lambda: W.WindowCache(cache.keys, cache.key_scales.double(), cache.values, cache.value_scales, width=8, window=4, sinks=1), "float32"),
        (lambda: W.WindowCache(cache.keys.transpose(0, 1), cache.key_scales, cache.values, cache.value_scales, width=8, window=4, sinks=1), "contiguous"),
        (lambda: W.WindowCache(cache.keys, cache.key_scales, cache.values.view(torch.float8_e4m3fn), cache.value_scales, width=8, window=4, sinks=1), "int8 or"),
    ]
    for call, message in calls:
        with pytest.raises(CudaThinkValidationError, match=message):
            call()
