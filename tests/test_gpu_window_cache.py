"""The 8-bit cache of the windowed attention (window.WindowCache) against plain torch.

Codes and scales have to be those of the definition, to the bit: scale = max(max |x| times 1 /
limit, 2^-126), 1 / limit rounded to float32, and x / scale are single correctly rounded
float32 operations, then rounded to nearest even. Reads are compared in float64 with the values that the codes stand for.
Bounds: a probability is off by the score's error, under E = 2^-19 (1 + the largest
|score|) (products with queries of 22 bits, fp32 sums and exponential), its product with the
value's scale by another 2^-21, so the output by 2 E sum_j p_j |v_j| and its own rounding.
Two planes end at fp16's smallest step: with the largest of a query at 2^14 or more, and the
largest p_j times its value's scale at 2^13 or more, each of them is off by up to half of 2^-24, so by
2^-39 and 2^-38 of the largest, however small itself; a score so by 2^-39 max |q| sum |k|,
the output by 2^-38 times the largest product and the sum of the |codes|.
"""

from __future__ import annotations

import math

import pytest
import torch

from koemi_amd import _native
from koemi_amd import window as W
from koemi_amd.think import CudaThinkValidationError

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
LIMIT = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def quantised(x, code):
    """Codes as bytes and scales of rows [..., width], by the definition."""

    x = x.float()
    fine = torch.isfinite(x).all(dim=-1)
    scale = (x.abs().amax(dim=-1) * torch.tensor(1.0 / LIMIT[code], device=x.device)).clamp(min=2.0 ** -126)
    y = torch.where(fine[..., None], x / scale[..., None], 0.0)
    y = y.round().clamp(-127, 127) if code == torch.int8 else y
    pad = torch.zeros(*y.shape[:-1], -y.shape[-1] % 32, device=y.device)
    return torch.cat([y, pad], dim=-1).to(code).view(torch.uint8), torch.where(fine, scale, float("nan"))


class Plain:
    """The cache as lists of entries."""

    def __init__(self, cache):
        self.cache, self.window, self.sinks = cache, cache.window, cache.sinks
        self.bytes = {n: getattr(cache, n).view(torch.uint8).clone() for n in ("keys", "values")}
        self.scales = {n: getattr(cache, n[:-1] + "_scales").clone() for n in ("keys", "values")}

    def slot(self, p):
        return p if p < self.sinks else self.sinks + (p - self.sinks) % self.window

    def append(self, b, p, key, value):
        for name, x in (("keys", key), ("values", value)):
            self.bytes[name][b, :, self.slot(p)], self.scales[name][b, :, self.slot(p)] = quantised(x, self.cache.keys.dtype)

    def check(self):
        for name in ("keys", "values"):
            assert torch.equal(getattr(self.cache, name).view(torch.uint8), self.bytes[name]), name
            got = getattr(self.cache, name[:-1] + "_scales")
            assert torch.equal(torch.nan_to_num(got, -1.0), torch.nan_to_num(self.scales[name], -1.0)), name

    def held(self, n):
        return list(range(min(n, self.sinks))) + list(range(max(self.sinks, n - self.window), n))

    def stands_for(self, name, b, slots, dtype=torch.float64):
        codes = self.bytes[name][b, :, slots].view(self.cache.keys.dtype).float()[..., :self.cache.width]
        return codes.to(dtype) * self.scales[name][b, :, slots][..., None].to(dtype)  # [groups, entries, width]

    def read(self, b, n, queries, scale):
        """Output and bound of queries [heads, width] in float64."""

        groups = self.bytes["keys"].shape[1]
        q = queries.double().reshape(groups, -1, self.cache.width)
        entries = self.held(n)
        if not entries:
            return torch.zeros_like(q).reshape(queries.shape), torch.zeros_like(q).reshape(queries.shape)
        slots = [self.slot(p) for p in entries]
        k, v = self.stands_for("keys", b, slots), self.stands_for("values", b, slots)
        s = torch.matmul(q, k.transpose(1, 2).contiguous()) * scale
        size = torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous()).amax(dim=-1, keepdim=True) * scale
        least = 2.0 ** -39 * scale * q.abs().amax(dim=-1, keepdim=True) * k.abs().sum(dim=-1).amax(dim=-1)[:, None, None]
        p = torch.softmax(s, dim=-1)
        off = 2 * (2.0 ** -19 * (1 + size) + 2.0 ** -21 + least)
        scales = self.scales["values"][b, :, slots].double()
        codes = v.abs() / scales[..., None]
        floor = 2.0 ** -38 * (p * scales[:, None]).amax(dim=-1, keepdim=True) * codes.sum(dim=1, keepdim=True)
        return torch.matmul(p, v).reshape(queries.shape), (off * torch.matmul(p, v.abs()) + floor).reshape(queries.shape)


def close(got, want, bound, what):
    assert torch.isfinite(got).all(), what
    allowed = bound + HALF_STEP[got.dtype] * (want.abs() + bound) + SMALLEST[got.dtype]
    worst = ((got.double() - want).abs() - allowed).max().item() if got.numel() else 0.0
    assert worst <= 0.0, (what, worst)


def rows(gen, *shape, dtype):
    wide = torch.randn(shape, device="cuda", generator=gen) * torch.exp(torch.randn(shape[:-1], device="cuda", generator=gen))[..., None]
    return wide.to(dtype)


CODES = [torch.int8, torch.float8_e4m3fn]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [  # batch, heads, groups, width, window, sinks
    (1, 1, 1, 8, 1, 0), (2, 4, 2, 32, 5, 2), (3, 6, 2, 72, 40, 3), (2, 8, 1, 64, 33, 0), (1, 34, 2, 128, 100, 4),
    (2, 5, 5, 100, 31, 40), (1, 2, 1, 251, 600, 1), (1, 3, 3, 160, 700, 0), (2, 2, 2, 192, 64, 1), (1, 4, 2, 224, 20, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch, heads, groups, width, window, sinks", SHAPES)
def test_chunks_and_steps(device, batch, heads, groups, width, window, sinks, dtype, code):
    """A row's life: chunks of several sizes, steps past the ring's end, everything read back."""

    gen = torch.Generator(device="cuda").manual_seed(width + window)
    cache = W.window_cache(batch, groups, width, window=window, sinks=sinks, dtype=code, device=device)
    plain = Plain(cache)
    lengths = torch.zeros(batch, dtype=torch.int64, device=device)
    scale = 1.0 / math.sqrt(width)
    for length in (3, 1, 2 * window + sinks + 5):
        keys, values = (rows(gen, batch, length, groups, width, dtype=dtype) for _ in range(2))
        counts = torch.randint(0, length + 1, (batch,), device=device, generator=gen)
        W.window_cache_write(cache, keys, values, lengths, counts)
        for b in range(batch):
            for t in range(int(counts[b])):
                plain.append(b, int(lengths[b]) + t, keys[b, t], values[b, t])
        plain.check()
        lengths += counts
        got_k, got_v, present = W.window_cache_entries(cache, lengths, dtype=dtype)
        for b in range(batch):
            n = int(lengths[b])
            entries = plain.held(n)
            places = [p if p < sinks else window + sinks - n + p for p in entries]
            want = torch.zeros(window + sinks, dtype=torch.bool, device=device)
            want[places] = True
            assert torch.equal(present[b], want)
            for got, name in ((got_k, "keys"), (got_v, "values")):
                full = torch.zeros(window + sinks, groups, width, device=device)
                if entries:
                    full[places] = plain.stands_for(name, b, [plain.slot(p) for p in entries], torch.float32).transpose(0, 1)
                assert torch.equal(got[b], full.to(dtype))
        for step in range(3):
            queries = rows(gen, batch, heads, width, dtype=dtype)
            key, value = (rows(gen, batch, groups, width, dtype=dtype) for _ in range(2))
            active = torch.rand(batch, device=device, generator=gen) < 0.7 if step else None
            out = W.window_cache_step(cache, queries, key, value, lengths, active)
            taken = torch.ones(batch, dtype=torch.bool, device=device) if active is None else active
            for b in range(batch):
                if taken[b]:
                    plain.append(b, int(lengths[b]), key[b], value[b])
            plain.check()
            lengths += taken
            for b in range(batch):
                want, bound = plain.read(b, int(lengths[b]) if taken[b] else 0, queries[b], scale)
                close(out[b], want, bound, (length, step, b))
            again = W.window_cache_read(cache, queries, lengths, active)
            for b in range(batch):
                want, bound = plain.read(b, int(lengths[b]) if taken[b] else 0, queries[b], scale)
                close(again[b], want, bound, (length, step, b, "read"))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [8, 32, 72, 96, 128, 200])
@pytest.mark.parametrize("code", CODES)
def test_long_windows_are_read_in_parts(device, code, width):
    batch, heads, groups, window, sinks = 2, 6, 2, 5000, 16
    gen = torch.Generator(device="cuda").manual_seed(3)
    cache = W.window_cache(batch, groups, width, window=window, sinks=sinks, dtype=code, device=device)
    assert _native.query("koemi_window_cache_step_workspace_bytes", batch, heads, groups, width, window, sinks) > 0
    lengths = torch.tensor([0, 0], device=device)
    keys, values = (rows(gen, batch, 9000, groups, width, dtype=torch.bfloat16) for _ in range(2))
    counts = torch.tensor([9000, 1700], device=device)
    W.window_cache_write(cache, keys, values, lengths, counts)
    plain = Plain(cache)  # codes are checked above
    queries, key, value = (rows(gen, batch, h, width, dtype=torch.float32) for h in (heads, groups, groups))
    out = W.window_cache_step(cache, queries, key, value, counts)
    for b in range(batch):
        plain.append(b, int(counts[b]), key[b], value[b])
        want, bound = plain.read(b, int(counts[b]) + 1, queries[b], 1.0 / math.sqrt(width))
        close(out[b], want, bound, b)
    plain.check()
