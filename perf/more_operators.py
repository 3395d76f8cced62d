"""Timed cases of the windowed attention with sinks, its 8-bit cache and the filtered draw of the next token.

Families (``op``):

* ``attend``: multi-head attention in which position i sees the last ``window``
  positions up to its own and the first ``sinks`` ones
  (``window.window_attention``), over a prompt's own keys or with ``carried``
  keys before them; with ``train`` also the gradients of queries, keys and values;
* ``cache``: a chunk of a prompt written into the 8-bit cache of the window and
  its sinks (``window.window_cache_write``) and the whole cache read back for
  the next chunk (``window.window_cache_entries``);
* ``step``: one generated position: its key and value written into that cache
  and its queries answered from it (``window.window_cache_step``);
* ``sample``: the next ids from logits and given uniform numbers, by temperature,
  top-k, top-p and min-p (``sampling.sample_tokens``), with ``full`` also the
  distribution they are drawn from.

``run`` computes each in plain torch, in 32 bits (the draw, whose borders decide
ids, in 64) and rounded once at the end; with ``own`` set it calls the package's
fronts. ``exact`` restates the definitions in 64 bits: the attention row block by
row block over all keys, the cache entry by entry, the draw row by row.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = Path(__file__).resolve().parent.parent / "koemi-5hom_amd"

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LIMIT = {"int8": 127.0, "e4m3": 448.0}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
SMALLEST_SCALE = 2.0 ** -126


def listed():
    return [
        # a few first bytes of a prompt: launch latency
        {"name": "attend_prompt_1x16", "op": "attend", "batch": 1, "length": 16, "carried": 0, "heads": 16, "groups": 16,
         "width": 64, "window": 16, "sinks": 4, "dtype": "bf16", "padded": False, "train": False},
        # one long prompt behind the keys of an earlier chunk
        {"name": "attend_prompt_1x16384", "op": "attend", "batch": 1, "length": 16384, "carried": 2052, "heads": 16, "groups": 4,
         "width": 128, "window": 2048, "sinks": 4, "dtype": "bf16", "padded": False, "train": False},
        # a training batch at the package's headline size (16 heads of 64: width 1024), rows padded to one length
        {"name": "attend_train_8x2048", "op": "attend", "batch": 8, "length": 2048, "carried": 0, "heads": 16, "groups": 4,
         "width": 64, "window": 512, "sinks": 4, "dtype": "bf16", "padded": True, "train": True},
        # one long document under training, a wide window
        {"name": "attend_train_1x16384", "op": "attend", "batch": 1, "length": 16384, "carried": 0, "heads": 8, "groups": 2,
         "width": 128, "window": 4096, "sinks": 1, "dtype": "bf16", "padded": False, "train": True},
        # odd sizes in half precision: heads shared by three, a width off the tiles
        {"name": "attend_train_5x777", "op": "attend", "batch": 5, "length": 777, "carried": 0, "heads": 6, "groups": 2,
         "width": 80, "window": 100, "sinks": 3, "dtype": "fp16", "padded": True, "train": True},
        # full precision, no sinks, one key head for all
        {"name": "attend_train_2x1500", "op": "attend", "batch": 2, "length": 1500, "carried": 0, "heads": 4, "groups": 1,
         "width": 48, "window": 256, "sinks": 0, "dtype": "fp32", "padded": False, "train": True},
        # a batch of prompts into an empty cache
        {"name": "cache_write_8x2048", "op": "cache", "batch": 8, "length": 2048, "groups": 4, "width": 64, "window": 2048,
         "sinks": 4, "dtype": "bf16", "codes": "int8", "padded": False, "filled": False},
        # a ragged chunk into a cache that has wrapped, odd sizes
        {"name": "cache_write_3x301", "op": "cache", "batch": 3, "length": 301, "groups": 5, "width": 72, "window": 500,
         "sinks": 3, "dtype": "fp16", "codes": "e4m3", "padded": True, "filled": True},
        # one generated position at the serving batch
        {"name": "step_64x1024", "op": "step", "batch": 64, "heads": 16, "groups": 4, "width": 64, "window": 1024, "sinks": 4,
         "dtype": "bf16", "codes": "int8", "padded": False},
        # few rows over a long window: the cache is read at the memory's rate
        {"name": "step_8x32768", "op": "step", "batch": 8, "heads": 32, "groups": 8, "width": 128, "window": 32768, "sinks": 16,
         "dtype": "bf16", "codes": "e4m3", "padded": True},
        # bytes and the padding id at the serving batch, with the distribution
        {"name": "sample_64x257", "op": "sample", "rows": 64, "vocab": 257, "dtype": "fp32", "temperature": 0.8, "top_k": 40,
         "top_p": 0.9, "min_p": 0.0, "exclude": 256, "full": True},
        # a large vocabulary
        {"name": "sample_128x131072", "op": "sample", "rows": 128, "vocab": 131072, "dtype": "bf16", "temperature": 1.0,
         "top_k": 0, "top_p": 0.95, "min_p": 0.02, "exclude": -1, "full": False},
    ]


def _log(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""

    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("attend", "attend", "attend", "cache", "step", "step", "sample"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    padded = rng.random() < 0.5
    if op == "sample":
        vocab = _log(rng, 2, 200000)
        return {"op": op, "rows": _log(rng, 1, min(256, (1 << 24) // vocab)), "vocab": vocab, "dtype": dtype,
                "temperature": round(rng.uniform(0.3, 1.7), 2), "top_k": rng.choice((0, 0, _log(rng, 1, vocab))),
                "top_p": rng.choice((1.0, 0.9, 0.95, 0.5)), "min_p": rng.choice((0.0, 0.0, 0.02, 0.1)),
                "exclude": rng.choice((-1, rng.randrange(vocab))), "full": rng.random() < 0.5}
    groups, shared = rng.choice((1, 2, 3, 4, 5, 8)), rng.choice((1, 1, 2, 3, 4, 8))
    width = rng.choice((64, 128, 64, 128, 32, 48, 72, 80, 96, 100, 192, 256, _log(rng, 8, 256)))
    sinks = rng.choice((0, 1, 4, _log(rng, 1, 64)))
    if op == "attend":
        heads = groups * shared
        length = _log(rng, 1, 16384)
        window = _log(rng, 1, 4096)
        carried = rng.choice((0, 0, _log(rng, 1, length)))
        def cells(n):
            return heads * n * (min(max(window, 16), n) + sinks)

        while cells(length + carried) > 1 << 28:
            length, carried = length // 2, carried // 2
        batch = _log(rng, 1, max(1, min(16, (1 << 28) // cells(length + carried))))
        return {"op": op, "batch": batch, "length": length, "carried": carried, "heads": heads, "groups": groups,
                "width": width, "window": window, "sinks": sinks, "dtype": dtype, "padded": padded,
                "train": rng.random() < 0.7}
    codes = rng.choice(("int8", "e4m3"))
    if op == "cache":
        window, length = _log(rng, 1, 8192), _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(32, (1 << 24) // (max(window, length) * groups * width))))
        return {"op": op, "batch": batch, "length": length, "groups": groups, "width": width, "window": window,
                "sinks": sinks, "dtype": dtype, "codes": codes, "padded": padded, "filled": rng.random() < 0.5}
    window = _log(rng, 1, 32768)
    batch = _log(rng, 1, max(1, min(128, (1 << 27) // (window * groups * width))))
    return {"op": op, "batch": batch, "heads": groups * shared, "groups": groups, "width": width, "window": window,
            "sinks": sinks, "dtype": dtype, "codes": codes, "padded": padded}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 40) + 29)


def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _stored(width):
    """Columns of a cached row: the head's width in whole blocks of 32."""

    return -(-width // 32) * 32


def _buffers(gen, case, filled):
    """The cache's four buffers: codes [batch, groups, slots, stored] and scales [batch, groups, slots]."""

    batch, groups, width, slots = case["batch"], case["groups"], case["width"], case["window"] + case["sinks"]
    stored, kind = _stored(width), case["codes"]
    out = {}
    for name in ("keys", "values"):
        codes = torch.zeros(batch, groups, slots, stored, dtype=CODES[kind], device="cuda")
        scales = torch.zeros(batch, groups, slots, device="cuda")
        if filled:  # rows of order one whose largest value has the largest code
            for b in range(batch):
                wide = _normal(gen, groups, slots, width, scale=LIMIT[kind] / 3.5).clamp(-LIMIT[kind], LIMIT[kind])
                codes[b, ..., :width] = (wide.round() if kind == "int8" else wide).to(CODES[kind])
            scales = (3.5 / LIMIT[kind]) * (0.5 + torch.rand(scales.shape, device="cuda", generator=gen))
        out[name], out[name[:-1] + "_scales"] = codes, scales
    return out


def prepare(case, seed):
    gen = _generator(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    state = {"case": case}
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # some ids are likelier than others in every row
        state["logits"] = (_normal(gen, rows, vocab, scale=2.0) + _normal(gen, vocab, scale=1.5)).to(dtype)
        state["uniforms"] = torch.rand(rows, device="cuda", generator=gen)
        return state
    batch, groups, width = case["batch"], case["groups"], case["width"]
    if op == "attend":
        length, total = case["length"], case["length"] + case["carried"]
        for name, rows, heads in (("queries", length, case["heads"]), ("keys", total, groups), ("values", total, groups)):
            state[name] = _normal(gen, batch, rows, heads, width, dtype=dtype)
            if case["train"]:
                state[name].requires_grad_()
        state["valid"] = None
        if case["padded"]:  # rows end at lengths of their own
            ends = torch.randint(0, total + 1, (batch,), device="cuda", generator=gen)
            state["valid"] = torch.arange(total, device="cuda")[None, :] < ends[:, None]
        if case["train"]:
            state["d_out"] = _normal(gen, batch, length, case["heads"], width, dtype=dtype)
        return state
    slots = case["window"] + case["sinks"]
    if op == "cache":
        length = case["length"]
        state |= _buffers(gen, case, case["filled"])
        state["new_keys"] = _normal(gen, batch, length, groups, width, dtype=dtype)
        state["new_values"] = _normal(gen, batch, length, groups, width, dtype=dtype)
        high = 2 * slots + 1 if case["filled"] else 1
        state["lengths"] = torch.randint(0, high, (batch,), device="cuda", generator=gen)
        state["counts"] = torch.randint(0, length + 1, (batch,), device="cuda", generator=gen) if case["padded"] else None
        state["after"] = state["lengths"] + (length if state["counts"] is None else state["counts"])
        return state
    state |= _buffers(gen, case, True)
    state["queries"] = _normal(gen, batch, case["heads"], width, dtype=dtype)
    state["new_keys"] = _normal(gen, batch, groups, width, dtype=dtype)
    state["new_values"] = _normal(gen, batch, groups, width, dtype=dtype)
    # most rows are past their window, some have not filled it
    state["lengths"] = torch.randint(slots // 2, 3 * slots + 1, (batch,), device="cuda", generator=gen)
    state["active"] = torch.rand(batch, device="cuda", generator=gen) < 0.85 if case["padded"] else None
    return state


# ------------------------------------------------------------- plain forms ---


def _banded(t, blocks, size, carry=True):
    """[B, blocks * size, G, W] -> [B, G, blocks, (2) size, W]: each block behind the one before it."""

    t = t.reshape(t.shape[0], blocks, size, *t.shape[2:]).permute(0, 3, 1, 2, 4)
    if not carry:
        return t
    before = torch.cat([torch.zeros_like(t[:, :, :1]), t[:, :, :-1]], dim=2)
    return torch.cat([before, t], dim=3)


def _unbanded(t, size):
    """The adjoint of _banded: every position's two copies added, [B, blocks * size, G, W]."""

    own_part, before = t[:, :, :, size:], t[:, :, 1:, :size]
    total = own_part + torch.cat([before, torch.zeros_like(own_part[:, :, :1])], dim=2)
    return total.permute(0, 2, 3, 1, 4).flatten(1, 2)


def _plain_attend(state):
    case, valid = state["case"], state["valid"]
    q, k, v = (state[name].detach() for name in ("queries", "keys", "values"))
    dtype, device = q.dtype, q.device
    (batch, length, heads, width), (total, groups) = q.shape, k.shape[1:3]
    shared, window, sinks = heads // groups, case["window"], min(case["sinks"], total)
    size = max(16, min(window, total))
    blocks = -(-total // size)
    room = blocks * size
    if valid is None:
        valid = torch.ones(batch, total, dtype=torch.bool, device=device)

    def full(t):  # [B, room, G, W] in 32 bits, behind each position's place
        wide = torch.zeros(batch, room, t.shape[2], width, device=device)
        wide[:, total - t.shape[1]:total] = t.float()
        return wide

    taken = torch.zeros(batch, room, dtype=torch.bool, device=device)
    taken[:, :total] = valid
    q, k, v = full(q), full(k), full(v)
    scale = 1.0 / math.sqrt(width)
    # rows: the heads that share a key head, then the block's positions
    rows = _banded(q.reshape(batch, room, groups, shared * width), blocks, size, carry=False)
    rows = rows.reshape(batch, groups, blocks, size, shared, width).transpose(3, 4).reshape(batch, groups, blocks, shared * size, width)
    first_k = k[:, None, :sinks].permute(0, 3, 1, 2, 4).expand(-1, -1, blocks, -1, -1)
    first_v = v[:, None, :sinks].permute(0, 3, 1, 2, 4).expand(-1, -1, blocks, -1, -1)
    kk = torch.cat([_banded(k, blocks, size), first_k], dim=3)
    vv = torch.cat([_banded(v, blocks, size), first_v], dim=3)
    place = torch.arange(room, device=device).reshape(blocks, size)
    column = torch.cat([place - size, place], dim=1)
    late = torch.arange(sinks, device=device).expand(blocks, -1)
    i, j = place[:, :, None], column[:, None, :]
    band = (j >= 0) & (j <= i) & ((i - j < window) | (j < sinks))
    # a sink within the block's band counts there, one before it in a column of its own
    before = (late[:, None, :] < column[:, None, :1]).expand(-1, size, -1)
    seen = torch.cat([band, before], dim=2)
    shown = torch.cat([torch.where(column >= 0, taken[:, column.clamp(min=0)], False), taken[:, None, :sinks].expand(-1, blocks, -1)], dim=2)
    mask = seen[None] & shown[:, :, None, :] & taken[:, :room].reshape(batch, blocks, size)[..., None]
    mask = mask[:, None, :, None].expand(-1, -1, -1, shared, -1, -1).reshape(batch, 1, blocks, shared * size, -1)
    s = torch.matmul(rows * scale, kk.transpose(3, 4)).masked_fill_(~mask, float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    p = s.sub_(torch.where(top > float("-inf"), top, 0.0)).exp_()
    p /= p.sum(dim=-1, keepdim=True).clamp(min=1e-30)

    def back(t):  # [B, G, blocks, shared * size, W] -> [B, length, heads, W]
        t = t.reshape(batch, groups, blocks, shared, size, width).permute(0, 2, 4, 1, 3, 5)
        return t.reshape(batch, room, heads, width)[:, total - length:total]

    out = {"out": back(torch.matmul(p, vv)).to(dtype)}
    if not case["train"]:
        return out
    up = _banded(full(state["d_out"]).reshape(batch, room, groups, shared * width), blocks, size, carry=False)
    up = up.reshape(batch, groups, blocks, size, shared, width).transpose(3, 4).reshape(batch, groups, blocks, shared * size, width)

    def gathered(t):  # the gradients of _banded keys and of the sinks behind them
        whole = _unbanded(t[:, :, :, :2 * size], size)
        whole[:, :sinks] += t[:, :, :, 2 * size:].sum(dim=2).permute(0, 2, 1, 3)
        return whole[:, :total].to(dtype)

    out["d_values"] = gathered(torch.matmul(p.transpose(3, 4), up))
    d = torch.matmul(up, vv.transpose(3, 4))
    d = p * (d - (p * d).sum(dim=-1, keepdim=True))
    out["d_queries"] = (back(torch.matmul(d, kk)) * scale).to(dtype)
    out["d_keys"] = gathered(torch.matmul(d.transpose(3, 4), rows * scale))
    return out


def _quantised(x, kind, stored):
    """Codes [..., stored], as bytes, and scales [...] of rows [..., width] in 32 bits: the largest value gets the largest code."""

    fine = torch.isfinite(x).all(dim=-1)
    scale = (x.abs().amax(dim=-1) / LIMIT[kind]).clamp(min=SMALLEST_SCALE)
    codes = torch.where(fine[..., None], x / scale[..., None], 0.0)
    codes = codes.round().clamp(-127.0, 127.0) if kind == "int8" else codes
    codes = torch.cat([codes, torch.zeros(*codes.shape[:-1], stored - codes.shape[-1], device=x.device)], dim=-1)
    return codes.to(CODES[kind]).view(torch.uint8), torch.where(fine, scale, float("nan"))


def _floats(codes, case):
    """What bytes of a cache stand for before their scale."""

    return codes.view(CODES[case["codes"]]).float()


def _plain_cache(state):
    case, lengths, after = state["case"], state["lengths"], state["after"]
    window, sinks, width, stored = case["window"], case["sinks"], case["width"], _stored(case["width"])
    device, batch = lengths.device, case["batch"]
    # the entry that every slot holds afterwards: the sinks their own, the ring the last one of its remainder
    slot = torch.arange(window + sinks, device=device)[None]
    last = after[:, None] - 1
    entry = torch.where(slot < sinks, slot, last - (last - slot) % window)
    fresh = (entry >= lengths[:, None]) & (entry <= last)
    source = torch.where(fresh, entry - lengths[:, None], 0)
    rows = torch.arange(batch, device=device)[:, None]
    out = {}
    # read back: the sinks, then the last `window` entries in their order
    place = torch.cat([torch.arange(sinks, device=device).expand(batch, -1),
                       after[:, None] - window + torch.arange(window, device=device)], dim=1)
    first = torch.arange(window + sinks, device=device)[None] < sinks
    present = torch.where(first, place < after[:, None], place >= sinks)
    at = torch.where(first, place, sinks + (place - sinks) % window)
    for name in ("keys", "values"):
        codes, scales = state[name].view(torch.uint8), state[name[:-1] + "_scales"]
        new, new_scales = _quantised(state["new_" + name].float(), case["codes"], stored)
        new, new_scales = new[rows, source].transpose(1, 2), new_scales[rows, source].transpose(1, 2)
        codes.copy_(torch.where(fresh[:, None, :, None], new, codes))
        scales.copy_(torch.where(fresh[:, None], new_scales, scales))
        wide = _floats(codes.transpose(1, 2)[rows, at], case)[..., :width] * scales.transpose(1, 2)[rows, at][..., None]
        out[name] = torch.where(present[:, :, None, None], wide, 0.0).to(DTYPES[case["dtype"]])
    return out | {"present": present}


def _plain_step(state):
    case, lengths, active = state["case"], state["lengths"], state["active"]
    window, sinks, width, stored = case["window"], case["sinks"], case["width"], _stored(case["width"])
    batch, groups, slots = case["batch"], case["groups"], window + sinks
    device, q = lengths.device, state["queries"]
    if active is None:
        active = torch.ones(batch, dtype=torch.bool, device=device)
    rows = torch.arange(batch, device=device)
    slot = torch.where(lengths < sinks, lengths, sinks + (lengths - sinks) % window)
    wide = {}
    for name in ("keys", "values"):
        codes, scales = state[name].view(torch.uint8), state[name[:-1] + "_scales"]
        new, new_scales = _quantised(state["new_" + name].float(), case["codes"], stored)
        old, old_scales = codes[rows, :, slot], scales[rows, :, slot]
        codes[rows, :, slot] = torch.where(active[:, None, None], new, old)
        scales[rows, :, slot] = torch.where(active[:, None], new_scales, old_scales)
        wide[name] = _floats(codes, case)[..., :width] * scales[..., None]
    held = torch.arange(slots, device=device)[None] < torch.where(active, lengths + 1, 0)[:, None]
    qq = q.float().reshape(batch, groups, -1, width) * (1.0 / math.sqrt(width))
    s = torch.matmul(qq, wide["keys"].transpose(2, 3)).masked_fill(~held[:, None, None], float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top > float("-inf"), top, 0.0))
    p = p / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    shown = torch.where(held[:, None, :, None], wide["values"], 0.0)
    out = {"out": torch.matmul(p, shown).reshape(q.shape).to(q.dtype)}
    return out | {name: state[name] for name in ("keys", "key_scales", "values", "value_scales")}


def _plain_sample(state):
    case, z = state["case"], state["logits"].double()
    rows, vocab = z.shape
    if case["exclude"] >= 0:
        z = torch.where(torch.arange(vocab, device=z.device) == case["exclude"], float("-inf"), z)
    ordered = torch.sort(z, dim=-1, descending=True)[0]
    if 0 < case["top_k"] < vocab:
        z = torch.where(z < ordered[:, case["top_k"] - 1:case["top_k"]], float("-inf"), z)
        ordered = torch.sort(z, dim=-1, descending=True)[0]
    top = ordered[:, :1]
    w = torch.where(z > float("-inf"), torch.exp((z - top) / case["temperature"]), 0.0)
    kept = w >= case["min_p"]
    if case["top_p"] < 1.0:
        # the mass of all strictly better ones decides, so equals stay together
        mass = torch.cumsum(torch.where(ordered > float("-inf"), torch.exp((ordered - top) / case["temperature"]), 0.0), dim=-1)
        first = torch.searchsorted(-ordered, (-z).contiguous())
        better = torch.where(first > 0, mass.gather(1, (first - 1).clamp(min=0)), 0.0)
        kept &= better < case["top_p"] * mass[:, -1:]
    w = torch.where(kept, w, 0.0)
    mass = torch.cumsum(w, dim=-1)
    beyond = (mass > state["uniforms"].double()[:, None] * mass[:, -1:]).to(torch.int32)
    out = {"ids": torch.argmax(beyond, dim=-1, keepdim=True)}
    if case["full"]:
        out["probabilities"] = (w / w.sum(dim=-1, keepdim=True)).float()
    return out


# ------------------------------------------------------ the package's calls ---


def _own_attend(state):
    from koemi_amd import window

    case = state["case"]
    leaves = (state["queries"], state["keys"], state["values"])
    y = window.window_attention(*leaves, state["valid"], window=case["window"], sinks=case["sinks"])
    out = {"out": y}
    if case["train"]:
        out["d_queries"], out["d_keys"], out["d_values"] = torch.autograd.grad(y, leaves, state["d_out"])
    return out


def _own_cache_of(state):
    from koemi_amd import window

    case = state["case"]
    return window.WindowCache(state["keys"], state["key_scales"], state["values"], state["value_scales"],
                              width=case["width"], window=case["window"], sinks=case["sinks"])


def _own_cache(state):
    from koemi_amd import window

    cache = _own_cache_of(state)
    window.window_cache_write(cache, state["new_keys"], state["new_values"], state["lengths"], state["counts"])
    keys, values, present = window.window_cache_entries(cache, state["after"], dtype=DTYPES[state["case"]["dtype"]])
    return {"keys": keys, "values": values, "present": present}


def _own_step(state):
    from koemi_amd import window

    cache = _own_cache_of(state)
    y = window.window_cache_step(cache, state["queries"], state["new_keys"], state["new_values"], state["lengths"],
                                 state["active"])
    return {"out": y} | {name: state[name] for name in ("keys", "key_scales", "values", "value_scales")}


def _own_sample(state):
    from koemi_amd import sampling

    case = state["case"]
    got = sampling.sample_tokens(
        state["logits"], state["uniforms"], temperature=case["temperature"], top_k=case["top_k"] or None,
        top_p=case["top_p"], min_p=case["min_p"], exclude=case["exclude"] if case["exclude"] >= 0 else None,
        with_probabilities=case["full"])
    return {"ids": got[0], "probabilities": got[1]} if case["full"] else {"ids": got}


def run(state):
    op = state["case"]["op"]
    if own:
        if str(_PACKAGE) not in sys.path:
            sys.path.insert(0, str(_PACKAGE))
        return {"attend": _own_attend, "cache": _own_cache, "step": _own_step, "sample": _own_sample}[op](state)
    with torch.no_grad():
        return {"attend": _plain_attend, "cache": _plain_cache, "step": _plain_step, "sample": _plain_sample}[op](state)


def _pairs(first, last, window, sinks):
    """Visible (query, key) pairs of the positions first .. last - 1."""

    def upto(n):  # of positions 0 .. n - 1
        ramp = min(n, window)
        total = ramp * (ramp + 1) // 2 + (n - ramp) * window
        late = max(0, n - window)  # positions whose window has left position 0
        ramp = min(late, sinks)
        return total + ramp * (ramp + 1) // 2 + (late - ramp) * sinks

    return upto(last) - upto(first)


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "sample":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * (size + (4 if case["full"] else 0)) + case["rows"] * 12, "flops": cells * 20}
    if case["op"] == "attend":
        total, half = case["length"] + case["carried"], 0.5 if case["padded"] else 1.0  # rows end anywhere
        pairs = case["batch"] * case["heads"] * _pairs(case["carried"], total, case["window"], case["sinks"]) * half
        rows = case["batch"] * case["width"] * size
        moved = rows * (2 * case["length"] * case["heads"] + 2 * total * case["groups"])
        if case["train"]:  # d_out and the three gradients
            moved += rows * (2 * case["length"] * case["heads"] + 2 * total * case["groups"])
        return {"bytes": moved, "flops": int(pairs * case["width"] * (14 if case["train"] else 4))}
    slots = case["window"] + case["sinks"]
    entry = _stored(case["width"]) + 4
    if case["op"] == "cache":
        new = min(case["length"], slots) * (0.5 if case["padded"] else 1.0)
        heads = case["batch"] * case["groups"] * 2
        return {"bytes": int(heads * (new * (case["width"] * size + entry) + slots * (entry + case["width"] * size))),
                "flops": int(heads * case["width"] * (new * 4 + slots))}
    rows = case["batch"] * (0.85 if case["padded"] else 1.0)
    moved = rows * (case["groups"] * 2 * slots * entry + 2 * (case["heads"] + case["groups"]) * case["width"] * size)
    return {"bytes": int(moved), "flops": int(rows * case["heads"] * slots * case["width"] * 4)}


# ------------------------------------------------------------------- 64 bits ---


def _exact_attend(state):
    case = state["case"]
    q, k, v = (state[name].detach().double() for name in ("queries", "keys", "values"))
    (batch, length, heads, width), (total, groups) = q.shape, k.shape[1:3]
    carried, shared, train = total - length, heads // groups, case["train"]
    out = torch.zeros_like(q)
    d_q, d_k, d_v = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    step = 512
    for b in range(batch):
        # head h reads key head h // shared
        kb, vb = k[b].transpose(0, 1).repeat_interleave(shared, dim=0), v[b].transpose(0, 1).repeat_interleave(shared, dim=0)
        for begin in range(0, length, step):
            end = min(length, begin + step)
            i = torch.arange(carried + begin, carried + end, device=q.device)
            low = max(0, carried + begin - case["window"] + 1)
            j = torch.cat([torch.arange(min(low, case["sinks"]), device=q.device),
                           torch.arange(low, carried + end, device=q.device)])
            see = (j[None] <= i[:, None]) & ((j[None] > i[:, None] - case["window"]) | (j[None] < case["sinks"]))
            if state["valid"] is not None:
                see = see & state["valid"][b, j][None] & state["valid"][b, i][:, None]
            qb, kj, vj = q[b, begin:end].transpose(0, 1), kb[:, j], vb[:, j]
            s = torch.matmul(qb, kj.transpose(1, 2)) / math.sqrt(width)
            p = torch.softmax(s.masked_fill(~see, float("-inf")), dim=-1)
            p = torch.where(see.any(dim=-1)[None, :, None], p, torch.zeros_like(p))
            out[b, begin:end] = torch.matmul(p, vj).transpose(0, 1)
            if train:
                up = state["d_out"][b, begin:end].double().transpose(0, 1)
                g = torch.matmul(up, vj.transpose(1, 2))
                g = p * (g - (up * out[b, begin:end].transpose(0, 1)).sum(dim=-1, keepdim=True)) / math.sqrt(width)
                d_q[b, begin:end] = torch.matmul(g, kj).transpose(0, 1)
                for grad, part in ((d_k, torch.matmul(g.transpose(1, 2), qb)), (d_v, torch.matmul(p.transpose(1, 2), up))):
                    grad[b].index_add_(0, j, part.reshape(groups, shared, j.numel(), width).sum(dim=1).transpose(0, 1))
    if not train:
        return {"out": out}
    return {"out": out, "d_queries": d_q, "d_keys": d_k, "d_values": d_v}


def _stands_for(x, kind):
    """The values that the codes of rows [..., width] stand for, the codes chosen in 64 bits but for the scale, which is held in 32."""

    x = x.double()
    scale = torch.clamp(x.abs().amax(dim=-1, keepdim=True) / LIMIT[kind], min=SMALLEST_SCALE).float().double()
    if kind == "int8":
        return torch.clamp(torch.round(x / scale), -127, 127) * scale, scale
    # steps of an eighth of the power of two below, none under 2^-9
    ratio = (x / scale).clamp(-448, 448)
    power = torch.floor(torch.log2(ratio.abs().clamp(min=2.0 ** -6)))
    unit = torch.exp2(power - 3)
    return torch.round(ratio / unit) * unit * scale, scale


def _exact_cache(state):
    case, window, sinks = state["case"], state["case"]["window"], state["case"]["sinks"]
    batch, groups, width, slots = case["batch"], case["groups"], case["width"], window + sinks
    out = {"present": torch.zeros(batch, slots, dtype=torch.bool, device="cuda")}
    for name in ("keys", "values"):
        held = state[name].double()[..., :width] * state[name[:-1] + "_scales"].double()[..., None]
        new = _stands_for(state["new_" + name], case["codes"])[0]
        got = torch.zeros(batch, slots, groups, width, dtype=torch.float64, device="cuda")
        for b in range(batch):
            n0, n1 = int(state["lengths"][b]), int(state["after"][b])
            entries = list(range(min(sinks, n1))) + list(range(max(sinks, n1 - window), n1))
            target = [e if e < sinks else slots - n1 + e for e in entries]
            fresh = [(t, e - n0) for t, e in zip(target, entries) if e >= n0]
            old = [(t, e if e < sinks else sinks + (e - sinks) % window) for t, e in zip(target, entries) if e < n0]
            out["present"][b, target] = True
            if fresh:
                got[b, [t for t, _ in fresh]] = new[b, [e for _, e in fresh]]
            if old:
                got[b, [t for t, _ in old]] = held[b, :, [s for _, s in old]].transpose(0, 1)
        out[name] = got
    return out


def _exact_step(state):
    case, window, sinks = state["case"], state["case"]["window"], state["case"]["sinks"]
    batch, groups, width, slots = case["batch"], case["groups"], case["width"], window + sinks
    q = state["queries"].double().reshape(batch, groups, -1, width)
    out = torch.zeros_like(q)
    scales = {name: state[name[:-1] + "_scales"].double() for name in ("keys", "values")}
    fresh = {name: _stands_for(state["new_" + name], case["codes"]) for name in ("keys", "values")}
    for b in range(batch):
        if state["active"] is not None and not bool(state["active"][b]):
            continue
        n = int(state["lengths"][b])
        slot = n if n < sinks else sinks + (n - sinks) % window
        wide = {}
        for name in ("keys", "values"):
            wide[name] = state[name][b, ..., :width].double() * scales[name][b][..., None]
            wide[name][:, slot] = fresh[name][0][b]
            scales[name][b, :, slot] = fresh[name][1][b, :, 0]
        kept = min(n + 1, slots)
        p = torch.softmax(torch.matmul(q[b], wide["keys"][:, :kept].transpose(1, 2)) / math.sqrt(width), dim=-1)
        out[b] = torch.matmul(p, wide["values"][:, :kept])
    return {"out": out.reshape(state["queries"].shape), "keys": None, "values": None, "key_scales": scales["keys"],
            "value_scales": scales["values"]}


def _exact_sample(state):
    case = state["case"]
    logits = state["logits"].double()
    rows, vocab = logits.shape
    ids = torch.zeros(rows, 1, dtype=torch.int64, device="cuda")
    full = torch.zeros_like(logits) if case["full"] else None
    for r in range(rows):
        z = logits[r].clone()
        if case["exclude"] >= 0:
            z[case["exclude"]] = -math.inf
        levels, index, count = torch.unique(-z, return_inverse=True, return_counts=True)
        levels = -levels  # falling
        if case["top_k"]:
            ahead = count.cumsum(0) - count
            levels[ahead >= case["top_k"]] = -math.inf
        weight = torch.exp((levels - levels[0]) / case["temperature"])
        mass = (weight * count).cumsum(0)
        keep = weight >= max(case["min_p"], 5e-324)
        if case["top_p"] < 1.0:
            keep &= torch.cat([mass.new_zeros(1), mass[:-1]]) < case["top_p"] * mass[-1]
        p = torch.where(keep, weight, 0.0)[index]
        p = p / p.sum()
        ids[r, 0] = min(vocab - 1, int(torch.searchsorted(p.cumsum(0), state["uniforms"][r].double(), right=True)))
        if full is not None:
            full[r] = p
    return {"ids": ids, "probabilities": full} if case["full"] else {"ids": ids}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"attend": _exact_attend, "cache": _exact_cache, "step": _exact_step, "sample": _exact_sample}[case["op"]](state)
