"""Timed cases of the operators that train a HERM layer's gates, router and experts.

Families (``op``):

* ``recurrence``: the bounded recurrent state from stacked gate pre-activations
  (``recurrent.gated_recurrence``): states and final state, with ``train`` also
  the gradients of the pre-activations and of the initial state;
* ``route``: the learned softmax top-k route with its per-expert counts and
  balance loss (``moe.route_topk_balanced``), with ``train`` also the gradient of
  the logits through the weights and the loss;
* ``experts``: the gated feed-forward experts of every token's route, weighted
  and summed (``moe.expert_mixture``), with ``train`` also the gradients of the
  context, the route's weights and all six parameters.

``run`` computes each in plain torch, in 32 bits and rounded once at the end;
with ``own`` set it calls the package's fronts. ``exact`` restates the
definitions in 64 bits: the recurrence position by position, the route from
sorted logits, the experts one by one.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = Path(__file__).resolve().parent.parent / "koemi-5hom_amd"

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
MIN_RETENTION = 2.0 ** -8
RETENTION_SPAN = 1.0 - 2.0 ** -7


def listed():
    return [
        # one generated position at the serving batch: launch latency
        {"name": "recurrence_step_64x1024", "op": "recurrence", "batch": 64, "length": 1, "width": 1024, "dtype": "bf16",
         "padded": False, "train": False},
        # a training batch at the package's headline width, ragged rows padded to one length
        {"name": "recurrence_train_8x2048x1024", "op": "recurrence", "batch": 8, "length": 2048, "width": 1024,
         "dtype": "bf16", "padded": True, "train": True},
        # one long document in full precision: few columns, many positions
        {"name": "recurrence_train_1x32768x512", "op": "recurrence", "batch": 1, "length": 32768, "width": 512,
         "dtype": "fp32", "padded": False, "train": True},
        # odd sizes in half precision
        {"name": "recurrence_train_5x777x300", "op": "recurrence", "batch": 5, "length": 777, "width": 300, "dtype": "fp16",
         "padded": True, "train": True},
        # the route of one generated position at the serving batch
        {"name": "route_step_64x16", "op": "route", "tokens": 64, "experts": 16, "top_k": 2, "dtype": "fp32",
         "padded": False, "masked": False, "train": False},
        # the route of a training batch over the package's sixteen experts
        {"name": "route_train_16384x16", "op": "route", "tokens": 16384, "experts": 16, "top_k": 2, "dtype": "fp32",
         "padded": True, "masked": False, "train": True},
        # many experts, several choices, half the logits' bytes: bandwidth
        {"name": "route_train_131072x128", "op": "route", "tokens": 131072, "experts": 128, "top_k": 4, "dtype": "bf16",
         "padded": False, "masked": False, "train": True},
        # an odd number of experts, some of them switched off by a logit of minus infinity
        {"name": "route_train_3000x37", "op": "route", "tokens": 3000, "experts": 37, "top_k": 3, "dtype": "fp16",
         "padded": True, "masked": True, "train": True},
        # the experts of one generated position at the serving batch: the weights are read for a few rows
        {"name": "experts_step_64", "op": "experts", "tokens": 64, "width": 1024, "hidden": 2048, "experts": 16,
         "top_k": 2, "dtype": "bf16", "padded": False, "train": False},
        # the expert layer of a training batch at the package's headline sizes
        {"name": "experts_train_16384", "op": "experts", "tokens": 16384, "width": 1024, "hidden": 2048, "experts": 16,
         "top_k": 2, "dtype": "bf16", "padded": True, "train": True},
        # a ragged batch in half precision, sizes off the tiles
        {"name": "experts_train_3000_fp16", "op": "experts", "tokens": 3000, "width": 768, "hidden": 2000, "experts": 12,
         "top_k": 2, "dtype": "fp16", "padded": True, "train": True},
        # a small model in full precision with odd sizes, one choice per token
        {"name": "experts_train_500_fp32", "op": "experts", "tokens": 500, "width": 201, "hidden": 333, "experts": 8,
         "top_k": 1, "dtype": "fp32", "padded": False, "train": True},
    ]


def _log(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""

    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("recurrence", "route", "experts"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    padded, train = rng.random() < 0.5, rng.random() < 0.75
    if op == "recurrence":
        width = rng.choice((_log(rng, 8, 2048), 64 * rng.randint(1, 24)))
        length = _log(rng, 1, 32768)
        batch = _log(rng, 1, max(1, min(64, (1 << 24) // (width * length))))
        return {"op": op, "batch": batch, "length": length, "width": width, "dtype": dtype, "padded": padded, "train": train}
    if op == "route":
        experts = _log(rng, 2, 512)
        return {"op": op, "tokens": _log(rng, 1, min(131072, (1 << 24) // experts)), "experts": experts,
                "top_k": rng.randint(1, min(8, experts)), "dtype": dtype, "padded": padded,
                "masked": rng.random() < 0.3, "train": train}
    if rng.random() < 0.5:  # the sizes that models are made of, else any
        width, hidden = 64 * rng.randint(2, 20), 64 * rng.randint(2, 36)
    else:
        width, hidden = _log(rng, 48, 1100), _log(rng, 48, 2100)
    experts = _log(rng, 1, 32)
    most = 16384 if dtype == "bf16" and width % 64 == 0 and hidden % 64 == 0 else 3000
    return {"op": op, "tokens": _log(rng, 1, most), "width": width, "hidden": hidden, "experts": experts,
            "top_k": rng.randint(1, min(2, experts)), "dtype": dtype, "padded": padded, "train": train}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 40) + 17)


def _normal(gen, *shape, dtype=torch.float32, scale=1.0, mean=0.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale + mean).to(dtype)


def _leaf(tensor, train):
    return tensor.requires_grad_() if train else tensor


def prepare(case, seed):
    gen = _generator(seed)
    dtype, train = DTYPES[case["dtype"]], case["train"]
    state = {"case": case}
    if case["op"] == "recurrence":
        batch, length, width = case["batch"], case["length"], case["width"]
        # retentions spread between short and long memories, candidates of order one
        z = torch.cat([_normal(gen, batch, length, width, scale=1.5, mean=1.0), _normal(gen, batch, length, width)], dim=-1)
        state["z"] = _leaf(z.to(dtype), train)
        state["initial"] = _leaf(_normal(gen, batch, width, scale=0.5), train)
        state["valid"] = None
        if case["padded"]:  # rows end at lengths of their own
            ends = torch.randint(0, length + 1, (batch,), device="cuda", generator=gen)
            state["valid"] = torch.arange(length, device="cuda")[None, :] < ends[:, None]
        if train:
            state["d_states"] = _normal(gen, batch, length, width, dtype=dtype)
            state["d_final"] = _normal(gen, batch, width)
        return state
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    valid = torch.ones(tokens, dtype=torch.bool, device="cuda")
    if case["padded"]:
        valid = torch.rand(tokens, device="cuda", generator=gen) < 0.85
    state["valid"] = valid
    # some experts are liked more than others
    logits = _normal(gen, tokens, experts) + _normal(gen, experts, scale=0.3)
    if case["op"] == "route":
        if case["masked"]:
            logits = logits.masked_fill(torch.rand(experts, device="cuda", generator=gen) < 0.2, float("-inf"))
        state["logits"] = _leaf(logits.to(dtype), train)
        if train:
            state["d_weights"] = _normal(gen, tokens, top_k)
            state["d_loss"] = torch.full((), 0.01 * tokens, device="cuda")
        return state
    width, hidden = case["width"], case["hidden"]
    weights, assignments = torch.softmax(logits, dim=-1).topk(top_k, dim=-1)
    state["assignments"] = assignments.masked_fill(~valid[:, None], -1).contiguous()
    state["weights"] = _leaf(weights.masked_fill(~valid[:, None], 0.0).contiguous(), train)
    counts = torch.bincount(assignments[valid].reshape(-1), minlength=experts)
    state["capacity"] = max(1, int(counts.max()))  # rows of the plain form's largest expert
    state["context"] = _leaf(_normal(gen, tokens, width, dtype=dtype), train)
    shapes = {"gate_w": (experts, hidden, width), "gate_b": (experts, hidden), "value_w": (experts, hidden, width),
              "value_b": (experts, hidden), "output_w": (experts, width, hidden), "output_b": (experts, width)}
    state["params"] = {
        name: _leaf(_normal(gen, *shape, dtype=dtype, scale=1.0 / math.sqrt(shape[-1]) if len(shape) == 3 else 0.1), train)
        for name, shape in shapes.items()}
    if train:
        state["d_out"] = _normal(gen, tokens, width, dtype=dtype)
    return state


# ------------------------------------------------------------- plain forms ---


def _scan(a, b, reverse=False):
    """h_t = a_t h_{t-1} + b_t from 0 along dimension 1 (from the end with
    ``reverse``) by doubling: after step d each position holds the map of the
    2 d positions up to it."""

    if reverse:
        return _scan(a.flip(1), b.flip(1)).flip(1)
    distance = 1
    while distance < a.shape[1]:
        b = torch.cat([b[:, :distance], a[:, distance:] * b[:, :-distance] + b[:, distance:]], dim=1)
        a = torch.cat([a[:, :distance], a[:, distance:] * a[:, :-distance]], dim=1)
        distance *= 2
    return b


def _plain_recurrence(state):
    z, valid, initial = state["z"].detach(), state["valid"], state["initial"].detach()
    r, c = z.float().chunk(2, dim=-1)
    s, t = 1.0 / (1.0 + torch.exp(-r)), torch.tanh(c)
    kept = MIN_RETENTION + RETENTION_SPAN * s
    a, b = kept, (1.0 - kept) * t
    if valid is not None:
        a = torch.where(valid[..., None], a, 1.0)
        b = torch.where(valid[..., None], b, 0.0)
    first = torch.cat([a[:, :1] * initial[:, None] + b[:, :1], b[:, 1:]], dim=1)
    states = _scan(a, first)
    out = {"states": states.to(z.dtype), "final": states[:, -1]}
    if state["case"]["train"]:
        upstream = state["d_states"].float()
        upstream = torch.cat([upstream[:, :-1], upstream[:, -1:] + state["d_final"][:, None]], dim=1)
        after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
        g = _scan(after, upstream, reverse=True)
        before = torch.cat([initial[:, None], states[:, :-1]], dim=1)
        d_r = g * (before - t) * RETENTION_SPAN * s * (1.0 - s)
        d_c = g * (1.0 - kept) * (1.0 - t * t)
        d_z = torch.cat([d_r, d_c], dim=-1)
        if valid is not None:
            d_z = torch.where(valid[..., None], d_z, 0.0)
        out["d_z"], out["d_initial"] = d_z.to(z.dtype), a[:, 0] * g[:, 0]
    return out


def _plain_route(state):
    logits, valid, top_k = state["logits"].detach(), state["valid"], state["case"]["top_k"]
    experts = logits.shape[-1]
    z = logits.float()
    valid = valid & (z > float("-inf")).any(dim=-1)
    e = torch.exp(z - z.amax(dim=-1, keepdim=True))
    p = torch.where(valid[:, None], e / e.sum(dim=-1, keepdim=True), 0.0)
    best, order = torch.sort(z, dim=-1, descending=True, stable=True)
    chosen = valid[:, None] & (best[:, :top_k] > float("-inf"))
    assignments = torch.where(chosen, order[:, :top_k], -1)
    slot = assignments.clamp(min=0)
    weights = torch.where(chosen, p.gather(1, slot), 0.0)
    mass, valid_count = p.sum(dim=0), valid.sum().float()
    counts = torch.zeros(experts, device=z.device).index_add_(0, slot.reshape(-1), chosen.reshape(-1).float())
    load = counts / counts.sum().clamp(min=1.0)
    loss = experts * (mass / valid_count.clamp(min=1.0) * load).sum()
    out = {"assignments": assignments, "weights": weights, "mass": mass, "counts": counts, "valid": valid_count, "loss": loss}
    if state["case"]["train"]:
        g = (state["d_loss"] * experts * load / valid_count.clamp(min=1.0)).expand_as(p)
        g = g.scatter_add(1, slot, torch.where(chosen, state["d_weights"], 0.0))
        out["d_logits"] = (p * (g - (p * g).sum(dim=-1, keepdim=True))).to(logits.dtype)
    return out


def _plain_experts(state):
    case, x, w = state["case"], state["context"].detach(), state["weights"].detach()
    p = {name: t.detach().float() for name, t in state["params"].items()}
    (tokens, width), (experts, top_k), room = x.shape, (case["experts"], case["top_k"]), state["capacity"]
    # every expert's pairs in rows of their own, room rows an expert; one spare row takes the pairs of no expert
    expert = state["assignments"].reshape(-1)
    expert = torch.where(expert < 0, experts, expert)
    key, order = torch.sort(expert, stable=True)
    starts = torch.searchsorted(key, torch.arange(experts + 1, device=x.device))
    row = torch.where(key < experts, key * room + torch.arange(key.numel(), device=x.device) - starts[key], experts * room)
    rows = torch.empty_like(row).scatter_(0, order, row)  # pair -> row
    used = torch.zeros(experts * room + 1, device=x.device)
    used[rows] = 1.0
    used[-1] = 0.0
    token = torch.zeros(experts * room + 1, dtype=torch.int64, device=x.device)
    token[rows] = torch.arange(tokens, device=x.device).repeat_interleave(top_k)
    weight = torch.zeros(experts * room + 1, device=x.device)
    weight[rows] = w.reshape(-1)
    used, token, weight = used[:-1, None], token[:-1], weight[:-1, None] * used[:-1, None]
    grouped = lambda t: t.reshape(experts, room, -1)  # noqa: E731

    def pairs(t):
        flat = torch.cat([t.reshape(experts * room, -1), torch.zeros_like(t[:1, 0])])
        return flat[rows].reshape(tokens, top_k, -1)

    xe = grouped(x.float()[token] * used)
    g = torch.bmm(xe, p["gate_w"].transpose(1, 2)) + p["gate_b"][:, None]
    v = torch.bmm(xe, p["value_w"].transpose(1, 2)) + p["value_b"][:, None]
    s = 1.0 / (1.0 + torch.exp(-g))
    h = g * s * v
    y = torch.bmm(h, p["output_w"].transpose(1, 2)) + p["output_b"][:, None]
    out = {"out": (pairs(y) * w[..., None]).sum(dim=1).to(x.dtype)}
    if case["train"]:
        d_out = state["d_out"].float()
        d_y = grouped(d_out[token] * weight)
        d_h = torch.bmm(d_y, p["output_w"])
        d_g, d_v = d_h * v * s * (1.0 + g * (1.0 - s)), d_h * g * s
        d_x = torch.bmm(d_g, p["gate_w"]) + torch.bmm(d_v, p["value_w"])
        out["d_weights"] = (pairs(y) * d_out[:, None]).sum(dim=-1)
        out["d_context"] = pairs(d_x).sum(dim=1).to(x.dtype)
        grads = {"gate_w": torch.bmm(d_g.transpose(1, 2), xe), "gate_b": d_g.sum(dim=1),
                 "value_w": torch.bmm(d_v.transpose(1, 2), xe), "value_b": d_v.sum(dim=1),
                 "output_w": torch.bmm(d_y.transpose(1, 2), h), "output_b": d_y.sum(dim=1)}
        out |= {"d_" + name: t.to(x.dtype) for name, t in grads.items()}
    return out


# ------------------------------------------------------ the package's calls ---


def _own_recurrence(state):
    from koemi_amd import recurrent

    states, final = recurrent.gated_recurrence(state["z"], state["valid"], state["initial"])
    out = {"states": states, "final": final}
    if state["case"]["train"]:
        out["d_z"], out["d_initial"] = torch.autograd.grad(
            (states, final), (state["z"], state["initial"]), (state["d_states"], state["d_final"]))
    return out


def _own_route(state):
    from koemi_amd import moe

    assignments, weights, statistics = moe.route_topk_balanced(state["logits"], state["valid"], top_k=state["case"]["top_k"])
    loss = statistics.balance_loss
    out = {"assignments": assignments, "weights": weights, "mass": statistics.probability_mass,
           "counts": statistics.assignment_counts, "valid": statistics.valid_count, "loss": loss}
    if state["case"]["train"]:
        out["d_logits"], = torch.autograd.grad((weights, loss), (state["logits"],), (state["d_weights"], state["d_loss"]))
    return out


def _own_experts(state):
    from koemi_amd import moe

    names = ("gate_w", "gate_b", "value_w", "value_b", "output_w", "output_b")
    params = [state["params"][name] for name in names]
    y = moe.expert_mixture(state["context"], state["assignments"], state["weights"], state["valid"], *params, validate=False)
    out = {"out": y}
    if state["case"]["train"]:
        grads = torch.autograd.grad(y, (state["weights"], state["context"], *params), state["d_out"])
        out |= {"d_" + name: t for name, t in zip(("weights", "context", *names), grads)}
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        if str(_PACKAGE) not in sys.path:
            sys.path.insert(0, str(_PACKAGE))
        return {"recurrence": _own_recurrence, "route": _own_route, "experts": _own_experts}[op](state)
    with torch.no_grad():
        return {"recurrence": _plain_recurrence, "route": _plain_route, "experts": _plain_experts}[op](state)


def work(case):
    size, train = SIZE[case["dtype"]], case["train"]
    if case["op"] == "recurrence":
        rows, width = case["batch"] * case["length"], case["width"]
        edge = case["batch"] * width * 4
        moved = rows * width * size * (6 if train else 3) + edge * (4 if train else 2)
        return {"bytes": moved + (rows if case["padded"] else 0), "flops": rows * width * (70 if train else 25)}
    if case["op"] == "route":
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        moved = tokens * (experts * size * (2 if train else 1) + 1 + top_k * (16 if train else 12)) + experts * 8
        return {"bytes": moved, "flops": tokens * experts * ((15 if train else 8) + top_k)}
    pairs = case["tokens"] * case["top_k"] * (0.85 if case["padded"] else 1.0)
    experts = min(case["experts"], max(1, round(pairs)))  # a few tokens do not reach every expert
    matrices = experts * 3 * case["width"] * case["hidden"] * size
    zeros = (case["experts"] * 3 * case["width"] * case["hidden"] * size) if train else 0
    rows = case["tokens"] * case["width"] * size
    moved = matrices + zeros + rows * (4 if train else 2) + case["tokens"] * case["top_k"] * (16 if train else 12)
    return {"bytes": int(moved), "flops": int(6 * pairs * case["width"] * case["hidden"] * (3 if train else 1))}


# ------------------------------------------------------------------- 64 bits ---


def _exact_recurrence(state):
    z, initial = state["z"].detach().double(), state["initial"].detach().double()
    batch, length, width = z.shape[0], z.shape[1], z.shape[2] // 2
    r, c = z[..., :width], z[..., width:]
    valid = state["valid"]
    kept = MIN_RETENTION + RETENTION_SPAN * torch.sigmoid(r)
    a, b = kept.clone(), (1.0 - kept) * torch.tanh(c)
    if valid is not None:
        a[~valid], b[~valid] = 1.0, 0.0
    states = torch.empty(batch, length, width, dtype=torch.float64, device=z.device)
    h = initial
    for t in range(length):
        h = torch.addcmul(b[:, t], a[:, t], h, out=states[:, t])
    out = {"states": states, "final": h}
    if state["case"]["train"]:
        upstream = state["d_states"].double()
        d_a, d_b = torch.empty_like(a), torch.empty_like(b)
        g = state["d_final"].double()
        for t in range(length - 1, -1, -1):
            g = torch.add(g, upstream[:, t], out=d_b[:, t])
            torch.mul(g, states[:, t - 1] if t else initial, out=d_a[:, t])
            g = g * a[:, t]
        # a and b by r and c: b holds (1 - kept)
        sigma, tangent = (kept - MIN_RETENTION) / RETENTION_SPAN, torch.tanh(c)
        d_r = (d_a - d_b * tangent) * RETENTION_SPAN * sigma * torch.sigmoid(-r)
        d_c = d_b * (1.0 - kept) / torch.cosh(c) ** 2
        if valid is not None:
            d_r[~valid], d_c[~valid] = 0.0, 0.0
        out["d_z"], out["d_initial"] = torch.cat([d_r, d_c], dim=-1), g
    return out


def _exact_route(state):
    z, valid, top_k = state["logits"].detach().double(), state["valid"], state["case"]["top_k"]
    train = state["case"]["train"]
    tokens, experts = z.shape
    routed = (valid & torch.isfinite(z).any(dim=-1)).nonzero().reshape(-1)
    rank = torch.argsort(z[routed], dim=-1, descending=True, stable=True)[:, :top_k]
    off = torch.isinf(torch.take_along_dim(z[routed], rank, dim=-1))
    p = torch.softmax(z[routed], dim=-1)
    assignments = torch.full((tokens, top_k), -1, dtype=torch.int64, device=z.device)
    assignments[routed] = rank.masked_fill(off, -1)
    weights = torch.zeros(tokens, top_k, dtype=torch.float64, device=z.device)
    weights[routed] = torch.take_along_dim(p, rank, dim=-1)
    mass = p.sum(dim=0)
    counts = torch.bincount(rank[~off], minlength=experts).double()
    n, total = max(int(routed.numel()), 1), max(float(counts.sum()), 1.0)
    loss = experts * torch.dot(mass / n, counts / total)
    out = {"assignments": assignments, "weights": weights, "mass": mass, "counts": counts,
           "valid": torch.tensor(float(routed.numel()), dtype=torch.float64, device=z.device), "loss": loss}
    if train:
        with torch.enable_grad():
            leaf = z[routed].clone().requires_grad_()
            q = torch.softmax(leaf, dim=-1)
            chosen = torch.take_along_dim(q, rank, dim=-1) * state["d_weights"].double()[routed].masked_fill(off, 0.0)
            total_loss = chosen.sum() + state["d_loss"].double() * experts * torch.dot(q.sum(dim=0) / n, counts / total)
            (part,) = torch.autograd.grad(total_loss, leaf)
        d_logits = torch.zeros_like(z)
        d_logits[routed] = part
        out["d_logits"] = d_logits
    return out


def _exact_experts(state):
    case = state["case"]
    x, w, assignments = state["context"].detach().double(), state["weights"].detach().double(), state["assignments"]
    p = {name: t.detach() for name, t in state["params"].items()}
    train = case["train"]
    d_out = state["d_out"].double() if train else None
    out = {"out": torch.zeros_like(x)}
    if train:
        out["d_weights"], out["d_context"] = torch.zeros_like(w), torch.zeros_like(x)
        out |= {"d_" + name: torch.zeros(t.shape, dtype=torch.float64, device=x.device) for name, t in p.items()}
    for e in range(case["experts"]):
        token, slot = (assignments == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        m = {name: t[e].double() for name, t in p.items()}
        rows, share = x[token], w[token, slot][:, None]
        with torch.enable_grad() if train else torch.no_grad():
            pre_g = (rows @ m["gate_w"].T + m["gate_b"]).detach().requires_grad_(train)
            pre_v = (rows @ m["value_w"].T + m["value_b"]).detach().requires_grad_(train)
            mid = torch.nn.functional.silu(pre_g) * pre_v
        y = mid.detach() @ m["output_w"].T + m["output_b"]
        out["out"].index_add_(0, token, share * y)
        if not train:
            continue
        up = d_out[token]
        out["d_weights"][token, slot] = (up * y).sum(dim=-1)
        up = up * share
        d_g, d_v = torch.autograd.grad(mid, (pre_g, pre_v), up @ m["output_w"])
        out["d_context"].index_add_(0, token, d_g @ m["gate_w"] + d_v @ m["value_w"])
        out["d_gate_w"][e], out["d_gate_b"][e] = d_g.T @ rows, d_g.sum(dim=0)
        out["d_value_w"][e], out["d_value_b"][e] = d_v.T @ rows, d_v.sum(dim=0)
        out["d_output_w"][e], out["d_output_b"][e] = up.T @ mid.detach(), up.sum(dim=0)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"recurrence": _exact_recurrence, "route": _exact_route, "experts": _exact_experts}[case["op"]](state)
