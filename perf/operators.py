"""Measured cases of the expert feed-forward operators and of the gated
residual norm: `route_experts`, `expert_ffn` and `sandwich_norm` of
`techjam_b200.kernels`.

`listed()` holds the cases, `draw()` makes more of the same ranges,
`prepare()` the inputs of one, `run()` one pass.  With `own` false, `run`
computes the operators from elementary torch operations in 32 bits (the
router's choices in 64, where two experts' values may lie next to each other);
with `own` true it makes the calls a program makes of this package.
`exact()` computes the same outputs in 64 bits, apart from both.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _kernels():
    import __graft_entry__

    return __graft_entry__.load_package().kernels


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _route(name, rows, experts, top_k, dtype, scoring, bias=False, groups=1, top_groups=1, group_top=1,
           renorm=True, scale=1.0, closed=0.0):
    return {"op": "route", "name": name, "rows": rows, "experts": experts, "top_k": top_k, "dtype": dtype,
            "scoring": scoring, "bias": bias, "groups": groups, "top_groups": top_groups,
            "group_top": group_top, "renorm": renorm, "scale": scale, "closed": closed}


def _ffn(name, rows, experts, top_k, d_model, ffn_dim, dtype, scoring="softmax", skew=0.5):
    return {"op": "ffn", "name": name, "rows": rows, "experts": experts, "top_k": top_k, "d_model": d_model,
            "ffn_dim": ffn_dim, "dtype": dtype, "scoring": scoring, "skew": skew}


def _norm(name, rows, d_model, dtype, kind, gate, gate_act="none", per_gate=1, post=True, top_k=0, experts=0,
          scale=1.0):
    return {"op": "norm", "name": name, "rows": rows, "d_model": d_model, "dtype": dtype, "kind": kind,
            "gate": gate, "gate_act": gate_act, "per_gate": per_gate, "post": post, "top_k": top_k,
            "experts": experts, "scale": scale}


def listed():
    return [
        # One token of one request: the router's latency.
        _route("route_1_token", 1, 8, 2, "fp32", "softmax"),
        # The valid rows of a packed batch of 32 sequences of up to 4096
        # tokens (an odd count); sigmoid scores, a bias that balances the
        # experts, groups, and a few rows closed to every expert (padding).
        _route("route_batch_sigmoid_groups", 90077, 64, 6, "fp32", "sigmoid", bias=True, groups=8, top_groups=3,
               group_top=2, scale=2.5, closed=0.01),
        # Many small experts, half-precision logits (equal values are common),
        # plain softmax weights.
        _route("route_256_experts_bf16", 16384, 256, 8, "bf16", "softmax", renorm=False),
        # One token: every byte of two experts' weights for two rows.
        _ffn("ffn_1_token", 1, 8, 2, 1024, 4096, "fp16"),
        # A small serving step: most experts see one to three rows.
        _ffn("ffn_33_tokens_64_experts", 33, 64, 4, 1024, 2048, "bf16"),
        # One ragged mid-size batch, widths of no round number.
        _ffn("ffn_ragged", 1777, 12, 2, 760, 1912, "fp16", scoring="sigmoid"),
        # Many narrow experts over a long batch.
        _ffn("ffn_narrow_experts_bf16", 16390, 32, 4, 1024, 1024, "bf16", scoring="sigmoid"),
        # A packed batch through eight full-width experts, some much busier.
        _ffn("ffn_batch", 24001, 8, 2, 1024, 4096, "fp16", skew=1.0),
        # One token's residual step.
        _norm("norm_1_token", 1, 1024, "fp16", "layer", "channel"),
        # The packed batch with a gate of each sample.
        _norm("norm_batch_sample_gate", 90077, 1024, "fp16", "layer", "sample", per_gate=4096, scale=0.5),
        # Wide rows: two experts' outputs combined, a sigmoid gate of each token.
        _norm("norm_experts_token_gate", 32768, 2048, "bf16", "rms", "token", gate_act="sigmoid", top_k=2,
              experts=16),
        # An odd width, which no wide load fits.
        _norm("norm_odd_width", 12345, 1021, "fp16", "layer", "channel", gate_act="tanh"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "ffn", "norm"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log_int(rng, 2, 256 // groups)
        top_groups = rng.randint(1, groups)
        per = experts // groups
        top_k = rng.randint(1, min(8, per * top_groups))
        rows = _log_int(rng, 1, 90077)
        while rows * experts > 90077 * 64:
            rows = max(1, rows // 2)
        bias = rng.random() < 0.5
        return _route(None, rows, experts, top_k, rng.choice(list(DTYPES)), rng.choice(["softmax", "sigmoid"]),
                      bias=bias, groups=groups, top_groups=top_groups,
                      group_top=rng.choice([1, 2]) if per > 1 else 1, renorm=rng.random() < 0.6,
                      scale=rng.choice([1.0, 2.5]), closed=rng.choice([0.0, 0.02]))
    if op == "ffn":
        experts = _log_int(rng, 2, 64)
        top_k = rng.randint(1, min(4, experts))
        d_model = 8 * _log_int(rng, 8, 128)
        ffn_dim = 8 * _log_int(rng, 8, 512)
        while experts * d_model * ffn_dim > 64 * 1024 * 2048:
            experts = max(top_k, experts // 2)
        rows = _log_int(rng, 1, 24001)
        while rows * top_k * d_model * ffn_dim > 24001 * 2 * 1024 * 4096:
            rows //= 2
        return _ffn(None, rows, experts, top_k, d_model, ffn_dim, rng.choice(["fp16", "bf16"]),
                    rng.choice(["softmax", "sigmoid"]), rng.choice([0.2, 1.0]))
    d_model = rng.choice([8 * _log_int(rng, 4, 512), _log_int(rng, 32, 2048)])
    top_k = rng.choice([0, 0, 1, 2, 4])
    rows = _log_int(rng, 1, 90077)
    while rows * d_model * (10 + 2 * top_k) > 32768 * 2048 * 16:
        rows //= 2
    rows = max(1, rows)
    gate = rng.choice(["none", "channel", "sample", "token"])
    return _norm(None, rows, d_model, rng.choice(["fp16", "bf16"]), rng.choice(["layer", "rms"]), gate,
                 rng.choice(["none", "sigmoid", "tanh"]) if gate != "none" else "none",
                 per_gate=_log_int(rng, 1, 4096) if gate == "sample" else 1, post=rng.random() < 0.8,
                 top_k=top_k, experts=max(top_k, rng.randint(2, 64)) if top_k else 0,
                 scale=rng.choice([1.0, 0.5]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _logits(case, g, skew):
    """Router logits: a popularity of each expert plus each row's own taste."""
    t, e = case["rows"], case["experts"]
    popular = torch.randn(e, generator=g, device=DEV) * skew
    return torch.randn(t, e, generator=g, device=DEV) * 1.5 + popular


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    t = case["rows"]
    dt = DTYPES[case["dtype"]]

    def rand(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)

    if case["op"] == "route":
        logits = _logits(case, g, 0.5)
        if case["closed"]:
            shut = torch.rand(t, 1, generator=g, device=DEV) < case["closed"]
            logits = logits.masked_fill(shut, -math.inf)
        s["logits"] = logits.to(dt)
        s["bias"] = rand(case["experts"], std=0.05) if case["bias"] else None
    elif case["op"] == "ffn":
        e, d, f = case["experts"], case["d_model"], case["ffn_dim"]
        s["logits"] = _logits(case, g, case["skew"])
        s["a"] = rand(t, d, dtype=dt)
        s["w_in"] = rand(e, f, d, std=d**-0.5, dtype=dt)
        s["b_in"] = rand(e, f, std=0.1)
        s["w_out"] = rand(e, d, f, std=f**-0.5, dtype=dt)
        s["b_out"] = rand(e, d, std=0.1)
    else:
        d, k = case["d_model"], case["top_k"]
        s["x"] = rand(t, d, std=2.0)
        s["post_gamma"] = rand(d, std=0.2, mean=1.0) if case["post"] else None
        s["post_beta"] = rand(d, std=0.1) if case["post"] and case["kind"] == "layer" else None
        s["pre_gamma"] = rand(d, std=0.2, mean=1.0)
        s["pre_beta"] = rand(d, std=0.1) if case["kind"] == "layer" else None
        if case["gate"] == "channel":
            s["gate"] = rand(d)
        elif case["gate"] == "sample":
            s["gate"] = rand(-(-t // case["per_gate"]), d)
        elif case["gate"] == "token":
            s["gate"] = rand(t, d, dtype=dt)
        else:
            s["gate"] = None
        if k:
            # Outputs of the experts in slot order (all slots of expert 0
            # first, then expert 1, ...; rows in order inside an expert).
            e = case["experts"]
            chosen = torch.rand(t, e, generator=g, device=DEV).argsort(1)[:, :k].to(torch.int32).contiguous()
            weights = torch.rand(t, k, generator=g, device=DEV) + 0.1
            weights = weights / weights.sum(1, keepdim=True)
            s["branch"] = rand(t * k, d, dtype=dt)
            s["weights"] = weights
            order = torch.argsort(chosen.reshape(-1).long(), stable=True)
            place = torch.empty_like(order)
            place[order] = torch.arange(t * k, device=DEV)
            s["row_slot"] = place.view(t, k)
            s["routing"] = _kernels().expert_plan(chosen, weights, e) if own else None
        else:
            s["branch"] = rand(t, d, std=1.5, dtype=dt)
            s["routing"] = None
    return s


# ---------------------------------------------------------------------------
# Plain form
# ---------------------------------------------------------------------------
def _plain_choice(logits, case, bias):
    """experts [T, k] int32 (-1: none left) and weights [T, k] fp32.  Values
    that decide a choice are computed in 64 bits: two of them may lie closer
    than 32 bits can tell apart."""
    groups = case.get("groups", 1)
    top_groups = case.get("top_groups", 1)
    x = logits.double()
    t, e = x.shape
    live = x > -math.inf
    if case["scoring"] == "softmax":
        top = torch.where(live, x, torch.full_like(x, -1e300)).amax(1, keepdim=True)
        ex = torch.where(live, torch.exp(x - top), torch.zeros_like(x))
        total = ex.sum(1, keepdim=True)
        score = torch.where(total > 0, ex / total, torch.zeros_like(ex))
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    value = score if bias is None else score + bias.double()
    value = torch.where(live, value, torch.full_like(value, -math.inf))
    if groups > 1:
        by_group = value.view(t, groups, e // groups).sort(2, descending=True)[0][:, :, : case["group_top"]]
        any_live = live.view(t, groups, -1).any(2)
        strength = torch.where(by_group > -math.inf, by_group, torch.zeros_like(by_group)).sum(2)
        strength = torch.where(any_live, strength, torch.full_like(strength, -math.inf))
        rank = strength.sort(stable=True, dim=1, descending=True)[1][:, :top_groups]
        keep = torch.zeros(t, groups, dtype=torch.bool, device=x.device).scatter_(1, rank, True)
        keep = keep.repeat_interleave(e // groups, 1)
        value = torch.where(keep, value, torch.full_like(value, -math.inf))
    got, chosen = value.sort(stable=True, dim=1, descending=True)
    got, chosen = got[:, : case["top_k"]], chosen[:, : case["top_k"]]
    found = got > -math.inf
    w = torch.where(found, score.gather(1, chosen), torch.zeros_like(got))
    if case.get("renorm", True):
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    w = (w * case.get("scale", 1.0)).float()
    return torch.where(found, chosen, torch.full_like(chosen, -1)).to(torch.int32), w


def _plain_plan(chosen, experts):
    """offsets [E+1], slot_row [T*k], row_slot [T, k] of the choices."""
    t, k = chosen.shape
    flat = chosen.reshape(-1).long()
    key = torch.where(flat < 0, torch.full_like(flat, experts), flat)
    sorted_key, order = key.sort(stable=True, dim=0)
    offsets = torch.searchsorted(sorted_key, torch.arange(experts + 1, device=flat.device))
    place = torch.arange(t * k, device=flat.device)
    slot_row = torch.where(place < offsets[-1], order // k, torch.full_like(order, -1))
    row_slot = torch.empty_like(order)
    row_slot[order] = place
    row_slot = torch.where(flat < 0, torch.full_like(row_slot, -1), row_slot)
    return offsets.to(torch.int32), slot_row.to(torch.int32), row_slot.view(t, k).to(torch.int32)


def _plain_norm(v, kind, gamma, beta, eps=1e-5):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + eps) * gamma
    return v if beta is None else v + beta


def _gate_rows(s):
    """The gate of each row, in 32 bits, before its activation."""
    case, gate = s["case"], s["gate"].float()
    if case["gate"] == "sample":
        gate = gate[torch.arange(case["rows"], device=gate.device) // case["per_gate"]]
    return gate


def _run_plain(s):
    case = s["case"]
    if case["op"] == "route":
        chosen, w = _plain_choice(s["logits"], case, s["bias"])
        offsets, slot_row, row_slot = _plain_plan(chosen, case["experts"])
        return {"experts": chosen, "weights": w, "offsets": offsets, "slot_row": slot_row, "row_slot": row_slot}
    if case["op"] == "ffn":
        chosen, w = _plain_choice(s["logits"], case, None)
        offsets, slot_row, row_slot = _plain_plan(chosen, case["experts"])
        a = s["a"].float()
        y = torch.zeros(slot_row.numel(), a.shape[1], device=a.device)
        ends = offsets.tolist()
        rows = slot_row.long()
        for e in range(case["experts"]):
            lo, hi = ends[e], ends[e + 1]
            if hi > lo:
                h = a[rows[lo:hi]] @ s["w_in"][e].float().t() + s["b_in"][e]
                h = 0.5 * h * (1.0 + torch.erf(h * math.sqrt(0.5)))
                y[lo:hi] = h @ s["w_out"][e].float().t() + s["b_out"][e]
        out = torch.zeros_like(a)
        for j in range(case["top_k"]):
            out += w[:, j : j + 1] * y[row_slot[:, j].long()]
        return {"out": out.to(s["a"].dtype), "experts": chosen, "weights": w}
    if case["top_k"]:
        b = torch.zeros_like(s["x"])
        for j in range(case["top_k"]):
            b += s["weights"][:, j : j + 1] * s["branch"][s["row_slot"][:, j]].float()
    else:
        b = s["branch"].float()
    if case["post"]:
        b = _plain_norm(b, case["kind"], s["post_gamma"], s["post_beta"])
    if s["gate"] is not None:
        gate = _gate_rows(s)
        if case["gate_act"] == "sigmoid":
            gate = 1.0 / (1.0 + torch.exp(-gate))
        elif case["gate_act"] == "tanh":
            gate = torch.tanh(gate)
        b = b * gate
    total = s["x"] + case["scale"] * b
    y = _plain_norm(total, case["kind"], s["pre_gamma"], s["pre_beta"])
    return {"sum": total, "y": y.to(s["branch"].dtype)}


# ---------------------------------------------------------------------------
# The package's operators
# ---------------------------------------------------------------------------
def _run_own(s):
    case = s["case"]
    k = _kernels()
    if case["op"] == "route":
        r = k.route_experts(s["logits"], case["top_k"], scoring=case["scoring"], bias=s["bias"],
                            num_groups=case["groups"], top_groups=case["top_groups"],
                            group_score_top=case["group_top"], renormalize=case["renorm"],
                            weight_scale=case["scale"])
        return {"experts": r.experts, "weights": r.weights, "offsets": r.offsets, "slot_row": r.slot_row,
                "row_slot": r.row_slot}
    if case["op"] == "ffn":
        r = k.route_experts(s["logits"], case["top_k"], scoring=case["scoring"])
        out = k.expert_ffn(s["a"], s["w_in"], s["b_in"], s["w_out"], s["b_out"], r)
        return {"out": out, "experts": r.experts, "weights": r.weights}
    total, y = k.sandwich_norm(s["x"], s["branch"], s["pre_gamma"], s["pre_beta"], post_gamma=s["post_gamma"],
                               post_beta=s["post_beta"], kind=case["kind"], gate=s["gate"],
                               gate_act=case["gate_act"], rows_per_gate=case["per_gate"],
                               residual_scale=case["scale"], routing=s["routing"])
    return {"sum": total, "y": y}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    t = case["rows"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "route":
        e, k = case["experts"], case["top_k"]
        return {"bytes": t * e * size + t * k * 16 + 4 * (e + 1) + (4 * e if case["bias"] else 0),
                "flops": t * e * 8}
    if case["op"] == "ffn":
        e, k, d, f = case["experts"], case["top_k"], case["d_model"], case["ffn_dim"]
        reached = e * (1.0 - (1.0 - k / e) ** t)  # experts that some row chooses
        return {"bytes": int(2 * t * d * size + reached * (2 * d * f * size + 4 * (d + f)) + t * e * 4 + t * k * 8),
                "flops": 4 * t * k * d * f}
    d, k = case["d_model"], case["top_k"]
    gates = {"none": 0, "channel": 4 * d, "sample": 4 * d * -(-t // case["per_gate"]), "token": t * d * size}
    return {"bytes": t * d * (8 + size + size * max(1, k)) + gates[case["gate"]] + t * k * 8 + 16 * d,
            "flops": t * d * (20 + 2 * k)}


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def _exact_choice(logits, case, bias):
    """numpy, row by row of sorted order: lexsort keeps the lowest index of
    equal values first."""
    x = logits.double().cpu().numpy()
    t, e = x.shape
    k, groups = case["top_k"], case.get("groups", 1)
    shut = np.isneginf(x)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if case["scoring"] == "softmax":
            m = np.where(shut.all(1, keepdims=True), 0.0, x.max(1, keepdims=True))
            p = np.exp(x - m)
            z = p.sum(1, keepdims=True)
            score = np.divide(p, z, out=np.zeros_like(p), where=z > 0)
        else:
            score = np.exp(-np.logaddexp(0.0, -x))
    value = score.copy()
    if bias is not None:
        value += bias.double().cpu().numpy()[None]
    value[shut] = -np.inf
    if groups > 1:
        per = e // groups
        g = -np.sort(-value.reshape(t, groups, per), axis=2)[:, :, : case["group_top"]]
        strength = np.where(np.isneginf(g), 0.0, g).sum(2)
        strength[shut.reshape(t, groups, per).all(2)] = -np.inf
        order = np.argsort(-strength, axis=1, kind="stable")[:, : case["top_groups"]]
        kept = np.zeros((t, groups), bool)
        np.put_along_axis(kept, order, True, axis=1)
        value[~np.repeat(kept, per, axis=1)] = -np.inf
    order = np.argsort(-value, axis=1, kind="stable")[:, :k]
    none = np.isneginf(np.take_along_axis(value, order, axis=1))
    w = np.where(none, 0.0, np.take_along_axis(score, order, axis=1))
    if case.get("renorm", True):
        z = w.sum(1, keepdims=True)
        w = np.divide(w, z, out=np.zeros_like(w), where=z > 0)
    return np.where(none, -1, order).astype(np.int32), w * case.get("scale", 1.0)


def exact(case, seed):
    s = prepare(case, seed)

    def tensor(v):
        return torch.from_numpy(np.ascontiguousarray(v)).to(DEV)

    if case["op"] == "route":
        chosen, w = _exact_choice(s["logits"], case, s["bias"])
        t, k = chosen.shape
        flat = chosen.reshape(-1)
        taken = np.flatnonzero(flat >= 0)
        slots = taken[np.lexsort((taken, flat[taken]))]
        slot_row = np.full(t * k, -1, np.int32)
        slot_row[: slots.size] = slots // k
        row_slot = np.full(t * k, -1, np.int32)
        row_slot[slots] = np.arange(slots.size)
        offsets = np.zeros(case["experts"] + 1, np.int32)
        offsets[1:] = np.cumsum(np.bincount(flat[taken], minlength=case["experts"]))
        return {"experts": tensor(chosen), "weights": tensor(w), "offsets": tensor(offsets),
                "slot_row": tensor(slot_row), "row_slot": tensor(row_slot.reshape(t, k))}
    if case["op"] == "ffn":
        chosen, w = _exact_choice(s["logits"], case, None)
        ids, w = tensor(chosen).long(), tensor(w)
        out = torch.zeros(s["a"].shape, dtype=torch.float64, device=DEV)
        for e in range(case["experts"]):
            share = torch.where(ids == e, w, torch.zeros_like(w)).sum(1)
            mine = (ids == e).any(1).nonzero().flatten()
            if mine.numel() == 0:
                continue
            z = torch.addmm(s["b_in"][e].double(), s["a"][mine].double(), s["w_in"][e].double().t())
            z = z * 0.5 * torch.erfc(-z / math.sqrt(2.0))
            z = torch.addmm(s["b_out"][e].double(), z, s["w_out"][e].double().t())
            out.index_add_(0, mine, z * share[mine, None])
        return {"out": out, "experts": tensor(chosen), "weights": w}

    def norm(v, gamma, beta):
        centre = v.mean(1, keepdim=True) if case["kind"] == "layer" else torch.zeros_like(v[:, :1])
        spread = torch.sqrt(((v - centre) ** 2).sum(1, keepdim=True) / v.shape[1] + 1e-5)
        v = (v - centre) / spread * gamma.double()
        return v + beta.double() if beta is not None else v

    if case["top_k"]:
        parts = s["branch"].double()[s["row_slot"].reshape(-1)].view(case["rows"], case["top_k"], -1)
        b = torch.einsum("tkd,tk->td", parts, s["weights"].double())
        del parts
    else:
        b = s["branch"].double()
    if case["post"]:
        b = norm(b, s["post_gamma"], s["post_beta"])
    if s["gate"] is not None:
        gate = s["gate"].double()
        if case["gate_act"] == "sigmoid":
            gate = torch.special.expit(gate)
        elif case["gate_act"] == "tanh":
            gate = torch.tanh(gate)
        if case["gate"] == "sample":
            gate = gate.repeat_interleave(case["per_gate"], 0)[: case["rows"]]
        b = b * gate
    total = s["x"].double() + b * case["scale"]
    return {"sum": total, "y": norm(total, s["pre_gamma"], s["pre_beta"])}
