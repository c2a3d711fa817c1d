"""What the measurement of the routed-expert operators (``fsctep_b200.experts``) runs.

``listed()`` names the cases and ``draw(rng)`` gives more of the same ranges; ``prepare`` makes what a
program has in hand before the call; ``run`` is one pass, in plain torch operations (``own`` false) or
through the framework's entry points (``own`` true); ``exact`` gives the same outputs from the
definitions in 64 bits; ``work`` counts the bytes and operations a pass cannot do without.
"""

import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---- the cases -----------------------------------------------------------------------------------

def listed():
    return [
        # one token of a serving step through a wide norm: latency alone
        dict(name="norm_step", op="norm", dtype="f16", rows=1, dim=4096),
        # a long prompt's hidden states, the residual stream updated on the way
        dict(name="norm_prompt", op="norm", dtype="bf16", rows=16384, dim=4096),
        # the same in front of an 8-bit product, a ragged number of tokens
        dict(name="norm_q8", op="norm_q8", dtype="bf16", rows=8191, dim=2048),
        # features of a 64,000-atom crystal (64 channels, 9 components), reverse pass
        dict(name="norm_atoms_back", op="norm_backward", dtype="f32", rows=64000, dim=576),
        # one token's choice of 6 experts in 64
        dict(name="route_step", op="route", dtype="bf16", tokens=1, experts=64, top_k=6, scores="softmax",
             groups=1, kept=1, renormalize=True, scale=1.0, bias=False),
        # a prompt's choice of 8 in 256, balanced by a bias, limited to 4 of 8 groups
        dict(name="route_groups", op="route", dtype="f32", tokens=16384, experts=256, top_k=8, scores="sigmoid",
             groups=8, kept=4, renormalize=True, scale=2.5, bias=True),
        # a training batch: choice and the logits' gradient, an odd number of experts
        dict(name="route_train", op="route_backward", dtype="f32", tokens=10007, experts=100, top_k=4,
             scores="softmax", groups=1, kept=1, renormalize=True, scale=1.0, bias=False),
        # one token through its 8 experts: the experts' weights are read, little else
        dict(name="expert_step", op="expert", dtype="bf16", tokens=1, comps=1, experts=64, top_k=8, inputs=2048,
             outputs=1024, padded=False, slots=False),
        # a ragged padded prompt through 4 of 64 experts
        dict(name="expert_prompt", op="expert", dtype="bf16", tokens=4001, comps=1, experts=64, top_k=4, inputs=2048,
             outputs=1024, padded=True, slots=False),
        # a training step of 8 experts: outputs and all three gradients
        dict(name="expert_train", op="expert_backward", dtype="bf16", tokens=8192, comps=1, experts=8, top_k=2,
             inputs=1024, outputs=2048, padded=False, slots=False, weight_gradient=True),
        # equivariant features of 50,021 atoms through 2 of 8 channel mixes, with the gradients that forces need
        dict(name="expert_atoms", op="expert_backward", dtype="f32", tokens=50021, comps=9, experts=8, top_k=2,
             inputs=64, outputs=64, padded=False, slots=False, weight_gradient=False),
        # a batch of prompts with 8-bit activations and weights
        dict(name="expert_q8", op="expert_q8", dtype="bf16", tokens=2000, comps=1, experts=16, top_k=2, inputs=2048,
             outputs=2048, padded=False, slots=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_q8", "norm_backward", "route", "route_backward", "expert", "expert",
                     "expert_backward", "expert_backward", "expert_q8"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op.startswith("norm"):
        dim = _log(rng, 32, 8192)
        if rng.random() < 0.7:  # most widths are multiples of 16, some odd
            dim = max(16, dim // 16 * 16)
        return dict(op=op, dtype=dtype, rows=min(_log(rng, 1, 64000), max(1, 36_000_000 // dim)), dim=dim)
    if op.startswith("route"):
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, max(2, 8 // groups), 256 // groups)
        kept = 1 if groups == 1 else rng.randint(1, groups)
        top_k = rng.randint(1, min(8, experts // groups * kept))
        return dict(op=op, dtype=dtype, tokens=_log(rng, 1, 16384), experts=experts, top_k=top_k,
                    scores=rng.choice(["softmax", "sigmoid"]), groups=groups, kept=kept,
                    renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), bias=rng.random() < 0.5)
    if op == "expert_q8":
        dtype = "bf16"
    comps = rng.choice([1, 1, 1, 4, 9]) if op != "expert_q8" else 1
    experts = _log(rng, 2, 64)
    top_k = rng.randint(1, min(8, experts))
    inputs, outputs = _log(rng, 32, 2048), _log(rng, 32, 2048)
    if rng.random() < 0.7:
        inputs, outputs = max(16, inputs // 16 * 16), max(16, outputs // 16 * 16)
    most = 2_000_000_000 if dtype == "f32" else 10_000_000_000  # multiply-adds of one product
    tokens = _log(rng, 1, 16384)
    while tokens > 1 and (tokens * top_k * comps * inputs * outputs > most
                          or tokens * top_k * comps * (inputs + outputs) > 60_000_000):
        tokens = max(1, tokens * 2 // 3)
    case = dict(op=op, dtype=dtype, tokens=tokens, comps=comps, experts=experts, top_k=top_k, inputs=inputs,
                outputs=outputs, padded=rng.random() < 0.3, slots=rng.random() < 0.3)
    if op == "expert_backward":
        case["weight_gradient"] = rng.random() < 0.6
    return case


# ---- inputs --------------------------------------------------------------------------------------

def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _choice(g, case):
    """Indices as a router gives them: distinct experts per token, some more popular than others."""
    t, x, k = case["tokens"], case["experts"], case["top_k"]
    popular = torch.randn((1, x), generator=g, device="cuda") * 0.5
    gumbel = -torch.log(-torch.log(torch.rand((t, x), generator=g, device="cuda").clamp(1e-9, 1 - 1e-7)))
    value, index = (popular + gumbel).topk(k, dim=1)
    weights, indices = torch.softmax(value, dim=1), index.to(torch.int32)
    if case["padded"]:  # the last tokens of the batch are padding: no expert, features undefined
        first = t - t // 10
        indices[first:] = -1
        weights[first:] = 0
    return weights.contiguous(), indices.contiguous()


def _to_e4m3(w):
    scale = w.abs().amax(-1) / E4M3_MAX
    return (w / scale.clamp_min(1e-30).unsqueeze(-1)).to(torch.float8_e4m3fn), scale.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if op.startswith("norm"):
        n, d = case["rows"], case["dim"]
        s["weight"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dtype)
        if op == "norm_backward":
            s["h"] = _normal(g, (n, d), dtype, 1.5)
            s["grad_y"], s["grad_h"] = _normal(g, (n, d), dtype), _normal(g, (n, d), dtype)
        else:
            s["x"], s["residual"] = _normal(g, (n, d), dtype), _normal(g, (n, d), dtype, 2.0)
        return s
    if op.startswith("route"):
        t, x = case["tokens"], case["experts"]
        s["logits"] = _normal(g, (t, x), dtype, 2.0)
        s["bias"] = 0.05 * torch.randn(x, generator=g, device="cuda") if case["bias"] else None
        if op == "route_backward":
            s["grad_weights"] = torch.randn((t, case["top_k"]), generator=g, device="cuda")
        return s
    t, k, x, i, o, n = (case[c] for c in ("tokens", "top_k", "experts", "inputs", "outputs", "comps"))
    weights, s["indices"] = _choice(g, case)
    s["weights"] = weights
    mid = (n,) if n > 1 else ()
    rows = (t, k) if case["slots"] else (t,)
    xs = torch.randn(rows + mid + (i,), generator=g, device="cuda")
    w = torch.randn((x, o, i), generator=g, device="cuda") / math.sqrt(i)
    if op == "expert_q8":
        s["x"], s["x_scale"] = _to_e4m3(xs)
        s["w"], s["w_scale"] = _to_e4m3(w)
        return s
    s["x"], s["w"] = xs.to(dtype), w.to(dtype)
    if op == "expert_backward":
        s["grad_out"] = _normal(g, (t,) + mid + (o,), dtype)
    if case["padded"]:  # what lies in padded rows does not count
        s["x"][t - t // 10:] = float("nan")
    return s


# ---- one pass ------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    op = case["op"]
    if op in ("norm", "norm_q8"):
        return _norm(state, op == "norm_q8")
    if op == "norm_backward":
        return _norm_backward(state)
    if op == "route":
        return _route(case, state)[:2]
    if op == "route_backward":
        return _route_backward(case, state)
    if op == "expert_backward":
        return _expert_backward(case, state)
    return _expert(case, state)


def _run_own(case, s):
    from fsctep_b200 import experts as E

    op = case["op"]
    if op == "norm":
        return E.add_rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
    if op == "norm_q8":
        return E.add_rms_norm_q8(s["x"], s["weight"], s["residual"], eps=EPS)
    if op == "norm_backward":
        return E.add_rms_norm_backward(s["grad_y"], s["h"], s["weight"], s["grad_h"], eps=EPS)
    if op.startswith("route"):
        kw = dict(scores=case["scores"], renormalize=case["renormalize"], scale=case["scale"])
        weights, indices = E.route_experts(s["logits"], case["top_k"], bias=s["bias"], num_groups=case["groups"],
                                           groups_kept=case["kept"], **kw)
        if op == "route":
            return weights, indices
        return weights, indices, E.route_experts_backward(s["grad_weights"], s["logits"], indices, **kw)
    if op == "expert":
        return E.expert_linear(s["x"], s["w"], s["indices"], s["weights"], slots=case["slots"])
    if op == "expert_q8":
        return E.expert_linear_q8(s["x"], s["x_scale"], s["w"], s["w_scale"], s["indices"], s["weights"],
                                  slots=case["slots"], out_dtype=torch.bfloat16)
    plan = E.expert_plan(s["indices"], case["experts"])
    y = E.expert_linear(s["x"], s["w"], s["indices"], s["weights"], slots=case["slots"], plan=plan)
    gx, gw, gwt = E.expert_linear_backward(s["grad_out"], s["x"], s["w"], s["indices"], s["weights"],
                                           slots=case["slots"], plan=plan, weight_gradient=case["weight_gradient"])
    return [t for t in (y, gx, gw, gwt) if t is not None]


# ---- the plain forms -----------------------------------------------------------------------------

def _norm(s, to_8_bits):
    dtype = s["x"].dtype
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    if not to_8_bits:
        return y.to(dtype), h.to(dtype)
    scale = y.abs().amax(-1) / E4M3_MAX
    q = torch.where(scale.unsqueeze(-1) > 0, y / scale.unsqueeze(-1), torch.zeros_like(y))
    return q.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale, h.to(dtype)


def _norm_backward(s):
    dtype, h, w = s["h"].dtype, s["h"].float(), s["weight"].float()
    gy = s["grad_y"].float()
    u = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    a = gy * w
    gx = u * a - h * (u * u * u) * (a * h).mean(-1, keepdim=True) + s["grad_h"].float()
    return gx.to(dtype), (gy * h * u).sum(0).to(s["weight"].dtype)


def _route(case, s):
    logits = s["logits"].double()  # the choice at the border of two scores needs 64 bits
    p = torch.softmax(logits, 1) if case["scores"] == "softmax" else 1 / (1 + torch.exp(-logits))
    t = p + s["bias"].double() if s["bias"] is not None else p
    n, x = p.shape
    if case["groups"] > 1:
        by = t.reshape(n, case["groups"], -1)
        best = by.sort(dim=-1, descending=True).values[..., :2].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, :case["kept"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter(1, kept, True)
        t = torch.where(open_.unsqueeze(-1), by, torch.full_like(by, -math.inf)).reshape(n, x)
    indices = t.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
    chosen = p.gather(1, indices)
    total = chosen.sum(1, keepdim=True) + 1e-20
    weights = chosen / total if case["renormalize"] else chosen
    return (weights * case["scale"]).float(), indices.to(torch.int32), p, chosen, total


def _route_backward(case, s):
    weights, indices, p, chosen, total = _route(case, s)
    g = s["grad_weights"].double() * case["scale"]
    if case["renormalize"]:
        g = (g - (g * chosen).sum(1, keepdim=True) / total) / total
    d = torch.zeros_like(p).scatter(1, indices.long(), g)
    if case["scores"] == "softmax":
        gl = p * (d - (d * p).sum(1, keepdim=True))
    else:
        gl = d * p * (1 - p)
    return weights, indices, gl.to(s["logits"].dtype)


def _blocks(indices, experts):
    """Slots in blocks of one expert each: (block, place) -> slot (-1: none), and each block's expert."""
    flat = indices.reshape(-1).long()
    n = flat.numel()
    size = max(1, min(128, n // experts))
    count = -(-n // size) + (experts if size > 1 else 0)
    key = torch.where(flat >= 0, flat, torch.full_like(flat, experts))
    order = torch.sort(key, stable=True).indices
    key = key[order]
    counts = torch.zeros(experts + 1, dtype=torch.long, device=flat.device).index_add(0, key, torch.ones_like(key))
    blocks = (counts + size - 1) // size
    blocks[experts] = 0
    first, start = torch.cumsum(blocks, 0) - blocks, torch.cumsum(counts, 0) - counts
    place = first[key] * size + torch.arange(n, device=flat.device) - start[key]
    place = torch.where(key < experts, place, torch.full_like(place, count * size))
    slot = torch.full((count * size + 1,), -1, dtype=torch.long, device=flat.device).scatter(0, place, order)
    expert = (torch.arange(count, device=flat.device)[:, None] >= first[None, :experts]).sum(1) - 1
    return slot[:-1].reshape(count, size), expert


def _rows(v, at, slot):
    """v[at] in 32 bits as (blocks, rows, width), zero where there is no slot."""
    got = v.reshape(v.shape[0], -1, v.shape[-1])[at.reshape(-1)].float()
    got = torch.where((slot >= 0).reshape(-1, 1, 1), got, torch.zeros_like(got))
    return got.reshape(slot.shape[0], -1, v.shape[-1])


def _to_slots(rows, slot, slots, comps):
    """Block rows back in slot order: (slots, comps, width); slots of no expert give zero."""
    width = rows.shape[-1]
    out = torch.zeros((slots + 1, comps, width), dtype=rows.dtype, device=rows.device)
    at = torch.where(slot >= 0, slot, torch.full_like(slot, slots)).reshape(-1)
    return out.index_copy(0, at, rows.reshape(-1, comps, width))[:slots]


def _expert_rows(case, s):
    """The products of every slot in 32 bits, (slots, comps, outputs), and what places them."""
    t, k, n = case["tokens"], case["top_k"], case["comps"]
    slot, expert = _blocks(s["indices"], case["experts"])
    at = slot.clamp_min(0)
    token = at // k
    x = s["x"].reshape((t * k if case["slots"] else t,) + tuple(s["x"].shape[2 if case["slots"] else 1:]))
    where = at if case["slots"] else token
    xr = _rows(x, where, slot)
    if case["op"] == "expert_q8":
        xr = xr * s["x_scale"].reshape(-1)[where].reshape(xr.shape[0], -1, 1)
        w = s["w"].float() * s["w_scale"].unsqueeze(-1)
    else:
        w = s["w"].float()
    w = w[expert]
    return _to_slots(xr @ w.transpose(1, 2), slot, t * k, n), slot, token, xr, w, expert


def _shape(case, width, rows):
    return rows + ((case["comps"],) if case["comps"] > 1 else ()) + (width,)


def _expert(case, s):
    t, k, n = case["tokens"], case["top_k"], case["comps"]
    z = _expert_rows(case, s)[0]
    y = (z.reshape(t, k, n, -1) * s["weights"].reshape(t, k, 1, 1)).sum(1)
    return y.reshape(_shape(case, case["outputs"], (t,))).to(DTYPES[case["dtype"]])


def _expert_backward(case, s):
    t, k, n, i, o = (case[c] for c in ("tokens", "top_k", "comps", "inputs", "outputs"))
    dtype = DTYPES[case["dtype"]]
    z, slot, token, xr, w, expert = _expert_rows(case, s)
    y = (z.reshape(t, k, n, o) * s["weights"].reshape(t, k, 1, 1)).sum(1)
    gy = s["grad_out"].float().reshape(t, 1, n, o)
    live = (s["indices"] >= 0).reshape(t, k, 1, 1)
    gwt = (torch.where(live, z.reshape(t, k, n, o), 0) * gy).sum((2, 3))
    gr = _rows(s["grad_out"], token, slot)
    gr = gr * s["weights"].reshape(-1)[slot.clamp_min(0)].reshape(slot.shape[0], slot.shape[1], 1, 1).expand(
        -1, -1, n, -1).reshape(slot.shape[0], -1, 1)
    gx = _to_slots(gr @ w, slot, t * k, n).reshape(t, k, n, i)
    gx = gx.reshape(_shape(case, i, (t, k))) if case["slots"] else gx.sum(1).reshape(_shape(case, i, (t,)))
    out = [y.reshape(_shape(case, o, (t,))).to(dtype), gx.to(dtype)]
    if case["weight_gradient"]:
        gw = torch.zeros((case["experts"], o, i), device=xr.device).index_add(0, expert, gr.transpose(1, 2) @ xr)
        out.append(gw.to(dtype))
    return out + [gwt]


# ---- 64 bits, from the definitions ---------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("norm"):
        g = s["weight"].double()
        if op == "norm_backward":
            h, gy = s["h"].double(), s["grad_y"].double()
            rms = (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt()
            unit = h / rms
            a = gy * g
            gx = (a - unit * (a * unit).sum(1, keepdim=True) / h.shape[1]) / rms + s["grad_h"].double()
            return gx, (gy * unit).sum(0)
        h = s["x"].double() + s["residual"].double()
        y = h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt() * g
        if op == "norm":
            return y, h
        top = y.abs().max(1).values / E4M3_MAX
        return y / top[:, None], top, h
    if op.startswith("route"):
        return _exact_route(case, s)
    return _exact_expert(case, s)


def _exact_route(case, s):
    logits = s["logits"].double()
    if case["scores"] == "softmax":
        e = (logits - logits.max(1, keepdim=True).values).exp()
        p = e / e.sum(1, keepdim=True)
    else:
        p = torch.sigmoid(logits)
    key = p if s["bias"] is None else p + s["bias"].double()
    per = case["experts"] // case["groups"]
    if case["groups"] > 1:
        parts = torch.stack([key[:, j * per:(j + 1) * per].topk(min(2, per), 1).values.sum(1)
                             for j in range(case["groups"])], 1)
        rank = parts.sort(dim=1, descending=True, stable=True).indices.argsort(1)
        key = key.masked_fill((rank >= case["kept"]).repeat_interleave(per, 1), -math.inf)
    index = key.argsort(dim=1, descending=True, stable=True)[:, :case["top_k"]]  # equal scores: lowest index first
    v = p.gather(1, index)
    total = v.sum(1, keepdim=True) + 1e-20
    weights = case["scale"] * (v / total if case["renormalize"] else v)
    if case["op"] == "route":
        return weights, None
    g = s["grad_weights"].double()
    x = logits.clone().requires_grad_(True)
    q = torch.softmax(x, 1) if case["scores"] == "softmax" else torch.sigmoid(x)
    q = q.gather(1, index)
    w = case["scale"] * (q / (q.sum(1, keepdim=True) + 1e-20) if case["renormalize"] else q)
    return weights, None, torch.autograd.grad((w * g).sum(), x)[0]


def _exact_expert(case, s):
    t, k, n, i, o = (case[c] for c in ("tokens", "top_k", "comps", "inputs", "outputs"))
    if t * k * n * i * o > 2e11:
        return None
    dev = s["w"].device
    x = s["x"].double().reshape(t, k if case["slots"] else 1, n, i)
    if case["op"] == "expert_q8":
        x = x * s["x_scale"].double().reshape(t, -1, 1, 1)
    y = torch.zeros(t, n, o, dtype=torch.float64, device=dev)
    back = case["op"] == "expert_backward"
    if back:
        gy = s["grad_out"].double().reshape(t, n, o)
        gx = torch.zeros(x.shape, dtype=torch.float64, device=dev)
        gwt = torch.zeros(t, k, dtype=torch.float64, device=dev)
        gw = torch.zeros(s["w"].shape, dtype=torch.float64, device=dev)
    for e in range(case["experts"]):
        w = s["w"][e].double()
        if case["op"] == "expert_q8":
            w = w * s["w_scale"][e].double()[:, None]
        for j in range(k):
            at = (s["indices"][:, j] == e).nonzero()[:, 0]
            jj = j if case["slots"] else 0
            xe, we = x[at, jj], s["weights"][at, j].double()[:, None, None]
            z = xe @ w.T
            y[at] += we * z
            if back:
                ge = gy[at]
                gwt[at, j] = (z * ge).sum((1, 2))
                gx[at, jj] += (we * ge) @ w
                if case["weight_gradient"]:
                    gw[e] += (we * ge).reshape(-1, o).T @ xe.reshape(-1, i)
    y = y.reshape(_shape(case, o, (t,)))
    if not back:
        return y
    gx = gx.reshape(_shape(case, i, (t, k) if case["slots"] else (t,)))
    return [y, gx] + ([gw] if case["weight_gradient"] else []) + [gwt]


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    op = case["op"]
    b = SIZE[case["dtype"]]
    if op.startswith("norm"):
        n, d = case["rows"], case["dim"]
        each = {"norm": 4 * b, "norm_q8": 3 * b + 1, "norm_backward": 4 * b}[op]
        return {"bytes": n * d * each + d * b * (2 if op == "norm_backward" else 1) + (4 * n if op == "norm_q8" else 0),
                "flops": n * d * (12 if op == "norm_backward" else 6)}
    if op.startswith("route"):
        t, x, k = case["tokens"], case["experts"], case["top_k"]
        back = op == "route_backward"
        return {"bytes": t * x * b * (2 if back else 1) + t * k * (12 if back else 8) + (4 * x if case["bias"] else 0),
                "flops": t * x * (12 if back else 6)}
    t, k, n, i, o, x = (case[c] for c in ("tokens", "top_k", "comps", "inputs", "outputs", "experts"))
    live = t - (t // 10 if case["padded"] else 0)
    rows = (k if case["slots"] else 1) * n * i
    used = min(x, live * k)
    if op == "expert_q8":
        return {"bytes": live * rows + live * (k if case["slots"] else 1) * 4 + used * o * (i + 4) + t * k * 8 + t * n * o * 2,
                "flops": 2 * live * k * n * i * o}
    size = live * rows * b + used * o * i * b + t * k * 8 + t * n * o * b
    flops = 2 * live * k * n * i * o
    if op == "expert_backward":
        size += live * n * o * b + t * rows * b + t * k * 4
        flops *= 2
        if case["weight_gradient"]:
            size += x * o * i * b
            flops = flops * 3 // 2
    return {"bytes": size, "flops": flops}
