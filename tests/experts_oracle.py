"""Plain 64-bit statements of the routed-expert operators and the error bounds of their kernels."""

import torch

STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a rounding step
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}  # the same near zero
U = 2.0 ** -24


def norm(x, weight, residual=None, eps=1e-6):
    s = x.double() + (0 if residual is None else residual.double())
    u = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s * u * weight.double(), s


def norm_backward(gy, h, weight, gh=None, eps=1e-6):
    """The formula; the second values bound the terms' magnitudes (for cancellation)."""
    h, g, gy = h.double(), weight.double(), gy.double()
    u = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    a = gy * g
    second = h * u ** 3 * (a * h).mean(-1, keepdim=True)
    gx = u * a - second + (0 if gh is None else gh.double())
    size = (u * a).abs() + h.abs() * u ** 3 * (a * h).abs().mean(-1, keepdim=True) + (0 if gh is None else gh.double().abs())
    return (gx, size), ((gy * h * u).sum(0), (gy * h * u).abs().sum(0))


def route(logits, top_k, bias=None, row_mask=None, num_groups=1, groups_kept=None, scores="softmax", renormalize=True,
          scale=1.0):
    """One row at a time, as the operator is defined."""
    import math

    rows, experts = logits.shape
    kept = num_groups if groups_kept is None else groups_kept
    weights = torch.zeros(rows, top_k, dtype=torch.float64)
    indices = torch.full((rows, top_k), -1, dtype=torch.int32)
    top = float(torch.finfo(torch.float32).max)
    all_logits = logits.detach().cpu().float()
    b = None if bias is None else bias.detach().cpu().double()
    for r in range(rows):
        if row_mask is not None and not bool(row_mask[r]):
            continue
        l = all_logits[r].double()
        ok = (l > -math.inf)  # False for NaN
        l = torch.where(ok, l.clamp(max=top), torch.full_like(l, -math.inf))
        if not bool(ok.any()):
            continue
        p = torch.exp(l - l.max()) / torch.exp(l - l.max()).sum() if scores == "softmax" else 1 / (1 + torch.exp(-l))
        wide = b is not None or kept < num_groups
        t = (p if b is None else p + b) if wide else l
        t = torch.where(ok & (t > -math.inf), t, torch.full_like(t, -math.inf))
        if kept < num_groups:
            per = experts // num_groups
            score = []
            for g in range(num_groups):
                best = sorted((v for v in t[g * per:(g + 1) * per].tolist() if v > -math.inf), reverse=True)[:2]
                score.append(sum(best) if best else -math.inf)
            order = sorted(range(num_groups), key=lambda g: (-score[g], g))[:kept]
            for g in range(num_groups):
                if g not in order:
                    t[g * per:(g + 1) * per] = -math.inf
        tl = t.tolist()
        pick = [e for e in sorted(range(experts), key=lambda e: (-tl[e], e)) if tl[e] > -math.inf][:top_k]
        for j, e in enumerate(pick):
            indices[r, j] = e
            weights[r, j] = p[e]
        if renormalize:
            weights[r] /= weights[r].sum() + 1e-20
    return weights * scale, indices


def route_weights(logits, indices, scores, renormalize, scale):
    """The weights of a fixed choice, differentiable in double logits."""
    l = logits.clamp(max=float(torch.finfo(torch.float32).max))
    p = torch.softmax(l, 1) if scores == "softmax" else torch.sigmoid(l)
    live = indices >= 0
    q = torch.where(live, p.gather(1, indices.clamp_min(0).long()), torch.zeros((), dtype=p.dtype, device=p.device))
    return scale * (q / (q.sum(1, keepdim=True) + 1e-20) if renormalize else q)


def rows_of(x, indices, slots):
    """x as double (rows, top_k, components, inputs), zero where there is no expert."""
    t, k = indices.shape
    x = x.double()
    x = x.reshape(t, k, -1, x.shape[-1]) if slots else x.reshape(t, 1, -1, x.shape[-1]).expand(-1, k, -1, -1)
    return x


def linear(x, w, indices, weights=None, slots=False, grad_out=None):
    """out, and with grad_out the gradients, each with the sum of its terms' magnitudes.  ``w`` and x may
    be any dtype; slots without an expert count as zero, whatever their rows hold."""
    t, k = indices.shape
    live = (indices >= 0) & (indices < w.shape[0])
    e = torch.where(live, indices, torch.zeros_like(indices)).long()
    xs = torch.where(live[:, :, None, None], rows_of(x, indices, slots), 0.0)
    c, i, o = xs.shape[2], w.shape[2], w.shape[1]
    we = w.double()[e]  # t k o i
    f = torch.ones(t, k, dtype=torch.float64, device=w.device) if weights is None else weights.double()
    f = torch.where(live, f, 0.0)
    z, za = torch.einsum("tkoi,tkci->tkco", we, xs), torch.einsum("tkoi,tkci->tkco", we.abs(), xs.abs())
    fz, fza = f[:, :, None, None] * z, f.abs()[:, :, None, None] * za
    out = (fz, fza) if weights is None else (fz.sum(1), fza.sum(1))
    if grad_out is None:
        return out
    g = grad_out.double()
    g = g.reshape(t, k, c, o) if weights is None else g.reshape(t, 1, c, o).expand(-1, k, -1, -1)
    fg = f[:, :, None, None] * torch.where(live[:, :, None, None], g, 0.0)
    gx, gxa = torch.einsum("tkoi,tkco->tkci", we, fg), torch.einsum("tkoi,tkco->tkci", we.abs(), fg.abs())
    if not slots:
        gx, gxa = gx.sum(1), gxa.sum(1)
    gw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    gwa = torch.zeros_like(gw)
    one, onea = torch.einsum("tkco,tkci->tkoi", fg, xs), torch.einsum("tkco,tkci->tkoi", fg.abs(), xs.abs())
    at = e[live]
    gw.index_add_(0, at, one[live])
    gwa.index_add_(0, at, onea[live])
    gl = torch.where(live[:, :, None, None], g, 0.0)
    gwt = ((gl * z).sum((2, 3)), (gl.abs() * za).sum((2, 3)))
    return out, (gx, gxa), (gw, gwa), gwt


def accumulate(terms):
    """Relative bound of a tensor-core sum: 16 products an instruction, at most six instructions for
    them (fp32 as three bf16), each of which cuts the running sum at 2^-23; the products left out are
    below 2^-21 (a part of the 40)."""
    return (6 * (terms // 16 + 2) + 40) * 2.0 ** -23


def within(got, want, bound, dtype, what):
    """|got - want| <= half a step of the result's rounding + ``bound``, everywhere."""
    bound = torch.broadcast_to(bound, want.shape)
    got, want = got.double(), want.reshape(got.shape)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - (STEP[dtype] * want.abs() * (1 + 2.0 ** -7) + TINY[dtype] + bound.reshape(got.shape))
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, (what, worst, (got - want).abs().max().item())
