"""Routed-expert operators on the GPU against their 64-bit statements (tests/experts_oracle.py)."""

import math

import pytest
import torch

import experts_oracle as O
import gpu_util as U
from fsctep_b200 import _native as N
from fsctep_b200 import experts as E

pytestmark = [pytest.mark.gpu, U.needs_gpu]

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DT = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


# ---- RMS norm ------------------------------------------------------------------------------------
# y = s u g: the sum of squares adds at most dim / 32 + 40 roundings in a chain, half of whose relative
# error reaches u; a few more roundings follow.
def norm_bound(dim):
    return (dim / 64 + 60) * O.U


DIMS = [1, 7, 32, 64, 100, 576, 1000, 1001, 2048, 2056, 4096, 4104, 8192, 8200, 9001, 20000, 40000]


@DT
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_forward(dtype, dim, residual):
    g = gen(dim)
    rows = 5 if dim > 4096 else 33
    x, w = rand(g, rows, dim, dtype=dtype), (1 + rand(g, dim, scale=0.1)).to(dtype)
    r = rand(g, rows, dim, dtype=dtype, scale=2.0) if residual else None
    x[1] = 0
    if residual:
        r[1] = 0
    got = E.add_rms_norm(x, w, r)
    y, s = O.norm(x, w, r)
    if residual:
        got, h = got
        O.within(h, s, s.abs() * O.U, dtype, "h")
    O.within(got, y, y.abs() * norm_bound(dim), dtype, "y")
    assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [37, 576, 4096])
def test_norm_with_a_32_bit_weight(dtype, dim):
    g = gen(3)
    x, w = rand(g, 9, dim, dtype=dtype), 1 + rand(g, dim, scale=0.1)
    y, _ = O.norm(x, w)
    O.within(E.add_rms_norm(x, w), y, y.abs() * norm_bound(dim), dtype, "y")
    gy = rand(g, 9, dim, dtype=dtype)
    gx, gw = E.add_rms_norm_backward(gy, x, w)
    (rx, sx), (rw, sw) = O.norm_backward(gy, x, w)
    O.within(gx, rx, sx * 4 * norm_bound(dim), dtype, "gx")
    assert gw.dtype == F32
    O.within(gw, rw, sw * (norm_bound(dim) + 30 * O.U), F32, "gw")


@DT
@pytest.mark.parametrize("dim", [16, 17, 576, 1024, 2050, 4096, 9000, 40000])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_8_bits(dtype, dim, residual):
    g = gen(dim + 1)
    x, w = rand(g, 7, dim, dtype=dtype), (1 + rand(g, dim, scale=0.1)).to(dtype)
    r = rand(g, 7, dim, dtype=dtype) if residual else None
    x[2] = 0
    if residual:
        r[2] = 0
    out = E.add_rms_norm_q8(x, w, r)
    q, scale = out[0], out[1]
    assert len(out) == (3 if residual else 2) and q.dtype == torch.float8_e4m3fn and scale.shape == (7,)
    y, s = O.norm(x, w, r)
    if residual:
        O.within(out[2], s, s.abs() * O.U, dtype, "h")
    top = y.abs().amax(1)
    assert ((scale.double() - top / 448).abs() <= top / 448 * (norm_bound(dim) + 4 * O.U)).all()
    assert scale[2] == 0 and (q[2].float() == 0).all()
    step = 2.0 ** -4 * y.abs() + scale[:, None].double() * 2.0 ** -10  # half a step of e4m3, also below 2^-6
    assert ((q.double() * scale[:, None].double() - y).abs() <= step * 1.001 + y.abs() * 4 * norm_bound(dim)).all()


@DT
@pytest.mark.parametrize("dim", [1, 7, 64, 576, 1001, 2048, 4096, 8192, 8200, 20000])
@pytest.mark.parametrize("rows", [1, 6, 700])
def test_norm_backward(dtype, dim, rows):
    if rows == 700 and dim > 4096:
        rows = 150
    g = gen(dim + rows)
    h, w, gy = rand(g, rows, dim, dtype=dtype, scale=1.5), (1 + rand(g, dim, scale=0.1)).to(dtype), rand(g, rows, dim, dtype=dtype)
    gh = rand(g, rows, dim, dtype=dtype) if rows != 6 else None
    gx, gw = E.add_rms_norm_backward(gy, h, w, gh)
    (rx, sx), (rw, sw) = O.norm_backward(gy, h, w, gh)
    O.within(gx, rx, sx * 4 * norm_bound(dim), dtype, "gx")
    # a column is summed over the rows of a block, its warps, then the blocks: at most rows terms in all
    O.within(gw, rw, sw * (norm_bound(dim) + (min(rows, 200) + 80) * O.U), dtype, "gw")
    only, none = E.add_rms_norm_backward(gy, h, w, gh, weight_gradient=False)
    assert none is None and torch.equal(only, gx)


def test_norm_gradient_against_differences():
    g = gen(8)
    h, w, gy, v = rand(g, 12, 96), 1 + rand(g, 96, scale=0.1), rand(g, 12, 96), rand(g, 12, 96)
    gx, gw = E.add_rms_norm_backward(gy, h, w)
    hd, wd, d = h.double(), w.double(), 1e-5

    def loss(hh, ww):
        return (O.norm(hh, ww)[0] * gy.double()).sum()

    want = (loss(hd + d * v.double(), wd) - loss(hd - d * v.double(), wd)) / (2 * d)
    size = (gx.double() * v.double()).abs().sum()
    assert abs((gx.double() * v.double()).sum() - want) <= 1e-5 * size  # rounding of gx; d^2 of the difference
    vw = v[0]
    want = (loss(hd, wd + d * vw.double()) - loss(hd, wd - d * vw.double())) / (2 * d)
    assert abs((gw.double() * vw.double()).sum() - want) <= 1e-5 * (gw.double() * vw.double()).abs().sum()


@DT
def test_norm_strides_and_alignment(dtype):
    g = gen(4)
    wide, w = rand(g, 40, 300, dtype=dtype), (1 + rand(g, 128, scale=0.1)).to(dtype)
    r = rand(g, 128, 40, dtype=dtype).t()  # columns are not contiguous
    for x in (wide[:, :128], wide[:, 3:131], wide[::2, 5:133].repeat_interleave(2, 0), wide[:1, :128].expand(40, -1)):
        y, h = E.add_rms_norm(x, w, r)
        ry, rh = O.norm(x, w, r)
        O.within(y, ry, ry.abs() * norm_bound(128), dtype, "y")
        O.within(h, rh, rh.abs() * O.U, dtype, "h")
        gx, gw = E.add_rms_norm_backward(x, x, w, r)
        (rx, sx), (rw, sw) = O.norm_backward(x, x, w, r)
        O.within(gx, rx, sx * 4 * norm_bound(128), dtype, "gx")
        O.within(gw, rw, sw * (norm_bound(128) + 120 * O.U), dtype, "gw")
    y = E.add_rms_norm(wide.view(4, 10, 300), torch.ones(300, device="cuda", dtype=dtype))
    assert y.shape == (4, 10, 300)


def test_norm_empty_and_non_finite_rows():
    w = torch.ones(8, device="cuda")
    assert E.add_rms_norm(torch.empty(0, 8, device="cuda"), w).shape == (0, 8)
    q, s = E.add_rms_norm_q8(torch.empty(0, 8, device="cuda"), w)
    assert q.shape == (0, 8) and s.shape == (0,)
    gx, gw = E.add_rms_norm_backward(torch.empty(0, 8, device="cuda"), torch.empty(0, 8, device="cuda"), w)
    assert gx.shape == (0, 8) and (gw == 0).all()
    x = torch.ones(3, 8, device="cuda")
    x[1, 3] = float("nan")
    y = E.add_rms_norm(x, w)
    assert torch.isfinite(y[[0, 2]]).all() and torch.isnan(y[1]).all()
    q, s = E.add_rms_norm_q8(x, w)
    assert torch.isnan(s[1]) and torch.isfinite(s[[0, 2]]).all() and torch.isnan(q[1].float()).all()


@DT
def test_norm_autograd(dtype):
    g = gen(6)
    x, r, w = (rand(g, 3, 5, 64, dtype=dtype).requires_grad_() for _ in range(2)), None, None
    x, r = x
    w = (1 + rand(g, 64, scale=0.1)).to(dtype).requires_grad_()
    y, h = E.add_rms_norm(x, w, r)
    gy, gh = rand(g, 3, 5, 64, dtype=dtype), rand(g, 3, 5, 64, dtype=dtype)
    gx, gr, gw = torch.autograd.grad([y, h], [x, r, w], [gy, gh])
    want = E.add_rms_norm_backward(gy, h.detach(), w.detach(), gh)
    assert torch.equal(gx, want[0]) and torch.equal(gr, want[0]) and torch.equal(gw, want[1])
    y, h = E.add_rms_norm(x, w, r)
    (gx,) = torch.autograd.grad(h, [x], gh, retain_graph=True)  # y unused
    assert torch.equal(gx, gh)
    (gx,) = torch.autograd.grad(y, [x], gy)  # h unused
    assert torch.equal(gx, E.add_rms_norm_backward(gy, h.detach(), w.detach())[0])
    y = E.add_rms_norm(x, w)
    (gx,) = torch.autograd.grad(y, [x], gy, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(gx.sum(), [x])


def test_norm_refusals():
    x, w = torch.zeros(3, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (lambda: E.add_rms_norm(x.double(), w.double()), lambda: E.add_rms_norm(x, w[:7]),
                lambda: E.add_rms_norm(x, w.bfloat16()), lambda: E.add_rms_norm(x, w, x[:2]),
                lambda: E.add_rms_norm(x, w, x.half()), lambda: E.add_rms_norm(x, w.cpu()),
                lambda: E.add_rms_norm_q8(x.requires_grad_(), w), lambda: E.add_rms_norm_backward(x[:2], x, w)):
        with pytest.raises(RuntimeError):
            bad()


# ---- router --------------------------------------------------------------------------------------

def check_route(logits, top_k, **kw):
    weights, indices = E.route_experts(logits, top_k, **kw)
    rw, ri = O.route(logits, top_k, **kw)
    assert weights.dtype == F32 and indices.dtype == torch.int32
    assert torch.equal(indices.cpu(), ri), (indices.cpu() - ri).abs().max()
    # a score is an exponential and a quotient (each a few units, and the exponent's rounding times its
    # argument, at most 104 before it underflows), sums of `experts` terms
    assert ((weights.cpu().double() - rw).abs() <= rw.abs() * 260 * O.U + 1e-37).all()
    return weights, indices


@DT
@pytest.mark.parametrize("experts, top_k", [(1, 1), (2, 1), (7, 7), (31, 3), (64, 6), (100, 4), (256, 8), (1000, 32), (1024, 2)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route(dtype, experts, top_k, scores):
    g = gen(experts)
    logits = rand(g, 37, experts, dtype=dtype, scale=2.0)  # 16-bit logits hold many ties
    check_route(logits, top_k, scores=scores, renormalize=False, scale=2.5)
    check_route(logits, top_k, scores=scores, bias=rand(g, experts, scale=0.05))


@pytest.mark.parametrize("experts, groups, kept, top_k", [(8, 8, 3, 3), (16, 4, 1, 4), (64, 8, 4, 8), (96, 32, 5, 6),
                                                          (256, 8, 4, 8), (120, 4, 4, 5), (1024, 2, 1, 32)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_groups(experts, groups, kept, top_k, scores):
    g = gen(experts + groups)
    logits = rand(g, 41, experts, dtype=BF16)
    check_route(logits, top_k, num_groups=groups, groups_kept=kept, scores=scores)
    check_route(logits, top_k, num_groups=groups, groups_kept=kept, scores=scores, bias=rand(g, experts, scale=0.1))


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_masked_logits(scores, biased, groups):
    g = gen(11)
    logits = rand(g, 12, 40)
    inf, low = math.inf, torch.finfo(F32).min
    logits[0] = -inf                       # nothing is available
    logits[1] = float("nan")
    logits[2, :38] = -inf                  # two are, fewer than top_k
    logits[3, ::2] = float("nan")
    logits[4] = low                        # masked with the type's lowest value: all equal
    logits[5, 1:] = low
    logits[6, 7] = inf
    logits[7, 3:9] = inf
    logits[8, :20] = -inf
    logits[9] = 0.0                        # ties
    logits[10, 5] = 90.0
    logits[11] = -200.0 + logits[11]
    bias = rand(g, 40, scale=0.1) if biased else None
    if biased:
        bias[6], bias[13] = -inf, inf
    kw = dict(scores=scores, bias=bias, num_groups=groups, groups_kept=max(1, groups // 2))
    w, i = check_route(logits, 5, **kw)
    assert (i[0] == -1).all() and (w[0] == 0).all() and (i[1] == -1).all()
    mask = torch.ones(12, dtype=torch.bool, device="cuda")
    mask[[3, 9]] = False
    w, i = check_route(logits, 5, row_mask=mask, **kw)
    assert (i[3] == -1).all() and (w[9] == 0).all()
    gw = rand(g, 12, 5)
    w, i = E.route_experts(logits, 5, **kw)
    gl = E.route_experts_backward(gw, logits, i, scores=scores)
    assert torch.isfinite(gl).all() and (gl[0] == 0).all() and (gl[2, :38] == 0).all()


def test_route_half_lowest_value_and_strides():
    g = gen(12)
    wide = rand(g, 20, 200, dtype=F16)
    wide[:, 40:60] = torch.finfo(F16).min
    check_route(wide[:, 30:130], 6)
    check_route(wide[::3, :64], 6, scores="sigmoid")
    check_route(wide.t().contiguous().t()[:, :50], 3)
    assert E.route_experts(wide[:0], 4)[0].shape == (0, 4)


@DT
@pytest.mark.parametrize("experts, top_k", [(1, 1), (5, 2), (64, 6), (100, 4), (700, 9)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_backward(dtype, experts, top_k, scores, renormalize):
    g = gen(experts + 5)
    logits = rand(g, 29, experts, dtype=dtype, scale=2.0)
    kw = dict(scores=scores, renormalize=renormalize, scale=1.5)
    w, i = E.route_experts(logits, top_k, **kw)
    i[3, 0] = -1
    gw = rand(g, 29, top_k)
    gl = E.route_experts_backward(gw, logits, i, **kw)
    l = logits.double().requires_grad_()
    out = O.route_weights(l, i, scores, renormalize, 1.5)
    (want,) = torch.autograd.grad((out * gw.double()).sum(), l)
    # terms cancel: every factor is at most 1, but a score's quotient by the chosen ones' sum
    size = 1.5 * gw.double().abs().sum(1, keepdim=True) * 4
    O.within(gl, want, size * 300 * O.U, dtype, "gl")
    # differences of the formula along a direction
    v, d = rand(g, 29, experts).double(), 1e-6
    up, down = (O.route_weights(logits.double() + sgn * d * v, i, scores, renormalize, 1.5) for sgn in (1, -1))
    diff = ((up - down) / (2 * d) * gw.double()).sum()
    bound = ((O.STEP[dtype] * want.abs() + size * 300 * O.U) * v.abs()).sum() + 1e-6 * size.sum()
    assert abs((gl.double() * v).sum() - diff) <= bound


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_backward_of_one_renormalised_choice_is_zero(scores):
    """Its weight is 1 whatever the logits: g - g p / p leaves a rounding of 64 bits over p at most."""
    g = gen(14)
    logits = rand(g, 50, 40, scale=2.0)
    w, i = E.route_experts(logits, 1, scores=scores)
    assert (w == 1).all()
    gw = rand(g, 50, 1)
    gl = E.route_experts_backward(gw, logits, i, scores=scores)
    assert (gl.double().abs() <= gw.double().abs() * 2.0 ** -50).all()


def test_route_autograd():
    g = gen(13)
    logits = rand(g, 9, 16).requires_grad_()
    w, i = E.route_experts(logits, 3, scores="sigmoid", bias=rand(g, 16, scale=0.1))
    assert not i.requires_grad
    gw = rand(g, 9, 3)
    (gl,) = torch.autograd.grad(w, [logits], gw)
    assert torch.equal(gl, E.route_experts_backward(gw, logits.detach(), i, scores="sigmoid"))


def test_route_refusals():
    l = torch.zeros(3, 8, device="cuda")
    b = torch.zeros(8, device="cuda")
    for bad in (lambda: E.route_experts(l, 9), lambda: E.route_experts(l, 0), lambda: E.route_experts(l[0], 2),
                lambda: E.route_experts(l.double(), 2), lambda: E.route_experts(l, 2, scores="relu"),
                lambda: E.route_experts(l, 2, bias=b[:7]), lambda: E.route_experts(l, 2, bias=b.half()),
                lambda: E.route_experts(l, 2, bias=b.requires_grad_()), lambda: E.route_experts(l, 2, num_groups=3),
                lambda: E.route_experts(l, 2, row_mask=l[:, 0]), lambda: E.route_experts(l, 2, bias=b.detach().cpu()),
                lambda: E.route_experts(l, 3, num_groups=4, groups_kept=1),
                lambda: E.route_experts_backward(l[:, :2], l, torch.zeros(3, 2, device="cuda", dtype=torch.int64))):
        with pytest.raises(RuntimeError):
            bad()


# ---- plan ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("experts", [1, 3, 8, 100, 1024])
@pytest.mark.parametrize("rows, top_k", [(0, 2), (1, 1), (1, 8), (31, 1), (33, 3), (4096, 1), (4097, 1), (5000, 3), (16385, 1), (70001, 3), (9000, 2), (600001, 1)])
def test_plan(experts, rows, top_k):
    g = gen(rows + experts)
    idx = torch.randint(0, experts, (rows, top_k), generator=g, device="cuda").int()
    idx[rows // 2:, 0] = torch.where(torch.rand(rows - rows // 2, generator=g, device="cuda") < 0.3, -1, idx[rows // 2:, 0]).int()
    if rows > 3:
        idx[1], idx[2] = experts, 2 ** 30  # out of range: no expert
    plan = E.expert_plan(idx, experts)
    flat = idx.cpu().reshape(-1).long()
    ok = (flat >= 0) & (flat < experts)
    counts = torch.bincount(flat[ok], minlength=experts)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
    assert torch.equal(plan.offsets.cpu().long(), offsets)
    slots = ok.nonzero()[:, 0]
    want = slots[torch.sort(flat[ok], stable=True).indices]
    assert torch.equal(plan.order[:int(offsets[-1])].cpu().long(), want)
    bins = N.lib().fsc_expert_joint_bins(rows, top_k, experts)
    assert (bins > 0) == (rows >= 16 * (experts + 1) ** top_k and (experts + 1) ** top_k <= 1024)
    if bins:
        digit = torch.where((idx >= 0) & (idx < experts), idx, experts).cpu().long()
        key = (digit * (experts + 1) ** torch.arange(top_k - 1, -1, -1)).sum(1)
        tail = plan._data[experts + 2 + rows * top_k:].cpu().long()
        assert torch.equal(tail[:bins + 1], torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(key, minlength=bins).cumsum(0)]))
        assert torch.equal(tail[bins + 1:], torch.sort(key, stable=True).indices)
    plan.check()


def test_plan_is_refused_for_other_indices():
    idx = torch.zeros(4, 2, device="cuda", dtype=torch.int32)
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(3, 8, 8, device="cuda")
    plan = E.expert_plan(idx, 3)
    E.expert_linear(x, w, idx, plan=plan)
    for bad in (lambda: E.expert_linear(x, w, idx.clone(), plan=plan), lambda: E.expert_linear(x, w[:2], idx, plan=plan)):
        with pytest.raises(RuntimeError, match="plan"):
            bad()
    idx[0] = 1
    with pytest.raises(RuntimeError, match="changed in place"):
        E.expert_linear(x, w, idx, plan=plan)


# ---- the experts' products -----------------------------------------------------------------------

def routing(g, rows, experts, top_k, dead=0.2):
    """Distinct experts a row, some popular, a few slots and whole rows without one."""
    score = torch.rand(rows, experts, generator=g, device="cuda") + torch.linspace(0, 0.7, experts, device="cuda")
    idx = score.topk(top_k, 1).indices.int()
    w = torch.rand(rows, top_k, generator=g, device="cuda") + 0.1
    gone = torch.rand(rows, top_k, generator=g, device="cuda") < dead
    idx[gone] = -1
    if rows > 4:
        idx[3] = -1
    return idx, w


def check_linear(dtype, rows, experts, top_k, inputs, outputs, comps=0, slots=False, weighted=True, seed=0, grads=True, shift=0):
    g = gen(seed + rows + inputs)
    idx, wt = routing(g, rows, experts, top_k)
    mid = (comps,) if comps else ()
    n = math.prod((rows, top_k) if slots else (rows,)) * math.prod(mid) * inputs
    flat = rand(g, n + shift, dtype=dtype)  # shift: rows that do not start on 16 bytes
    x = flat[shift:].view(*((rows, top_k) if slots else (rows,)), *mid, inputs)
    dead = idx < 0
    if slots:
        x[dead] = float("nan")  # what lies in rows without an expert does not count
    else:
        x[dead.all(1)] = float("nan")
    w = rand(g, experts, outputs, inputs, dtype=dtype, scale=1 / math.sqrt(inputs))
    weights = wt if weighted else None
    if weighted:
        wt[dead] = float("nan")
    out = E.expert_linear(x, w, idx, weights, slots=slots)
    gy = rand(g, *out.shape, dtype=dtype)
    if weighted:
        gy[dead.all(1)] = float("nan")
    else:
        gy[dead] = float("nan")
    clean = torch.nan_to_num(wt) if weighted else None
    (ry, sy), (rx, sx), (rw, sw), (rt, st) = O.linear(torch.nan_to_num(x), w, idx, clean, slots, torch.nan_to_num(gy))
    O.within(out, ry, sy * O.accumulate(inputs), dtype, "out")
    if not grads:
        return
    gx, gw, gt = E.expert_linear_backward(gy, x, w, idx, weights, slots=slots)
    O.within(gx, rx, sx * O.accumulate(outputs), dtype, "gx")
    # w g is rounded to the rows' type before the product
    O.within(gw, rw, sw * (O.accumulate(rows * top_k * max(comps, 1)) + (O.STEP[dtype] if weighted else 0)), dtype, "gw")
    if weighted:
        O.within(gt, rt, st * (O.accumulate(outputs) + O.accumulate(inputs * max(comps, 1))), F32, "gt")
        assert (gt[dead] == 0).all()
    else:
        assert gt is None


@DT
@pytest.mark.parametrize("rows", [1, 2, 5, 130])
@pytest.mark.parametrize("inputs, outputs", [(64, 64), (128, 192), (40, 72)])
def test_linear(dtype, rows, inputs, outputs):
    check_linear(dtype, rows, 6, 2, inputs, outputs)


@DT
@pytest.mark.parametrize("inputs, outputs", [(1, 1), (1, 70), (33, 65), (130, 7), (67, 129), (300, 31)])
@pytest.mark.parametrize("rows", [3, 140])
def test_linear_odd_sizes(dtype, rows, inputs, outputs):
    check_linear(dtype, rows, 5, 3, inputs, outputs)


@DT
@pytest.mark.parametrize("comps", [1, 3, 9])
@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
def test_linear_forms(dtype, comps, slots, weighted):
    check_linear(dtype, 77, 4, 2, 64, 64, comps=comps, slots=slots, weighted=weighted)
    check_linear(dtype, 20, 4, 1, 48, 80, comps=comps, slots=slots, weighted=weighted)


@DT
@pytest.mark.parametrize("experts, top_k", [(1, 1), (3, 3), (64, 8), (200, 12), (1024, 32)])
def test_linear_experts(dtype, experts, top_k):
    check_linear(dtype, 50, experts, top_k, 32, 24)


@DT
def test_linear_long_contraction_and_many_rows(dtype):
    check_linear(dtype, 9, 3, 2, 2048, 136)
    check_linear(dtype, 3000, 3, 2, 64, 64)
    check_linear(dtype, 4100, 2, 1, 32, 40, comps=4)  # the weight gradient is cut into parts


@DT
@pytest.mark.parametrize("rows, top_k, comps, inputs, outputs", [
    (1, 8, 0, 2048, 130), (1, 1, 0, 1, 1), (4, 8, 0, 96, 33), (3, 2, 9, 64, 64), (2, 3, 16, 40, 12), (1, 6, 3, 100, 21),
    (32, 1, 0, 64, 5), (2, 2, 0, 4096, 16), (1, 2, 1, 12288, 3), (5, 6, 2, 37, 9)])
def test_linear_few_rows(dtype, rows, top_k, comps, inputs, outputs):
    """The matrix-vector form (up to 32 slots), all layouts; its sums are fp32 over inputs / 32 terms a lane."""
    assert E._few(rows, top_k, (comps,) if comps else (), inputs, False)
    for weighted in (True, False):
        check_linear(dtype, rows, 9, top_k, inputs, outputs, comps=comps, weighted=weighted, grads=False)
    if E._few(rows, top_k, (comps,) if comps else (), inputs, True):
        check_linear(dtype, rows, 9, top_k, inputs, outputs, comps=comps, slots=True, grads=False)


@DT
@pytest.mark.parametrize("experts, top_k, comps, inputs, outputs", [
    (2, 2, 9, 64, 64), (8, 1, 1, 32, 48), (4, 2, 3, 64, 128), (3, 2, 13, 128, 64), (2, 2, 1, 128, 128), (2, 2, 0, 33, 71),
    (2, 4, 5, 16, 24), (1, 1, 128, 64, 64), (3, 3, 2, 100, 17), (3, 1, 2, 128, 128), (1, 1, 100, 8, 128)])
def test_linear_narrow_rows_of_many_tokens(dtype, experts, top_k, comps, inputs, outputs):
    """Enough tokens for the joint grouping: every choice (missing experts among them) has some."""
    top_k = min(top_k, experts)
    rows = max(16 * (experts + 1) ** top_k + 3, 700)
    assert N.lib().fsc_expert_joint_bins(rows, top_k, experts) > 0
    check_linear(dtype, rows, experts, top_k, inputs, outputs, comps=comps)
    check_linear(dtype, rows, experts, top_k, inputs, outputs, comps=comps, weighted=False)


def test_linear_repeated_expert_of_many_tokens():
    g = gen(23)
    idx = torch.randint(-1, 3, (500, 4), generator=g, device="cuda").int()  # the same expert twice and more
    x, w, wt = rand(g, 500, 2, 40), rand(g, 3, 24, 40), torch.rand(500, 4, generator=g, device="cuda")
    assert N.lib().fsc_expert_joint_bins(500, 4, 3) == 0 and N.lib().fsc_expert_joint_bins(5000, 4, 3) == 256
    idx, x, wt = idx.repeat(10, 1), x.repeat(10, 1, 1), wt.repeat(10, 1)
    ry, sy = O.linear(x, w, idx, wt)
    O.within(E.expert_linear(x, w, idx, wt), ry, sy * O.accumulate(40), F32, "out")


@DT
def test_linear_wide_layers_of_many_rows(dtype):
    """Several row tiles an expert and feature tiles past the last feature; a weight gradient in parts."""
    check_linear(dtype, 700, 2, 2, 320, 392)
    check_linear(dtype, 530, 2, 1, 264, 129, slots=True)
    check_linear(dtype, 5000, 2, 1, 136, 24, weighted=False)


def test_linear_of_one_popular_expert():
    """All rows with one expert of many, the others without any."""
    g = gen(24)
    idx = torch.full((600, 1), 37, device="cuda", dtype=torch.int32)
    x, w = rand(g, 600, 200, dtype=BF16), rand(g, 64, 260, 200, dtype=BF16)
    plan = E.expert_plan(idx, 64)
    y = E.expert_linear(x, w, idx, plan=plan)[:, 0]
    want = x.double() @ w[37].double().T
    O.within(y, want, (x.double().abs() @ w[37].double().abs().T) * O.accumulate(200), BF16, "y")
    gx, gw, _ = E.expert_linear_backward(y[:, None], x, w, idx, plan=plan)
    assert (gw[:37] == 0).all() and (gw[38:] == 0).all() and (gw[37] != 0).any()
    plan.check()


def test_linear_layouts_of_the_arguments():
    """Transposed indices and weights, expanded and sliced rows, and a call without grad mode or in inference mode."""
    g = gen(25)
    idx, wt = routing(g, 70, 5, 2)
    x, w = rand(g, 70, 64), rand(g, 5, 64, 64)
    want = E.expert_linear(x, w, idx, wt)
    it, tt = idx.t().contiguous().t(), wt.t().contiguous().t()
    assert torch.equal(E.expert_linear(x, w, it, tt, plan=E.expert_plan(it, 5)), want)
    wide = torch.zeros(70, 100, device="cuda")
    wide[:, 3:67] = x
    assert torch.equal(E.expert_linear(wide[:, 3:67], w.transpose(1, 2).contiguous().transpose(1, 2), idx, wt), want)
    one = x[:1].expand(70, -1)
    assert torch.equal(E.expert_linear(one, w, idx, wt), E.expert_linear(one.contiguous(), w, idx, wt))
    with torch.inference_mode():
        a, b, c, d = x.clone(), w.clone(), idx.clone(), wt.clone()
        assert torch.equal(E.expert_linear(a, b, c, d, plan=E.expert_plan(c, 5)), want)


@DT
@pytest.mark.parametrize("shift", [1, 4])
def test_linear_alignment(dtype, shift):
    check_linear(dtype, 40, 4, 2, 64, 64, shift=shift)


@DT
def test_linear_repeated_expert_and_out_of_range(dtype):
    g = gen(20)
    idx = torch.tensor([[1, 1], [0, 1], [7, 0], [-5, 2 ** 30]], device="cuda", dtype=torch.int32)
    x, w, wt = rand(g, 4, 64, dtype=dtype), rand(g, 2, 32, 64, dtype=dtype), torch.rand(4, 2, generator=g, device="cuda")
    ry, sy = O.linear(x, w, idx, wt)
    out = E.expert_linear(x, w, idx, wt)
    O.within(out, ry, sy * O.accumulate(64), dtype, "out")
    assert (out[3] == 0).all()


def test_linear_empty():
    x, w = torch.empty(0, 16, device="cuda"), torch.ones(3, 8, 16, device="cuda")
    idx, wt = torch.empty(0, 2, device="cuda", dtype=torch.int32), torch.empty(0, 2, device="cuda")
    assert E.expert_linear(x, w, idx, wt).shape == (0, 8) and E.expert_linear(x, w, idx).shape == (0, 2, 8)
    gx, gw, gt = E.expert_linear_backward(torch.empty(0, 8, device="cuda"), x, w, idx, wt)
    assert gx.shape == (0, 16) and (gw == 0).all() and gt.shape == (0, 2)
    none = torch.full((5, 2), -1, device="cuda", dtype=torch.int32)
    x = torch.full((5, 16), float("nan"), device="cuda")
    y = E.expert_linear(x, w, none, torch.ones(5, 2, device="cuda"))
    assert (y == 0).all()
    gx, gw, gt = E.expert_linear_backward(y, x, w, none, torch.ones(5, 2, device="cuda"))
    assert (gx == 0).all() and (gw == 0).all() and (gt == 0).all()


def test_linear_32_bit_range():
    """Values near the largest and smallest floats survive the split into three bfloat16."""
    big = torch.finfo(F32).max
    x = torch.tensor([[big, 0.0], [1e-30, 0.0], [-big, 0.0], [1.0, 2.0 ** -23]], device="cuda")
    w = torch.tensor([[[1.0, 0.0], [0.5, 1.0]]], device="cuda")
    y = E.expert_linear(x, w, torch.zeros(4, 1, device="cuda", dtype=torch.int32))[:, 0]
    want = x.double() @ w[0].double().T
    assert ((y.double() - want).abs() <= want.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, top_k, inputs, outputs", [(1, 1, 16, 16), (5, 2, 100, 33), (150, 3, 256, 200), (60, 2, 2048, 128)])
@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("weighted", [False, True])
def test_linear_8_bits(out_dtype, rows, top_k, inputs, outputs, slots, weighted):
    g = gen(rows)
    idx, wt = routing(g, rows, 5, top_k)
    x, xs = E.add_rms_norm_q8(rand(g, *((rows, top_k) if slots else (rows,)), inputs), torch.ones(inputs, device="cuda"))
    w, ws = E.quantize_experts(rand(g, 5, outputs, inputs))
    y = E.expert_linear_q8(x, xs, w, ws, idx, wt if weighted else None, slots=slots, out_dtype=out_dtype)
    ry, sy = O.linear(x.double() * xs[..., None].double(), w.double() * ws[..., None].double(), idx,
                      wt if weighted else None, slots)
    O.within(y, ry, sy * O.accumulate(inputs), out_dtype, "y")


def test_linear_gradient_against_differences():
    g = gen(21)
    idx, wt = routing(g, 30, 4, 2, dead=0.1)
    x, w, gy = rand(g, 30, 3, 24), rand(g, 4, 20, 24), rand(g, 30, 3, 20)
    gx, gw, gt = E.expert_linear_backward(gy, x, w, idx, wt)
    vx, vw, vt = rand(g, 30, 3, 24).double(), rand(g, 4, 20, 24).double(), rand(g, 30, 2).double()

    def loss(s):
        return (O.linear(x.double() + s * vx, w.double() + s * vw, idx, wt.double() + s * vt)[0].reshape(gy.shape) * gy.double()).sum()

    d = 1e-4
    want = (loss(d) - loss(-d)) / (2 * d)  # trilinear: the rest is d^2 times one term
    terms = [(a.double() * b) for a, b in ((gx, vx), (gw, vw), (gt, vt))]
    size = sum(t.abs().sum() for t in terms)
    assert abs(sum(t.sum() for t in terms) - want) <= 1e-5 * size


@DT
def test_linear_autograd(dtype):
    g = gen(22)
    idx, wt = routing(g, 25, 4, 2)
    x, w = rand(g, 25, 64, dtype=dtype).requires_grad_(), rand(g, 4, 32, 64, dtype=dtype).requires_grad_()
    wt.requires_grad_()
    plan = E.expert_plan(idx, 4)
    y = E.expert_linear(x, w, idx, wt, plan=plan)
    gy = rand(g, 25, 32, dtype=dtype)
    got = torch.autograd.grad(y, [x, w, wt], gy)
    want = E.expert_linear_backward(gy, x.detach(), w.detach(), idx, wt.detach())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    h = E.expert_linear(x, w, idx)  # an expert MLP's first product, its activation, and the second
    z = E.expert_linear(torch.nn.functional.silu(h), w.transpose(1, 2), idx, wt, slots=True)
    gx, gw, gt = torch.autograd.grad(z, [x, w, wt], rand(g, 25, 64, dtype=dtype))
    assert gx.shape == x.shape and gw.shape == w.shape and torch.isfinite(gx).all() and torch.isfinite(gw).all()
    (g1,) = torch.autograd.grad(E.expert_linear(x, w, idx, wt), [x], gy, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(g1.sum(), [x])


def test_linear_refusals():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(3, 6, 8, device="cuda")
    i, f = torch.zeros(4, 2, device="cuda", dtype=torch.int32), torch.zeros(4, 2, device="cuda")
    q = torch.zeros(4, 8, device="cuda").to(torch.float8_e4m3fn)
    wq, ws = E.quantize_experts(w)
    for bad in (lambda: E.expert_linear(x, w.half(), i), lambda: E.expert_linear(x, w, i.long()),
                lambda: E.expert_linear(x, w, i[:3]), lambda: E.expert_linear(x[:, :7], w, i),
                lambda: E.expert_linear(x, w[0], i), lambda: E.expert_linear(x, w, i, f.half()),
                lambda: E.expert_linear(x, w, i, f[:, :1]), lambda: E.expert_linear(x, w, i, f, slots=True),
                lambda: E.expert_linear(x, w, i.cpu()), lambda: E.expert_linear(x.double(), w.double(), i),
                lambda: E.expert_linear(x, w, torch.zeros(4, 33, device="cuda", dtype=torch.int32)),
                lambda: E.expert_linear_backward(x, x, w, i, f), lambda: E.expert_plan(i, 0), lambda: E.expert_plan(i, 1025),
                lambda: E.expert_linear_q8(q, f[:, 0], wq, ws, i, f, out_dtype=torch.float64),
                lambda: E.expert_linear_q8(q, f, wq, ws, i, f), lambda: E.expert_linear_q8(x, f[:, 0], wq, ws, i, f),
                lambda: E.expert_linear_q8(q, f[:, 0], wq, ws[:2], i, f),
                lambda: E.expert_linear_q8(q, f[:, 0], wq, ws, i, f.requires_grad_())):
        with pytest.raises(RuntimeError):
            bad()


# ---- together ------------------------------------------------------------------------------------

def block(x, r, wn, wr, we, top_k):
    """Norm, router, experts as a program runs them, and the gradients by the explicit functions."""
    y, h = E.add_rms_norm(x, wn, r)
    logits = y @ wr.t()
    wt, idx = E.route_experts(logits, top_k)
    plan = E.expert_plan(idx, we.shape[0])
    z = E.expert_linear(y, we, idx, wt, plan=plan)
    gy, gwe, gwt = E.expert_linear_backward(z, y, we, idx, wt, plan=plan)
    gl = E.route_experts_backward(gwt, logits, idx)
    gy = gy + gl @ wr
    gx, gwn = E.add_rms_norm_backward(gy, h, wn, z)
    return z, h, gx, gwn, gwe


def block_inputs(seed, rows=96, dim=64, experts=6):
    g = gen(seed)
    return (rand(g, rows, dim), rand(g, rows, dim), 1 + rand(g, dim, scale=0.1), rand(g, experts, dim, scale=0.2),
            rand(g, experts, dim, dim, scale=0.125))


def test_block_matches_autograd_in_64_bits():
    x, r, wn, wr, we = block_inputs(30)
    z, h, gx, gwn, gwe = block(x, r, wn, wr, we, 2)
    idx = E.route_experts(E.add_rms_norm(x, wn, r)[0] @ wr.t(), 2)[1].long()
    leaves = [t.double().requires_grad_() for t in (x, wn, we)]
    s = leaves[0] + r.double()
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + 1e-6) * leaves[1]
    p = torch.softmax(y @ wr.double().t(), 1).gather(1, idx)
    p = p / p.sum(1, keepdim=True)
    zr = torch.einsum("tk,tkoi,ti->to", p, leaves[2][idx], y)
    grads = torch.autograd.grad([zr, s], leaves, [z.double(), z.double()])
    # the chain's sums have at most 96 terms of the results' size; 1e-5 is 170 roundings of each
    for got, want in ((z, zr), (h, s), (gx, grads[0]), (gwn, grads[1]), (gwe, grads[2])):
        assert (got.double() - want).abs().max() <= 1e-5 * want.abs().max()


def test_equal_calls_give_equal_bits():
    first = block(*block_inputs(31, rows=3000), 2)
    again = block(*block_inputs(31, rows=3000), 2)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_other_stream_and_two_captured_graphs():
    """Two graphs captured from the same program and an eager run in between keep their own workspaces."""
    ins = [block_inputs(s) for s in (32, 33)]
    want = [block(*i, 2) for i in ins]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = block(*ins[0], 2)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))
    static = [tuple(t.clone() for t in i) for i in ins]
    graphs = []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = block(*s, 2)
        graphs.append((g, out))
    for k in (0, 1, 0):  # replay each with the other's inputs, then its own
        for a, b in zip(static[k], ins[1 - k]):
            a.copy_(b)
        graphs[k][0].replay()
        block(*ins[k], 2)
        assert all(torch.equal(a, b) for a, b in zip(graphs[k][1], want[1 - k]))
        for a, b in zip(static[k], ins[k]):
            a.copy_(b)
        graphs[k][0].replay()
        assert all(torch.equal(a, b) for a, b in zip(graphs[k][1], want[k]))


def test_channel_mix_keeps_an_empty_block_empty():
    """The o3 model's 1e block is identically zero and stays so."""
    torch.manual_seed(1)
    mix = E.RoutedChannelMix(32, num_experts=4, top_k=2, degrees=(0, 1, 1, 2)).cuda()
    f = torch.randn(40, 32 * 12, device="cuda")
    f[:, 32:32 + 96] = 0
    out = mix(f)
    assert out.shape == f.shape and (out[:, 32:32 + 96] == 0).all() and torch.isfinite(out).all()
    out.square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in mix.parameters())


def test_channel_mix_is_equivariant_and_the_models_hook():
    """RoutedChannelMix as a model's sync_after_scatter: forces against energy differences."""
    from test_gpu_hooks import _args, _model

    m, c, cfg = _model("ictd")
    channels = int(cfg["channels"])
    torch.manual_seed(0)
    mix = E.RoutedChannelMix(channels, num_experts=4, top_k=2, layers=2).cuda()
    with torch.no_grad():
        mix.router.mul_(0.05)
        mix.experts.mul_(0.3)
    # rotations act on each block's components; any orthogonal matrix per block commutes with the layer
    f = torch.randn(31, channels * 9, device="cuda")
    q = [torch.linalg.qr(torch.randn(k, k, dtype=torch.float64))[0].float().cuda() for k in (3, 5)]
    rows = mix._to_rows(f)
    turned = torch.cat([rows[:, :1], torch.einsum("ab,nbc->nac", q[0], rows[:, 1:4]),
                        torch.einsum("ab,nbc->nac", q[1], rows[:, 4:])], 1)
    out, out2 = mix._to_rows(mix(f)), mix._to_rows(mix(mix._from_rows(turned)))
    want = torch.cat([out[:, :1], torch.einsum("ab,nbc->nac", q[0], out[:, 1:4]),
                      torch.einsum("ab,nbc->nac", q[1], out[:, 4:])], 1)
    assert (out2 - want).abs().max() <= 1e-4 * want.abs().max()

    pos = torch.tensor(c["pos"], device="cuda", dtype=torch.float32)
    args = _args(c, torch.device("cuda"))

    def energy(p):
        return m(p, *args, sync_after_scatter=mix).sum()

    p = pos.clone().requires_grad_()
    (grad,) = torch.autograd.grad(energy(p), [p])
    plain = pos.clone().requires_grad_()
    (without,) = torch.autograd.grad(m(plain, *args).sum(), [plain])
    assert (grad - without).abs().max() > 1e-3 * without.abs().max()  # the layer acts
    v = torch.randn(pos.shape, generator=gen(40), device="cuda")
    v = v * (grad.abs() + grad.abs().mean()) * grad.sign()  # along the gradient, so that nothing cancels
    v = v.abs() * grad.sign()
    d = 2e-3 / v.abs().max()
    with torch.no_grad():
        diff = (energy(pos + d * v).double() - energy(pos - d * v).double()) / (2 * d)
    want = (grad.double() * v.double()).sum()
    # fp32 energies of size |E| carry about 1e-6 |E|; the displacement of 2e-3 leaves a second-order rest
    noise = 2e-6 * abs(energy(pos).item()) / d
    assert abs(diff - want) <= noise + 2e-2 * abs(want)
