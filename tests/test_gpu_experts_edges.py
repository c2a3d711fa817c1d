"""Routed-expert operators at the edges of what their documentation allows, against the 64-bit statements."""

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


# ---- router --------------------------------------------------------------------------------------

@DT
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("experts", [4, 40, 300, 700])
def test_route_takes_zeros_of_either_sign_as_equal(dtype, scores, biased, experts):
    """Logits of 0.0 and -0.0 have the same score: the lowest index comes first, also at the border of the top-k."""
    logits = torch.zeros(6, experts, device="cuda", dtype=dtype)
    logits[0, 0] = -0.0
    logits[1] = -0.0
    logits[2, ::2] = -0.0
    logits[3, 1::2] = -0.0
    logits[4, :2], logits[4, -1] = -0.0, -1.0
    logits[5, 1:] = -0.0
    logits[5, 2] = 1.0
    bias = torch.zeros(experts, device="cuda") if biased else None
    for top_k in (1, 2, 3):
        weights, indices = E.route_experts(logits, top_k, scores=scores, bias=bias)
        want_w, want_i = O.route(logits, top_k, scores=scores, bias=bias)
        assert torch.equal(indices.cpu(), want_i)
        assert indices[0].tolist() == list(range(top_k)) and indices[5].tolist() == [2, 0, 1][:top_k]
        assert ((weights.cpu().double() - want_w).abs() <= want_w * 260 * O.U).all()


# ---- the experts' products -----------------------------------------------------------------------

def at_16(t):
    """A copy of ``t`` that starts on 16 bytes and not on 32."""
    flat = torch.empty(t.numel() * t.element_size() + 64, device="cuda", dtype=torch.uint8)
    return flat[16:16 + t.numel() * t.element_size()].view(t.dtype).view(t.shape).copy_(t)


@DT
@pytest.mark.parametrize("rows, experts, top_k, inputs, outputs", [
    (70, 6, 2, 64, 192), (70, 6, 1, 640, 72), (70, 6, 2, 648, 1024), (40, 6, 4, 64, 520), (1300, 3, 2, 64, 48)])
def test_linear_with_all_pointers_on_16_bytes_only(dtype, rows, experts, top_k, inputs, outputs):
    """Sixteen bytes are what the C interface asks of its pointers, the workspace among them."""
    g = gen(rows + inputs)
    idx = torch.rand(rows, experts, generator=g, device="cuda").topk(top_k, 1).indices.int()
    idx[3] = -1
    wt = torch.rand(rows, top_k, generator=g, device="cuda")
    x, w = rand(g, rows, inputs, dtype=dtype), rand(g, experts, outputs, inputs, dtype=dtype)
    gy = rand(g, rows, outputs, dtype=dtype)
    plan = E.expert_plan(idx, experts)
    want = [E.expert_linear(x, w, idx, wt, plan=plan), *E.expert_linear_backward(gy, x, w, idx, wt, plan=plan)]
    lib, dt, stream = N.lib(), E._DTYPES[dtype], torch.cuda.current_stream().cuda_stream
    x, w, gy = at_16(x), at_16(w), at_16(gy)
    out, gx, gw = (at_16(torch.zeros_like(t)) for t in want[:3])
    gt = torch.zeros_like(wt)
    joint = plan._joint_offsets is not None
    need = lib.fsc_expert_linear_workspace_bytes(dt, rows, top_k, 1, experts, inputs, outputs, 0, 1, joint)
    ws = at_16(torch.zeros(max(need, 1), device="cuda", dtype=torch.uint8))
    assert all(t.data_ptr() % 32 == 16 for t in (x, w, gy, out, gx, gw, ws))
    groups = (plan._offsets, plan._order, plan._joint_offsets, plan._joint_order, plan._status)
    assert lib.fsc_expert_linear(dt, x.data_ptr(), w.data_ptr(), idx.data_ptr(), wt.data_ptr(), *groups, out.data_ptr(),
                                 rows, top_k, 1, experts, inputs, outputs, 0, ws.data_ptr(), need, stream) == 0
    need = lib.fsc_expert_linear_backward_workspace_bytes(dt, rows, top_k, 1, experts, inputs, outputs, 0, 1, 1, 1, joint)
    ws = at_16(torch.zeros(need, device="cuda", dtype=torch.uint8))
    assert lib.fsc_expert_linear_backward(dt, gy.data_ptr(), x.data_ptr(), w.data_ptr(), idx.data_ptr(), wt.data_ptr(),
                                          *groups, gx.data_ptr(), gw.data_ptr(), gt.data_ptr(), rows, top_k, 1, experts,
                                          inputs, outputs, 0, ws.data_ptr(), need, stream) == 0
    assert all(torch.equal(a, b) for a, b in zip(want, (out, gx, gw, gt)))
    plan.check()


# ---- derivatives that there are not --------------------------------------------------------------

def test_forward_mode_is_refused():
    from torch.autograd import forward_ad

    g = gen(1)
    x, weight, logits = rand(g, 4, 16), rand(g, 16), rand(g, 4, 3)
    w, wt = rand(g, 3, 8, 16), torch.rand(4, 2, generator=g, device="cuda")
    idx = torch.zeros(4, 2, device="cuda", dtype=torch.int32)
    q, qs = E.quantize_experts(w)
    xq, xs = E.add_rms_norm_q8(x, weight)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: E.add_rms_norm(dual(x), weight), lambda: E.add_rms_norm(x, dual(weight)),
                 lambda: E.add_rms_norm(x, weight, dual(x)), lambda: E.add_rms_norm_q8(dual(x), weight),
                 lambda: E.route_experts(dual(logits), 2), lambda: E.route_experts(logits, 2, bias=dual(logits[0])),
                 lambda: E.expert_linear(dual(x), w, idx, wt), lambda: E.expert_linear(x, dual(w), idx),
                 lambda: E.expert_linear(x, w, idx, dual(wt)), lambda: E.expert_linear_q8(xq, xs, q, qs, idx, dual(wt)),
                 lambda: E.expert_linear_q8(xq, dual(xs), q, qs, idx), lambda: E.expert_linear_q8(xq, xs, q, dual(qs), idx),
                 lambda: E.add_rms_norm_backward(x, dual(x), weight), lambda: E.route_experts_backward(dual(wt), logits, idx),
                 lambda: E.expert_linear_backward(dual(x[:, :8]), x, w, idx, wt)]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert E.add_rms_norm(x, weight).shape == x.shape  # a call without a tangent runs
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: E.add_rms_norm(t, weight), (x,), (x,))


# ---- two host threads ----------------------------------------------------------------------------

def in_threads(*jobs, turns=3000):
    """Each job over and over in a thread and on a stream of its own; what they returned last, or the first error."""
    import threading

    start, errors, last = threading.Barrier(len(jobs)), [], [None] * len(jobs)

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(turns):
                    last[i] = jobs[i]()
                    if errors:
                        break
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if errors:
        raise errors[0]
    return last


def test_threads_with_plans_of_different_sizes():
    """A launch's shared memory is its own: a smaller plan in another thread does not lower the larger one's."""
    lib, g = N.lib(), gen(2)

    def job(experts):
        idx = torch.randint(0, experts, (64, 1), generator=g, device="cuda").int()
        out = torch.zeros(experts + 2 + 64, device="cuda", dtype=torch.int32)
        at = out.data_ptr()

        def call():
            stream = torch.cuda.current_stream().cuda_stream
            for _ in range(10):
                N.check(lib.fsc_expert_plan(idx.data_ptr(), 64, 1, experts, at, at + 4 * (experts + 2), None, None,
                                            at + 4 * (experts + 1), None, 0, stream), "expert_plan")
            return out, idx
        return call

    for out, idx in in_threads(job(1024), job(400)):
        experts = out.shape[0] - 2 - 64
        assert torch.equal(out[experts + 2:].long(), torch.sort(idx[:, 0], stable=True).indices)


def test_threads_with_products_of_different_sizes():
    """The same for the products of few rows and of narrow rows."""
    g = gen(3)

    def few(slots):
        x = rand(g, 1, 3 * 4096)
        w = rand(g, 2, 24, 3 * 4096)
        idx = torch.zeros(1, slots, device="cuda", dtype=torch.int32)
        want = E.expert_linear(x, w, idx)
        return lambda: (E.expert_linear(x, w, idx), want)

    def joint(top_k):
        idx = torch.rand(1000, 2, generator=g, device="cuda").topk(top_k, 1).indices.int()
        x, w, wt = rand(g, 1000, 64), rand(g, 2, 64, 64), torch.rand(1000, top_k, generator=g, device="cuda")
        plan = E.expert_plan(idx, 2)
        torch.cuda.synchronize()
        want = E.expert_linear(x, w, idx, wt, plan=plan)
        return lambda: (E.expert_linear(x, w, idx, wt, plan=plan), want)

    for jobs in ((few(1), few(32)), (joint(1), joint(2))):
        for got, want in in_threads(*jobs, turns=2000):
            assert torch.equal(got, want)


# ---- the gradient in the experts' weights --------------------------------------------------------

def weight_gradient_bound(rows):
    """Beside the result's own rounding, of the terms' magnitudes: a row times its weight is the sum of two bfloat16 to
    2^-16; of fp16 rows the product of the two second parts is left out, 2^-7 * 2^-8 of the term; the sums are those of
    the oracle's bound with three products for each sixteen rows."""
    return 2.0 ** -16 + 2.0 ** -15 + (3 * (rows // 16 + 2) + 8) * 2.0 ** -23


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows, experts, top_k, inputs, outputs, comps, slots", [
    (300, 3, 2, 64, 64, 1, False), (200, 2, 1, 72, 200, 1, False), (257, 2, 2, 300, 40, 1, True), (90, 2, 2, 33, 17, 5, False),
    (90, 2, 2, 136, 264, 3, True), (4200, 2, 1, 32, 40, 1, False), (40, 1, 1, 7, 9, 1, False)])
def test_weight_gradient_keeps_more_bits_than_the_rows_have(dtype, rows, experts, top_k, inputs, outputs, comps, slots):
    """One rounding, the result's: the product of a row and its weight is not rounded to 16 bits before the sum."""
    g = gen(rows + outputs)
    idx = torch.rand(rows, experts, generator=g, device="cuda").topk(top_k, 1).indices.int()
    idx[1] = -1
    wt = torch.rand(rows, top_k, generator=g, device="cuda") + 0.1
    # terms of one sign: all that is cut adds up
    x = rand(g, *((rows, top_k) if slots else (rows,)), comps, inputs, dtype=dtype).abs()
    gy = rand(g, rows, comps, outputs, dtype=dtype).abs()
    w = rand(g, experts, outputs, inputs, dtype=dtype)
    _, got, _ = E.expert_linear_backward(gy, x, w, idx, wt, slots=slots, input_gradient=False, routing_gradient=False)
    want, size = O.linear(x, w, idx, wt, slots, gy)[2]
    O.within(got, want, size * weight_gradient_bound(rows * top_k * comps), dtype, "gw")
    # every term with one of nearly the same size and the other sign: the result is a hundredth of its terms
    both = torch.cat([x, -x]), torch.cat([gy, gy]), torch.cat([idx, idx]), torch.cat([wt, wt * 1.01])
    _, got, _ = E.expert_linear_backward(both[1], both[0], w, both[2], both[3], slots=slots)
    want, size = O.linear(both[0], w, both[2], both[3], slots, both[1])[2]
    O.within(got, want, size * weight_gradient_bound(2 * rows * top_k * comps), dtype, "gw of pairs")


@pytest.mark.parametrize("factor, size, grad", [(1e-5, 1.0, 1000.0), (3e-8, 1.0, 1000.0), (40.0, 1000.0, 1e-3), (1000.0, 1000.0, 1e-4)])
@pytest.mark.parametrize("outputs", [24, 200])
def test_weight_gradient_of_f16_rows_beyond_the_range_of_f16(factor, size, grad, outputs):
    """weight * x below 6e-5 is subnormal in fp16 and above 65504 infinite; the sum of its products with g is neither."""
    g = gen(outputs)
    rows, inputs = 150, 136
    idx = torch.randint(0, 2, (rows, 1), generator=g, device="cuda").int()
    wt = (torch.rand(rows, 1, generator=g, device="cuda") + 0.5) * factor
    x, gy = rand(g, rows, inputs, scale=size, dtype=F16), rand(g, rows, outputs, scale=grad, dtype=F16)
    if factor == 40.0:
        x[::7, ::5] = 60000.0
    w = rand(g, 2, outputs, inputs, dtype=F16)
    _, got, _ = E.expert_linear_backward(gy, x, w, idx, wt, input_gradient=False, routing_gradient=False)
    want, sizes = O.linear(x, w, idx, wt, False, gy)[2]
    assert 1e-5 < want.abs().median() and want.abs().max() < 65504
    O.within(got, want, sizes * weight_gradient_bound(rows), F16, "gw")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_weight_gradient_without_weights_is_exact_to_its_rounding(dtype):
    g = gen(31)
    idx = torch.randint(-1, 3, (200, 2), generator=g, device="cuda").int()
    x, w, gy = rand(g, 200, 72, dtype=dtype), rand(g, 3, 56, 72, dtype=dtype), rand(g, 200, 2, 56, dtype=dtype)
    _, got, _ = E.expert_linear_backward(gy, x, w, idx)
    want, size = O.linear(x, w, idx, None, False, gy)[2]
    O.within(got, want, size * O.accumulate(400), dtype, "gw")


# ---- a bounded wait that ran out -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows, inputs, outputs, joint", [(90, 72, 40, False), (150, 200, 328, False), (600, 64, 48, True)])
def test_products_of_a_failed_plan_are_nan(dtype, rows, inputs, outputs, joint):
    """The status word is set by hand, as a kernel whose wait ran out leaves it: the next products begin no work and
    write NaN for every slot with an expert; slots without one stay zero, and a new plan works again."""
    g = gen(rows)
    idx = torch.randint(0, 2, (rows, 2), generator=g, device="cuda").int()
    idx[5] = -1
    x, w, wt = rand(g, rows, inputs, dtype=dtype), rand(g, 2, outputs, inputs, dtype=dtype), torch.rand(rows, 2, generator=g, device="cuda")
    gy = rand(g, rows, outputs, dtype=dtype)
    plan = E.expert_plan(idx, 2)
    assert (plan._joint_offsets is not None and max(inputs, outputs) <= 128) == joint  # the narrow rows' kernel
    want = [E.expert_linear(x, w, idx, wt, plan=plan), *E.expert_linear_backward(gy, x, w, idx, wt, plan=plan)]
    plan.check()
    plan._data[3] = 3
    live = torch.arange(rows, device="cuda") != 5
    y = E.expert_linear(x, w, idx, wt, plan=plan)
    apart = E.expert_linear(x, w, idx, plan=plan)
    gx, gw, gt = E.expert_linear_backward(gy, x, w, idx, wt, plan=plan)
    assert torch.isnan(gw).all()
    for t in (y, apart, gx, gt):
        assert torch.isnan(t[live]).all()
    assert (apart[5] == 0).all() and (gt[5] == 0).all()
    if not joint:  # the narrow rows' kernel owns every token, also those without an expert
        assert (y[5] == 0).all() and (gx[5] == 0).all()
    (gw_apart,) = E.expert_linear_backward(torch.stack([gy, gy], 1), x, w, idx, plan=plan, input_gradient=False)[1:2]
    assert torch.isnan(gw_apart).all()
    with pytest.raises(N.NativeError, match="wait ran out"):
        plan.check()
    plan = E.expert_plan(idx, 2)
    again = [E.expert_linear(x, w, idx, wt, plan=plan), *E.expert_linear_backward(gy, x, w, idx, wt, plan=plan)]
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    plan.check()


def test_8_bit_products_of_a_failed_plan_are_nan():
    g = gen(9)
    idx = torch.randint(0, 3, (50, 2), generator=g, device="cuda").int()
    x, xs = E.add_rms_norm_q8(rand(g, 50, 64), torch.ones(64, device="cuda"))
    w, ws = E.quantize_experts(rand(g, 3, 200, 64))
    plan = E.expert_plan(idx, 3)
    plan._data[4] = 2
    for weights in (None, torch.ones(50, 2, device="cuda")):
        for out_dtype in (F32, BF16):
            assert torch.isnan(E.expert_linear_q8(x, xs, w, ws, idx, weights, plan=plan, out_dtype=out_dtype)).all()


# ---- norm ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim", [7, 64, 1000, 4096, 9001])
@pytest.mark.parametrize("size, eps", [(1e14, 1e-6), (1e16, 1e-6), (1e-13, 0.0), (1e-14, 1e-32), (1e-16, 1e-34)])
def test_norm_gradient_of_large_and_small_rows(dtype, dim, size, eps):
    """1 / rms cubed leaves the range of fp32 where the gradient does not."""
    g = gen(dim)
    h, w, gy = rand(g, 9, dim, scale=size, dtype=dtype), (1 + rand(g, dim, scale=0.1)).to(dtype), rand(g, 9, dim, dtype=dtype)
    gy = (gy * size).to(dtype)  # a gradient of about one
    gx, gw = E.add_rms_norm_backward(gy, h, w, eps=eps)
    (rx, sx), (rw, sw) = O.norm_backward(gy, h, w, eps=eps)
    bound = (dim / 64 + 60) * O.U  # as of rows of ordinary size
    O.within(gx, rx, sx * 4 * bound, dtype, "gx")
    O.within(gw, rw, sw * (bound + 100 * O.U), dtype, "gw")
    y, _ = O.norm(h, w, eps=eps)
    O.within(E.add_rms_norm(h, w, eps=eps), y, y.abs() * bound, dtype, "y")


# ---- the layer -----------------------------------------------------------------------------------

@pytest.mark.parametrize("layers", [1, 2])
def test_channel_mix_of_no_atoms(layers):
    mix = E.RoutedChannelMix(16, 4, 2, layers=layers).cuda()
    f = torch.empty(0, 16 * 9, device="cuda", requires_grad=True)
    out = mix(f)
    assert out.shape == (0, 16 * 9)
    out.sum().backward()
    assert f.grad.shape == f.shape and all((p.grad == 0).all() for p in mix.parameters())


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_channel_mix_in_16_bits(dtype):
    """The layer converted as a whole; against itself in 32 bits on the same (rounded) parameters."""
    torch.manual_seed(3)
    mix = E.RoutedChannelMix(32, 4, 2).cuda().to(dtype)
    f = torch.randn(50, 32 * 9, device="cuda").to(dtype).requires_grad_()
    out = mix(f)
    assert out.dtype == dtype and torch.isfinite(out).all()
    out.float().square().sum().backward()
    assert all(p.grad.dtype == dtype and torch.isfinite(p.grad).all() for p in mix.parameters())
    wide = E.RoutedChannelMix(32, 4, 2).cuda()
    wide.load_state_dict({k: v.float() for k, v in mix.state_dict().items()})
    want = wide(f.detach().float())
    # rows whose two best scores are apart by more than the logits' rounding meet the same experts
    rows = wide._to_rows(f.detach().float())
    y = E.add_rms_norm(rows.reshape(50, -1), wide.norm[0][wide.block].reshape(-1))
    score = (y[:, :32] @ wide.router[0].t()).sort(1, descending=True).values
    sure = score[:, 1] - score[:, 2] > 0.1
    assert sure.sum() > 25
    # roundings of y, of the logits (weights move by at most their error), of the products and of the sum, each half a
    # step of values of up to the rows' largest
    got = out.detach().float()[sure]
    assert (got - want[sure]).abs().max() <= 8 * O.STEP[dtype] * want[sure].abs().max()


# ---- sums on the tensor cores that are taken over into registers -----------------------------------

def promoted(terms):
    """Relative bound of fp32 results: an accumulator runs for 256 terms (16 instructions for the large products, each of
    which cuts the running sum at 2^-23; five times as many for the small ones, 2^-7 of it) and is then added to the
    register's sum (2^-24 each).  Of a product's nine parts the three from 2^-24 on are left out: with parts cut after
    eight bits they are at most 2^-22 of it together and once more 2^-23.  Up to 64 parts of rows are added at the end."""
    return (16 + 1 + 5 * 16 * 2.0 ** -7 + 4) * 2.0 ** -23 + (terms / 256 + 2) * O.U


@pytest.mark.parametrize("rows, inputs, outputs, top_k", [(70, 4096, 40, 1), (40, 16384, 24, 1), (130, 2048, 200, 2), (20000, 40, 24, 1)])
def test_32_bit_sums_of_one_sign(rows, inputs, outputs, top_k):
    """Terms of one sign, so that every cut adds up: only short accumulators keep these bounds."""
    g = gen(rows)
    idx = torch.rand(rows, 2, generator=g, device="cuda").topk(top_k, 1).indices.int()
    x, w = rand(g, rows, inputs).abs() + 0.1, rand(g, 2, outputs, inputs).abs() + 0.1
    wt, gy = torch.rand(rows, top_k, generator=g, device="cuda") + 0.1, rand(g, rows, outputs).abs() + 0.1
    y = E.expert_linear(x, w, idx, wt)
    gx, gw, gt = E.expert_linear_backward(gy, x, w, idx, wt)
    slots = E.expert_linear(x, w, idx)
    gws = E.expert_linear_backward(gy[:, None].expand(-1, top_k, -1), x, w, idx)[1]
    xd, wd, gd = x.double(), w.double(), gy.double()
    for e in range(2):
        f = torch.where(idx == e, wt, 0.0).double()
        at = (idx == e).any(1)
        z = xd[at] @ wd[e].T
        O.within(slots[idx == e], z, z * promoted(inputs), F32, "apart")
        want = (f.sum(1)[:, None] * gd).T @ xd
        O.within(gw[e], want, want * (promoted(rows) + 2 * O.U), F32, "gw")
        want = gd[at].T @ xd[at]
        O.within(gws[e], want, want * promoted(rows), F32, "gw apart")
        if top_k == 1:
            O.within(y[at], f.sum(1)[at][:, None] * z, (f.sum(1)[at][:, None] * z) * (promoted(inputs) + O.U), F32, "y")
            want = (f.sum(1)[at][:, None] * gd[at]) @ wd[e]
            O.within(gx[at], want, want * (promoted(outputs) + O.U), F32, "gx")
            want = (z * gd[at]).sum(1)
            # <W^T g, x> over the inputs: a lane's share of the row, then the lanes
            O.within(gt[at, 0], want, want * (promoted(outputs) + (inputs / 128 + 12) * O.U), F32, "gt")


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows, inputs, outputs", [(20000, 40, 24), (9000, 136, 264)])
def test_16_bit_weight_gradient_of_one_sign(dtype, rows, inputs, outputs):
    """Accumulators of 512 rows (96 instructions for them where rows are two operands) in the weights' gradient too."""
    g = gen(rows + 1)
    idx = torch.randint(0, 2, (rows, 1), generator=g, device="cuda").int()
    x, gy = (rand(g, rows, inputs).abs() + 0.1).to(dtype), (rand(g, rows, outputs).abs() / 64 + 0.01).to(dtype)
    w, wt = rand(g, 2, outputs, inputs, dtype=dtype), torch.rand(rows, 1, generator=g, device="cuda") + 0.1
    for weights, grad in ((wt, gy), (None, gy[:, None])):
        _, gw, _ = E.expert_linear_backward(grad, x, w, idx, weights, input_gradient=False, routing_gradient=False)
        for e in range(2):
            f = torch.where(idx == e, 1.0 if weights is None else wt, 0.0).double()
            want = (f * gy.double()).T @ x.double()
            terms = (32 if weights is None else 96) * 2.0 ** -23 + (rows / 512 + 66) * O.U
            O.within(gw[e], want, want * (terms + (0 if weights is None else 2.0 ** -16 + 2.0 ** -15)), dtype, "gw")


@DT
@pytest.mark.parametrize("inputs, outputs", [(128, 64), (64, 128)])
def test_narrow_rows_of_one_sign(dtype, inputs, outputs):
    """The narrow rows' kernel: one accumulator for the whole row, the small products of 32-bit rows first."""
    g = gen(inputs)
    rows = 900
    idx = torch.rand(rows, 2, generator=g, device="cuda").topk(1, 1).indices.int()
    x, w = (rand(g, rows, inputs).abs() + 0.1).to(dtype), (rand(g, 2, outputs, inputs).abs() + 0.1).to(dtype)
    wt, gy = torch.rand(rows, 1, generator=g, device="cuda") + 0.1, (rand(g, rows, outputs).abs() + 0.1).to(dtype)
    y = E.expert_linear(x, w, idx, wt)
    gx, _, gt = E.expert_linear_backward(gy, x, w, idx, wt, weight_gradient=False)
    wi = w.double()[idx[:, 0].long()]
    z = torch.einsum("toi,ti->to", wi, x.double())
    f = wt.double()

    def bound(terms):  # large products: terms / 16 instructions; small ones before them: 2^-7 of the sum
        return (terms / 16 + 1 + 5 * terms / 16 * 2.0 ** -7 + 4) * 2.0 ** -23

    O.within(y, f * z, f * z * (bound(inputs) + 2 * O.U), dtype, "y")
    want = f * torch.einsum("toi,to->ti", wi, gy.double())
    O.within(gx, want, want * (bound(outputs) + 2 * O.U), dtype, "gx")
    want = (z * gy.double()).sum(1)
    O.within(gt[:, 0], want, want * (bound(outputs) + (inputs + 4) * O.U), F32, "gt")


# ---- offsets beyond 32 bits ----------------------------------------------------------------------

def test_norm_of_more_than_2_31_elements():
    g = gen(50)
    rows, dim = 523_300, 4104  # 2,147,623,200 elements
    x = torch.empty(rows, dim, device="cuda", dtype=BF16).normal_(generator=g)
    w = (1 + rand(g, dim, scale=0.1)).to(BF16)
    some = torch.tensor([0, 261_651, 523_264, rows - 2, rows - 1], device="cuda")
    y, h = E.add_rms_norm(x, w, x)
    want, s = O.norm(x[some], w, x[some])
    O.within(y[some], want, want.abs() * 130 * O.U, BF16, "y")
    O.within(h[some], s, s.abs() * O.U, BF16, "h")
    del y
    gx, gw = E.add_rms_norm_backward(x, h, w, x)
    (want, size), _ = O.norm_backward(x[some], h[some], w, x[some])
    O.within(gx[some], want, size * 520 * O.U, BF16, "gx")
    del gx, h
    q, scale = E.add_rms_norm_q8(x, w)
    y, _ = O.norm(x[some], w)
    got = q[some].double() * scale[some][:, None].double()
    assert ((got - y).abs() <= (2.0 ** -4 + 530 * O.U) * y.abs() + scale[some][:, None].double() * 2.0 ** -10 * 1.001).all()


@pytest.mark.parametrize("weighted", [False, True])
def test_linear_of_more_than_2_31_elements(weighted):
    """Wide outputs of many slots (the products, and without weights the outputs), then wide rows for each slot."""
    g = gen(51)
    rows, top_k, narrow, wide = 131_100, 2, 64, 8200  # 262,200 x 8200 = 2,150,040,000 elements
    idx = torch.rand(rows, 3, generator=g, device="cuda").topk(top_k, 1).indices.int()
    wt = torch.rand(rows, top_k, generator=g, device="cuda") + 0.1 if weighted else None
    some = torch.tensor([0, 65_000, 131_000, rows - 2, rows - 1], device="cuda")
    few = (idx[some], None if wt is None else wt[some])

    def check(x, w, slots):
        out = E.expert_linear(x, w, idx, wt, slots=slots)
        gx, _, gt = E.expert_linear_backward(out, x, w, idx, wt, slots=slots, weight_gradient=False)
        (ry, sy), (rx, sx), _, (rt, st) = O.linear(x[some], w, *few, slots, out[some])
        i, o = w.shape[2], w.shape[1]
        O.within(out[some], ry, sy * O.accumulate(i), BF16, "out")
        O.within(gx[some], rx, sx * O.accumulate(o), BF16, "gx")
        if weighted:
            O.within(gt[some], rt, st * (O.accumulate(o) + O.accumulate(i)), F32, "gt")

    x = torch.empty(rows, narrow, device="cuda", dtype=BF16).normal_(generator=g)
    check(x, rand(g, 3, wide, narrow, dtype=BF16, scale=0.125), False)
    x = torch.empty(rows, top_k, wide, device="cuda", dtype=BF16).normal_(generator=g)
    check(x, rand(g, 3, narrow, wide, dtype=BF16, scale=0.01), True)


@DT
def test_linear_names_an_expert_more_than_once_among_many_rows(dtype):
    g = gen(52)
    idx = torch.randint(-1, 3, (300, 3), generator=g, device="cuda").int()
    idx[7] = 2
    x, w = rand(g, 300, 72, dtype=dtype), rand(g, 3, 136, 72, dtype=dtype)
    wt, gy = torch.rand(300, 3, generator=g, device="cuda"), rand(g, 300, 136, dtype=dtype)
    (ry, sy), (rx, sx), (rw, sw), (rt, st) = O.linear(x, w, idx, wt, False, gy)
    O.within(E.expert_linear(x, w, idx, wt), ry, sy * O.accumulate(72), dtype, "out")
    gx, gw, gt = E.expert_linear_backward(gy, x, w, idx, wt)
    O.within(gx, rx, sx * O.accumulate(136), dtype, "gx")
    O.within(gw, rw, sw * (O.accumulate(900) + weight_gradient_bound(900)), dtype, "gw")
    O.within(gt, rt, st * (O.accumulate(72) + O.accumulate(136)), F32, "gt")


def test_route_of_scores_that_only_the_logits_tell_apart():
    """Sigmoids of 40 and 50 are both 1 in 64 bits: the logits decide without a bias, the index with one of zeros."""
    logits = torch.tensor([[40.0, 50.0, -3.0], [40.0, 40.0, 39.0]], device="cuda")
    assert E.route_experts(logits, 2, scores="sigmoid")[1].tolist() == [[1, 0], [0, 1]]
    zeros = torch.zeros(3, device="cuda")
    assert E.route_experts(logits, 2, scores="sigmoid", bias=zeros)[1].tolist() == [[0, 1], [0, 1]]


def test_a_models_hook_keeps_its_parameters_gradients_as_they_were():
    """The models differentiate in positions alone; the layer by itself in its parameters too."""
    from test_gpu_hooks import _args, _model

    m, c, cfg = _model("ictd")
    mix = E.RoutedChannelMix(int(cfg["channels"]), num_experts=4, top_k=2).cuda()
    pos = torch.tensor(c["pos"], device="cuda", dtype=torch.float32).requires_grad_()
    m(pos, *_args(c, torch.device("cuda")), sync_after_scatter=mix).sum().backward()
    assert pos.grad.abs().max() > 0 and all(p.grad is None for p in mix.parameters())
    mix(torch.randn(20, int(cfg["channels"]) * 9, device="cuda")).square().sum().backward()
    assert all(p.grad is not None for p in mix.parameters())


def test_weight_gradient_of_an_infinite_row_of_bf16():
    """The second part of an infinity is zero, not infinity less infinity."""
    g = gen(60)
    idx = torch.zeros(40, 1, device="cuda", dtype=torch.int32)
    x, gy, wt = rand(g, 40, 16, dtype=BF16), rand(g, 40, 8, dtype=BF16).abs() + 1, torch.rand(40, 1, generator=g, device="cuda") + 0.1
    x[3, 5] = float("inf")
    _, gw, _ = E.expert_linear_backward(gy, x, rand(g, 1, 8, 16, dtype=BF16), idx, wt, input_gradient=False)
    assert (gw[0, :, 5] == float("inf")).all()
    rest = torch.arange(16, device="cuda") != 5
    assert torch.isfinite(gw[0][:, rest]).all()


@pytest.mark.parametrize("experts", [512, 1024])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_of_many_experts_whose_small_scores_add_up(experts, groups):
    """Scores of less than half a last place each, which a sum in 32 bits loses one by one, decide a choice by bias."""
    n = experts // 32
    logits = torch.full((1, experts), -60.0, device="cuda")
    logits[0, 0] = 0.0
    logits[0, 32::32] = -16.65  # n - 1 times 5.9e-8: the first expert's score is 1 - (n - 1) 5.9e-8
    lost = (n - 1) * 5.87e-8
    for share in (0.55, 0.7, 0.8, 0.9, 1.1, 1.3):
        bias = torch.zeros(experts, device="cuda")
        bias[experts // 2 + 1] = 1.0 - share * lost  # another's score: just above or just below it
        kw = dict(bias=bias, num_groups=groups, groups_kept=max(1, groups // 2))
        want = O.route(logits, 1, **kw)[1]
        assert want.item() == (0 if share > 1 else experts // 2 + 1)
        assert torch.equal(E.route_experts(logits, 1, **kw)[1].cpu(), want)
