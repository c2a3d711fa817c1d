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
