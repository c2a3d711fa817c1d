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
