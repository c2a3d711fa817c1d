"""Routed-expert operators without a GPU: argument checks at the C ABI and of the Python functions."""


import pytest
import torch

from fsctep_b200 import _native as N
from fsctep_b200 import experts as E

FAKE = 4096  # a pointer that no call below gets to follow


def _refused(status, text):
    assert status == 1, status
    assert text in N.lib().fsc_last_error().decode()


def _norm(dtype=0, wdtype=0, x=FAKE, w=FAKE, y=FAKE, q=None, scale=None, rows=1, dim=8):
    return N.lib().fsc_rms_norm_forward(dtype, wdtype, x, dim, None, 0, w, 1e-6, y, None, q, scale, rows, dim, None)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=1), "dtype"), (dict(dtype=4), "dtype"), (dict(dtype=2, wdtype=3), "weight"), (dict(rows=-1), "rows"),
    (dict(dim=0), "dim"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "y or q"),
    (dict(q=FAKE), "y or q"), (dict(y=None, q=FAKE), "together"), (dict(scale=FAKE), "together"),
])
def test_norm_refusals(kw, text):
    _refused(_norm(**kw), text)


def test_norm_of_no_rows_needs_no_device():
    assert _norm(rows=0, x=None, w=None) == 0


def test_norm_backward_refusals():
    lib = N.lib()

    def call(gy=FAKE, h=FAKE, ws=FAKE, nbytes=1 << 30, dim=8):
        return lib.fsc_rms_norm_backward(0, 0, gy, dim, None, 0, h, dim, FAKE, 1e-6, FAKE, FAKE, 3, dim, ws, nbytes, None)

    _refused(call(gy=None), "null")
    _refused(call(h=None), "null")
    _refused(call(ws=None), "workspace")
    _refused(call(nbytes=3 * 8 * 4 - 1), "workspace")
    assert lib.fsc_rms_norm_backward_workspace_bytes(3, 8) == 3 * 8 * 4
    assert lib.fsc_rms_norm_backward_workspace_bytes(0, 8) == 0


def _route(dtype=0, logits=FAKE, tokens=1, experts=8, top_k=2, groups=1, kept=1, scores=0):
    return N.lib().fsc_route_experts(dtype, logits, experts, None, None, FAKE, FAKE, tokens, experts, top_k, groups,
                                     kept, scores, 1, 1.0, None)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=1), "dtype"), (dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(top_k=0), "top_k"),
    (dict(top_k=9), "top_k"), (dict(experts=64, top_k=33), "top_k"), (dict(groups=3), "groups"),
    (dict(groups=0), "groups"), (dict(groups=4, kept=5), "groups_kept"), (dict(groups=4, kept=0), "groups_kept"),
    (dict(groups=4, kept=1, top_k=3), "kept groups"), (dict(scores=2), "scores"), (dict(logits=None), "null"),
    (dict(tokens=-1), "tokens"),
])
def test_route_refusals(kw, text):
    _refused(_route(**kw), text)


def test_plan_refusals_and_sizes():
    lib = N.lib()

    def call(indices=FAKE, tokens=10, per_token=2, experts=8, offsets=FAKE, joint=None, nbytes=0):
        return lib.fsc_expert_plan(indices, tokens, per_token, experts, offsets, FAKE, joint, FAKE, FAKE, None, nbytes, None)

    _refused(call(experts=0), "experts")
    _refused(call(experts=1025), "experts")
    _refused(call(tokens=-1), "slots")
    _refused(call(per_token=33), "slots")
    _refused(call(tokens=1 << 30, per_token=4), "slots")
    _refused(call(indices=None), "null")
    _refused(call(offsets=None), "null")
    _refused(call(joint=FAKE), "joint")
    _refused(call(tokens=100000), "workspace")
    assert lib.fsc_expert_plan_workspace_bytes(2048, 2, 8) == 0
    assert lib.fsc_expert_plan_workspace_bytes(100000, 2, 8) >= 200000 // 4096 * 8 * 4
    assert lib.fsc_expert_joint_bins(100000, 2, 8) == 81 and lib.fsc_expert_joint_bins(100000, 4, 8) == 0
    assert lib.fsc_expert_joint_bins(1000, 2, 8) == 0 and lib.fsc_expert_joint_bins(100000, 1, 1024) == 0


def _linear(dtype=0, x=FAKE, tokens=4, per_token=2, comps=1, experts=8, inputs=16, outputs=16, nbytes=1 << 30):
    return N.lib().fsc_expert_linear(dtype, x, FAKE, FAKE, FAKE, FAKE, FAKE, None, None, FAKE, FAKE, tokens, per_token, comps,
                                     experts, inputs, outputs, 0, FAKE, nbytes, None)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=1), "dtype"), (dict(dtype=4), "dtype"), (dict(x=None), "null"), (dict(per_token=0), "slots"),
    (dict(per_token=33), "slots"), (dict(comps=0), "components"), (dict(comps=2000), "components"),
    (dict(experts=0), "experts"), (dict(inputs=0), "inputs"), (dict(outputs=0), "outputs"),
    (dict(tokens=1 << 30), "rows"), (dict(tokens=1 << 40), "slots"), (dict(tokens=100, nbytes=8), "workspace"),
])
def test_linear_refusals(kw, text):
    _refused(_linear(**kw), text)


def test_q8_and_backward_refusals():
    lib = N.lib()
    args = [FAKE] * 10
    _refused(lib.fsc_expert_linear_q8(4, *args, 4, 2, 1, 8, 16, 16, 0, FAKE, 1 << 30, None), "out_dtype")
    _refused(lib.fsc_expert_linear_q8(2, *args, 4, 2, 3, 8, 16, 16, 0, FAKE, 1 << 30, None), "component")
    _refused(lib.fsc_expert_linear_q8(2, *args, 100, 2, 1, 8, 16, 16, 0, FAKE, 8, None), "workspace")
    back = [FAKE, FAKE, FAKE, FAKE, None, FAKE, FAKE, None, None, FAKE, FAKE, FAKE, FAKE]  # no weights, but their gradient asked for
    _refused(lib.fsc_expert_linear_backward(0, *back, 4, 2, 1, 8, 16, 16, 0, FAKE, 1 << 30, None), "grad_weights")
    back[4] = FAKE
    _refused(lib.fsc_expert_linear_backward(0, *back, 100, 2, 1, 8, 16, 16, 0, FAKE, 8, None), "workspace")


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=1), "dtype"), (dict(out_dtype=2), "out_dtype"), (dict(tokens=17), "32 slots"), (dict(comps=17), "16 components"),
    (dict(inputs=20000), "12288"), (dict(x=None), "null"), (dict(experts=0), "experts"), (dict(w=FAKE + 2), "16 bytes"),
    (dict(dtype=4, comps=2), "one component"), (dict(dtype=4, out_dtype=4), "out_dtype"), (dict(dtype=4, xs=None), "null"),
])
def test_few_refusals(kw, text):
    a = dict(dtype=0, out_dtype=0, x=FAKE, xs=FAKE, w=FAKE, tokens=4, per_token=2, comps=1, experts=8, inputs=16, outputs=16)
    a.update(kw)
    _refused(N.lib().fsc_expert_linear_few(a["dtype"], a["out_dtype"], a["x"], a["xs"], a["w"], FAKE, FAKE, FAKE, FAKE,
                                           a["tokens"], a["per_token"], a["comps"], a["experts"], a["inputs"],
                                           a["outputs"], 0, None), text)


def test_few_rows_rule_is_the_librarys():
    for t in (0, 1, 3, 16, 32, 33):
        for k in (1, 2, 8, 32):
            for c in (0, 1, 9, 16, 17):
                for i in (1, 64, 1024, 12288, 12289):
                    for slots in (False, True):
                        fits = bool(N.lib().fsc_expert_few_fits(t, k, max(c, 1), i, slots))
                        assert E._few(t, k, (c,) if c else (), i, slots) == fits, (t, k, c, i, slots)


def test_workspace_queries():
    lib = N.lib()
    assert lib.fsc_expert_linear_workspace_bytes(2, 0, 2, 9, 8, 64, 64, 0, 1, 0) == 0
    assert lib.fsc_expert_linear_workspace_bytes(0, 1 << 40, 2, 9, 8, 64, 64, 0, 1, 0) == 0  # refused sizes
    assert lib.fsc_expert_linear_backward_workspace_bytes(0, 4, 2, 1, 8, 16, 16, 0, 1, 1, 1, 0) >= 4 * 2 * 16 * 4
    # narrow rows with a joint grouping need no rows in between: fp32 matrices in three planes are all
    assert lib.fsc_expert_linear_workspace_bytes(0, 50000, 2, 9, 8, 64, 64, 0, 1, 1) == 3 * 8 * 64 * 64 * 2
    assert lib.fsc_expert_linear_workspace_bytes(2, 50000, 2, 9, 8, 64, 64, 0, 1, 1) == 0


def test_python_functions_refuse_cpu_tensors():
    x, w = torch.zeros(3, 8), torch.ones(8)
    i = torch.zeros(3, 2, dtype=torch.int32)
    for call in (lambda: E.add_rms_norm(x, w), lambda: E.add_rms_norm_q8(x, w),
                 lambda: E.add_rms_norm_backward(x, x, w), lambda: E.route_experts(x, 2),
                 lambda: E.route_experts_backward(torch.zeros(3, 2), x, i), lambda: E.expert_plan(i, 4),
                 lambda: E.expert_linear(x, torch.zeros(4, 5, 8), i),
                 lambda: E.expert_linear_backward(torch.zeros(3, 2, 5), x, torch.zeros(4, 5, 8), i)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_quantize_experts_scales_each_output():
    w = torch.randn(3, 5, 7)
    w[1, 2] = 0
    q, s = E.quantize_experts(w)
    assert q.dtype == torch.float8_e4m3fn and q.shape == w.shape and s.shape == (3, 5)
    assert s[1, 2] == 0 and (q[1, 2].float() == 0).all()
    err = (q.float() * s[..., None] - w).abs()
    assert (err <= 2.0 ** -4 * w.abs() + s[..., None] * 2.0 ** -10 + 1e-9).all()


def test_channel_mix_layout_round_trip_and_degrees():
    m = E.RoutedChannelMix(4, 3, 2, degrees=(0, 1, 1, 2), layers=2)
    f = torch.randn(5, 4 * 12)
    rows = m._to_rows(f)
    assert rows.shape == (5, 12, 4) and torch.equal(m._from_rows(rows), f)
    assert torch.equal(rows[:, 1:4], f[:, 4:16].reshape(5, 4, 3).transpose(1, 2))
    assert m.block.tolist() == [0, 1, 1, 1, 2, 2, 2, 3, 3, 3, 3, 3]
    with pytest.raises(RuntimeError, match="invariant"):
        E.RoutedChannelMix(4, degrees=(1, 2))
    with pytest.raises(RuntimeError, match="shape"):
        m(torch.randn(5, 7))


def test_forward_mode_tangents_are_refused():
    """The kernels see values alone: a tangent would come out as zero without a word."""
    from torch.autograd import forward_ad

    x, plain = torch.ones(3, 4), torch.ones(3, 4)
    with forward_ad.dual_level():
        assert not E._differentiable(x, None)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        i = torch.zeros(3, 4, dtype=torch.int32)
        for call in (lambda: E._differentiable(plain, None, dual), lambda: E.add_rms_norm_backward(dual, plain, plain[0]),
                     lambda: E.route_experts_backward(plain, dual, i),
                     lambda: E.expert_linear_backward(plain, dual, torch.ones(2, 3, 4), i)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
    assert not E._differentiable(x)


def test_a_plan_reports_a_wait_that_ran_out():
    plan = object.__new__(E.ExpertPlan)
    plan.num_experts, plan._data = 2, torch.zeros(9, dtype=torch.int32)
    plan.check()
    plan._data[3] = 13  # after the three offsets
    with pytest.raises(N.NativeError, match="wait ran out.*13"):
        plan.check()


def test_channel_mix_layout_of_no_atoms():
    m = E.RoutedChannelMix(4, 3, 2, degrees=(0, 1))
    f = torch.empty(0, 16)
    rows = m._to_rows(f)
    assert rows.shape == (0, 4, 4) and m._from_rows(rows).shape == (0, 16)


@pytest.mark.parametrize("kw", [dict(layers=0), dict(top_k=0), dict(num_experts=4, top_k=5), dict(num_experts=0, top_k=1),
                                dict(num_experts=40, top_k=33), dict(num_experts=1025), dict(scores="relu")])
def test_channel_mix_refuses_what_its_calls_would(kw):
    with pytest.raises(RuntimeError):
        E.RoutedChannelMix(8, **kw)


def test_quantize_experts_of_the_smallest_floats():
    """A scale below the normal floats is coarse: the largest weight over it may exceed what e4m3 holds."""
    w = torch.tensor([[[9e-43, -9e-43, 3e-43], [2e-42, 1e-42, 0.0], [1e-44, 1e-45, 0.0], [3e38, -3e38, 1e38]]])
    q, s = E.quantize_experts(w)
    assert torch.isfinite(q.float()).all()
    # half a step of e4m3, and of the scale's last place (2^-149) up to 448 times
    err = (q.double() * s[..., None].double() - w.double()).abs()
    assert (err <= 2.0 ** -4 * w.double().abs() + s[..., None].double() * 2.0 ** -10 + 448 * 2.0 ** -150).all()
