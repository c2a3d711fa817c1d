"""Routed-expert operators at the edges of what their documentation allows, against the 64-bit statements."""

import pytest
import torch

import experts_oracle as O
import gpu_util as U
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
