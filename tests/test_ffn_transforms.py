"""The feed-forward operators under torch's other ways of calling them: forward-mode derivatives."""

import pytest
import torch
from torch.autograd import forward_ad

import cernels_b200
from tests import ffn_reference as R
from tests import w4_reference as Q

gpu = pytest.mark.gpu


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def calls(device):
    """(name, function of its floating inputs, those inputs) for each operator."""
    *ffn, _ = R.case(3, 64, 32, device=device)
    q1, s1 = Q.codes((4, 64, 64), 32, 1, device)
    q2, s2 = Q.codes((4, 64, 32), 32, 2, device)
    x, idx, w = ffn[0], torch.zeros(3, 2, dtype=torch.int32, device=device), torch.rand(3, 2, device=device)
    return [("gated_ffn", cernels_b200.gated_ffn, ffn),
            ("linear_w4", lambda x, s: cernels_b200.linear_w4(x, q1[0], s), [x, s1[0]]),
            ("moe", lambda x, s1, s2, w: cernels_b200.moe_experts_decode_w4(x, q1, s1, q2, s2, idx, w, 2), [x, s1, s2, w])]


def refuses_duals(device):
    for name, f, args in calls(device):
        for i in range(len(args)):
            with forward_ad.dual_level(), torch.no_grad():
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    f(*(dual(a) if j == i else a for j, a in enumerate(args)))


def test_tangents_are_refused():
    refuses_duals("cpu")


@gpu
def test_tangents_are_refused_on_cuda():
    refuses_duals("cuda")
    ops = torch.ops.cernels_b200
    (_, _, ffn), (_, _, (x, s)), _ = calls("cuda")
    q = Q.codes((4, 64, 64), 32, 1)[0][0]
    with forward_ad.dual_level(), torch.no_grad():
        for f, args in ((ops.gated_ffn, ffn), (lambda x, s: ops.linear_w4(x, q, s), [x, s])):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                f(dual(args[0]), *args[1:])
        for _, f, args in calls("cuda"):  # other tensors' tangents are nobody's business
            assert torch.isfinite(f(*args)).all()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda v: cernels_b200.gated_ffn(v, *ffn[1:]), (ffn[0],), (ffn[0],))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: cernels_b200.gated_ffn(v, *ffn[1:]).float().sum())(ffn[0])
