"""The feed-forward operators under torch's other ways of calling them: forward-mode derivatives, fake
tensors and traces (torch.compile, torch.export, make_fx), function transforms."""

import contextlib
import ctypes
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import cernels_b200
from cernels_b200 import _lib, ffn
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


# ---------------------------------------------------------------- fake tensors (CPU)
def fakes():
    def t(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    u8, f32, i32 = torch.uint8, torch.float32, torch.int32
    block = [t(5, 64), t(32, 64), t(32, 64), t(64, 32)]
    linear = [t(3, 64), t(10, 32, dtype=u8), t(10, 2)]
    experts = [t(3, 64), t(4, 64, 32, dtype=u8), t(4, 64, 2), t(4, 64, 16, dtype=u8), t(4, 64, 1), t(3, 2, dtype=i32),
               t(3, 2, dtype=f32), 2]
    return [("gated_ffn", block, (5, 64)), ("linear_w4", linear, (3, 10)), ("moe_experts_decode_w4", experts, (3, 64))]


MODES = {"grad": contextlib.nullcontext, "no_grad": torch.no_grad, "inference": torch.inference_mode}


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("where", [cernels_b200, torch.ops.cernels_b200], ids=["function", "op"])
def test_fake_tensors_take_the_meta_form(where, mode):
    with warnings.catch_warnings(), FakeTensorMode(), MODES[mode]():
        warnings.simplefilter("error")  # reading a fake tensor's address warns
        for name, args, shape in fakes():
            y = getattr(where, name)(*args)
            assert y.shape == shape and y.dtype == torch.bfloat16 and y.device.type == "cuda"


@pytest.mark.parametrize("need", [(1, 1, 1, 1), (1, 0, 0, 0), (0, 1, 0, 1), (0, 0, 0, 1)])
def test_fake_tensors_differentiate(need):
    with warnings.catch_warnings(), FakeTensorMode():
        warnings.simplefilter("error")
        args = [a.requires_grad_(bool(n)) for a, n in zip(fakes()[0][1], need)]
        for f in (cernels_b200.gated_ffn, torch.ops.cernels_b200.gated_ffn):
            y = f(*args)
            assert y.requires_grad
            with torch.no_grad():
                got = y.grad_fn.apply(torch.empty_like(y))  # the node itself: the engine wants a device
            assert [None if g is None else g.shape for g in got] == [a.shape if n else None for a, n in zip(args, need)]


def test_four_bit_products_of_fakes_refuse_gradients():
    with FakeTensorMode():
        for name, args, _ in fakes()[1:]:
            args[0].requires_grad_()
            for where in (cernels_b200, torch.ops.cernels_b200):
                with pytest.raises(RuntimeError, match="no gradient"):
                    getattr(where, name)(*args)


def test_traces_record_the_operators():
    with FakeTensorMode(), torch.no_grad():
        for name, args, _ in fakes():
            tensors = [a for a in args if isinstance(a, torch.Tensor)]
            rest = args[len(tensors):]
            for where in (cernels_b200, torch.ops.cernels_b200):
                graph = make_fx(lambda *t: getattr(where, name)(*t, *rest))(*tensors).graph
                targets = [n.target for n in graph.nodes if n.op == "call_function"]
                assert targets == [getattr(torch.ops.cernels_b200, name).default]


@pytest.mark.parametrize("T,F", [(0, 8), (1, 8), (32, 40), (33, 8), (700, 264)])
def test_meta_sizes_of_what_a_training_step_keeps(T, F):
    s, n = _lib.FfnShape(T, 64, F), ctypes.c_size_t(0)
    assert _lib.load().cernels_gated_ffn_saved_bytes(ctypes.byref(s), ctypes.byref(n)) == 0
    x, w, wd = (torch.empty(a, b, dtype=torch.bfloat16, device="meta") for a, b in ((T, 64), (F, 64), (64, F)))
    out, act, saved = torch.ops.cernels_b200.gated_ffn_train(x, w, w, wd)
    assert out.shape == (T, 64) and act.shape == (T, F) and saved.numel() * 4 == n.value


# ---------------------------------------------------------------- compiled (GPU)
@gpu
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_training_step_is_the_eager_one(dynamic):
    def step(x, wg, wu, wd):
        return (cernels_b200.gated_ffn(x * 2, wg, wu, wd) + torch.ops.cernels_b200.gated_ffn(x, wg, wu, wd)).float().square().mean()

    compiled = torch.compile(step, backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for T in (5, 40, 200):
        results = []
        for f in (step, compiled):
            t = [a.requires_grad_() for a in R.case(T, 64, 48, seed=T)[:4]]
            y = f(*t)
            results.append((y.detach(), *torch.autograd.grad(y, t)))
        assert all(torch.equal(a, b) for a, b in zip(*results))
    assert ffn.status() == 0


@gpu
def test_compiled_inference_is_the_eager_one():
    compiled = [torch.compile(f, backend="aot_eager", fullgraph=True) for _, f, _ in calls("cuda")]
    with torch.no_grad():
        for (_, f, args), c in zip(calls("cuda"), compiled):
            assert torch.equal(f(*args), c(*args))


@gpu
def test_traces_with_real_tensors_and_modes_see_the_operators():
    _, f, args = calls("cuda")[0]
    with torch.no_grad():
        traced = make_fx(f, tracing_mode="real")(*args)
        assert torch.ops.cernels_b200.gated_ffn.default in [n.target for n in traced.graph.nodes]
        assert torch.equal(traced(*args), f(*args))
    t = [a.clone().requires_grad_() for a in args]
    seen = []

    class Mode(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func)
            return func(*args, **(kwargs or {}))

    dy = torch.randn_like(t[0])
    want = torch.autograd.grad(f(*t), t, dy)
    with Mode():
        got = torch.autograd.grad(f(*t), t, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    o = torch.ops.cernels_b200
    assert o.gated_ffn_train.default in seen and o.gated_ffn_backward.default in seen


@gpu
@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_jit_traces_record_the_operators():
    """A trace made from one set of inputs computes with those of later calls."""
    with torch.no_grad():
        for name, f, args in calls("cuda"):
            traced = torch.jit.trace(f, [a.clone() for a in args], check_trace=False)
            other = [a * 0.5 for a in args]
            assert torch.equal(traced(*other), f(*other)) and not torch.equal(f(*other), f(*args))


@gpu
def test_plain_subclasses_of_tensors_are_taken():
    class Named(torch.Tensor):
        pass

    for name, f, args in calls("cuda"):
        with torch.no_grad():
            y = f(*(a.as_subclass(Named) for a in args))
            assert isinstance(y, Named) and torch.equal(y.as_subclass(torch.Tensor), f(*args))
    f, args = calls("cuda")[0][1:]
    t, n = ([a.clone().requires_grad_() for a in args] for _ in range(2))
    dy = torch.randn_like(args[0])
    got = torch.autograd.grad(f(*(a.as_subclass(Named) for a in n)), n, dy.as_subclass(Named))
    for g, w in zip(got, torch.autograd.grad(f(*t), t, dy)):
        assert torch.equal(g.as_subclass(torch.Tensor), w)


@gpu
def test_exported_programs_hold_the_operators():
    class Call(torch.nn.Module):
        def __init__(self, f):
            super().__init__()
            self.f = f

        def forward(self, *args):
            return self.f(*args)

    for name, f, args in calls("cuda"):
        with torch.no_grad():
            program = torch.export.export(Call(f), tuple(args)).module()
            other = [a * 0.5 for a in args]
            assert torch.equal(program(*other), f(*other))
