"""The feed-forward operators as modules and models use them: loaders, in-model swaps, and a run
of training and decoding that takes all of them."""

import types

import pytest
import torch

import cernels_b200
from cernels_b200 import ffn, ops, swaps
from cernels_b200.registry import gated_ffn, moe_experts_w4
from tests import ffn_reference as R
from tests import w4_reference as Q

gpu = pytest.mark.gpu


class DeepseekV2MLP(torch.nn.Module):  # name- and layout-matched stand-ins for the transformers classes
    def __init__(self, hidden=64, inter=96, bias=False, act=None, device=None):
        super().__init__()
        kw = dict(bias=bias, dtype=torch.bfloat16, device=device)
        self.gate_proj = torch.nn.Linear(hidden, inter, **kw)
        self.up_proj = torch.nn.Linear(hidden, inter, **kw)
        self.down_proj = torch.nn.Linear(inter, hidden, **kw)
        self.act_fn = act or torch.nn.SiLU()

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x))


class DeepseekV2Experts(torch.nn.Module):
    def __init__(self, experts=4, hidden=64, inter=32, device=None):
        super().__init__()
        self.gate_up_proj = torch.nn.Parameter(torch.randn(experts, 2 * inter, hidden, device=device).bfloat16() * 0.1)
        self.down_proj = torch.nn.Parameter(torch.randn(experts, hidden, inter, device=device).bfloat16() * 0.1)

    def forward(self, h, idx, w):
        return "stock"


# ---------------------------------------------------------------- CPU
def test_loader_refuses_other_mlps():
    gated_ffn.check_module(DeepseekV2MLP())
    gated_ffn.check_module(DeepseekV2MLP(act=torch.nn.functional.silu))
    with pytest.raises(RuntimeError, match="bias"):
        gated_ffn.check_module(DeepseekV2MLP(bias=True))
    with pytest.raises(RuntimeError, match="silu"):
        gated_ffn.check_module(DeepseekV2MLP(act=torch.nn.GELU()))
    with pytest.raises(RuntimeError, match="not available"):
        gated_ffn.kernel(torch.zeros(1, 64), None)


def test_mlp_swap_sets_and_restores():
    m = torch.nn.ModuleList([DeepseekV2MLP(), torch.nn.Linear(2, 2), DeepseekV2MLP()])
    apply, variants = swaps.SWAPS["deepseek_v2_mlp"]
    assert variants == ("stock", "custom")
    assert apply(m, "custom") == 2 and "forward" in vars(m[0])
    with pytest.raises(RuntimeError, match="CUDA tensor"):  # the operator, and no CPU fallback
        m[0](torch.zeros(1, 64, dtype=torch.bfloat16))
    assert apply(m, "stock") == 2 and "forward" not in vars(m[0])
    assert m[0](torch.zeros(1, 64, dtype=torch.bfloat16)).shape == (1, 64)
    with pytest.raises(RuntimeError, match="no Qwen3NextMLP"):
        swaps.SWAPS["qwen3_next_mlp"][0](m, "custom")


def test_a_refused_swap_changes_nothing():
    m = torch.nn.ModuleList([DeepseekV2MLP(), DeepseekV2MLP(bias=True)])
    with pytest.raises(RuntimeError, match="bias"):
        swaps.SWAPS["deepseek_v2_mlp"][0](m, "custom")
    assert not any("forward" in vars(mod) for mod in m)
    m = torch.nn.ModuleList([DeepseekV2Experts(), DeepseekV2Experts(hidden=48)])
    with pytest.raises(RuntimeError, match="multiples"):
        swaps.SWAPS["deepseek_v2"][0](m, "custom_w4")
    assert not any(hasattr(mod, "_cernels_w4") or "forward" in vars(mod) for mod in m)


def test_w4_copies_are_prepared_and_released():
    e = DeepseekV2Experts()
    with pytest.raises(RuntimeError, match="prepare"):
        moe_experts_w4.decode_kernel(torch.zeros(1, 64), torch.zeros(1, 2), torch.zeros(1, 2), e)
    m = torch.nn.ModuleList([e])
    assert swaps.SWAPS["deepseek_v2"][0](m, "custom_w4") == 1
    q1, s1, q2, s2 = e._cernels_w4
    assert q1.shape == (4, 64, 32) and s1.shape == (4, 64, 2) and q2.shape == (4, 64, 16) and s2.shape == (4, 64, 1)
    for q, s, w in ((q1, s1, e.gate_up_proj), (q2, s2, e.down_proj)):
        step = s.double().repeat_interleave(32, -1)
        assert ((Q.values(q, s) - w.detach().double()).abs() <= step * (0.5 + 7 * R.HALF)).all()
    swaps.SWAPS["deepseek_v2"][0](m, "stock")
    assert not hasattr(e, "_cernels_w4") and e(torch.zeros(1, 64), None, None) == "stock"
    with pytest.raises(RuntimeError, match="not available"):
        moe_experts_w4.prepare(None)


def test_w4_group_choice():
    assert [moe_experts_w4.group_of(*s) for s in ((2048, 1408), (2048, 832), (2880, 2880), (64, 96))] == [128, 64, 64, 32]
    with pytest.raises(RuntimeError, match="multiples"):
        moe_experts_w4.group_of(48, 64)


# ---------------------------------------------------------------- GPU
@gpu
@pytest.mark.parametrize("shape", [(1, 1), (2, 5), (3, 40)])
def test_swapped_mlp_trains(shape):
    torch.manual_seed(0)
    mlp = DeepseekV2MLP(device="cuda")
    model = torch.nn.Sequential(mlp)
    swaps.SWAPS["deepseek_v2_mlp"][0](model, "custom")
    x = torch.randn(*shape, 64, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(*shape, 64, device="cuda").bfloat16()
    y = model(x)
    y.backward(dy)
    w = [p.detach() for p in (mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight)]
    want, bound, state = R.forward(x.reshape(-1, 64), *w)
    assert y.shape == x.shape
    R.assert_within("y", y.detach().reshape(-1, 64), want, bound)
    got = (x.grad.reshape(-1, 64), mlp.gate_proj.weight.grad, mlp.up_proj.weight.grad, mlp.down_proj.weight.grad)
    for g, (v, b) in zip(got, R.backward(state, dy.reshape(-1, 64))):
        R.assert_within("gradient", g, v, b)
    with torch.no_grad():  # a transposed batch: rows that cannot be read where they lie
        t = x.detach().transpose(0, 1)
        R.assert_within("y", model(t).transpose(0, 1).reshape(-1, 64), want, bound)


@gpu
def test_swapped_experts_decode_in_4_bits():
    torch.manual_seed(1)
    e = DeepseekV2Experts(device="cuda")
    m = torch.nn.ModuleList([e])
    swaps.SWAPS["deepseek_v2"][0](m, "custom_w4")
    x = torch.randn(3, 64, device="cuda").bfloat16()
    w, idx = torch.rand(3, 4, device="cuda").topk(2, -1)
    want, bound = Q.experts(x, *e._cernels_w4, idx, w)
    R.assert_within("y", e(x, idx, w), want, bound)
    x5, w5, i5 = (torch.cat((v, v[:2])) for v in (x, w, idx))  # five tokens: the bf16 prefill entry
    full = cernels_b200.cohere2_moe_experts(x5, e.gate_up_proj.data, e.down_proj.data, i5.int(), w5, 2)
    assert torch.equal(e(x5, i5, w5), full)


@gpu
@pytest.mark.parametrize("T", [1, 20, 130])
def test_calls_see_what_the_kernels_right_before_them_wrote(T):
    """Inputs, weights, codes and expert ids written by kernels queued just before the call (which may start
    under them): the results are those of a call made after everything has ended."""
    H, F, E = 1024, 2048, 8
    sets = []
    for seed in (1, 2):
        x, wg, wu, wd, _ = R.case(T, H, F, seed=seed, std=0.03)
        t = min(T, 20)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        idx = torch.randint(0, E, (t, 2), generator=gen, device="cuda").int()
        sets.append([x, wg, wu, wd, *Q.codes((E, 2 * F, H), 64, seed), *Q.codes((E, H, F), 64, seed), idx,
                     torch.rand(t, 2, generator=gen, device="cuda")])

    def calls(v):
        x, wg, wu, wd, q1, s1, q2, s2, idx, w = v
        t = idx.shape[0]
        return (cernels_b200.gated_ffn(x, wg, wu, wd), cernels_b200.linear_w4(x, q1[0], s1[0]),
                cernels_b200.moe_experts_decode_w4(x[:t], q1, s1, q2, s2, idx, w, 2))

    want = []
    for v in sets:
        torch.cuda.synchronize()
        want.append([])
        for i in range(3):
            want[-1].append(calls(v)[i])
            torch.cuda.synchronize()
    live = [v.clone() for v in sets[0]]
    for i in range(12):
        for a, b in zip(live, sets[i % 2]):
            a.copy_(b)
        for a, b in zip(calls(live), want[i % 2]):
            assert torch.equal(a, b)
        x, wg, wu, wd = (v.detach().requires_grad_() for v in live[:4])  # and a training step after them
        torch.autograd.grad(cernels_b200.gated_ffn(x, wg, wu, wd).sum(), (x, wg, wu, wd))


@gpu
def test_train_the_dense_block_then_decode_everything_in_a_graph():
    """A layer of a routed model in small: its shared block is trained for a few steps; then tokens are
    decoded from one graph: router, 4-bit experts, the shared block, a 4-bit output projection. The
    graph's results are those of the calls made one by one, for several tokens, and each operator's
    result is within its bound for the inputs that it got."""
    H, F, E, V, k = 128, 64, 8, 200, 2
    gen = torch.Generator(device="cuda").manual_seed(2)

    def rnd(*shape, scale=0.1):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(torch.bfloat16)

    shared = [torch.nn.Parameter(rnd(F, H)), torch.nn.Parameter(rnd(F, H)), torch.nn.Parameter(rnd(H, F))]
    opt = torch.optim.SGD(shared, lr=0.05)
    before = [p.detach().clone() for p in shared]
    for _ in range(3):
        data, target = rnd(50, H, scale=1.0), rnd(50, H, scale=1.0)
        opt.zero_grad()
        ((cernels_b200.gated_ffn(data, *shared).float() - target.float()) ** 2).mean().backward()
        opt.step()
    assert all(torch.isfinite(p).all() for p in shared) and any(not torch.equal(p, b) for p, b in zip(shared, before))

    experts = types.SimpleNamespace(gate_up_proj=torch.nn.Parameter(rnd(E, 2 * F, H)),
                                    down_proj=torch.nn.Parameter(rnd(E, H, F)))
    copies = moe_experts_w4.prepare(experts)
    router = rnd(E, H, scale=1.0)
    head = cernels_b200.quantize_w4(rnd(V, H), 64)

    def layer(x):
        idx, w = ops.router(x, router, None, E, k, ops.ROUTER_SOFTMAX_TOPK)
        routed = cernels_b200.moe_experts_decode_w4(x, *copies, idx, w, k)
        dense = cernels_b200.gated_ffn(x, *shared)
        mixed = routed + dense
        return idx, w, routed, dense, mixed, cernels_b200.linear_w4(mixed, *head)

    with torch.no_grad():
        x = rnd(2, H, scale=1.0)
        layer(x)  # first calls, outside the capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x)
        for _ in range(3):
            x.copy_(rnd(2, H, scale=1.0))
            graph.replay()
            for a, b in zip(out, layer(x)):
                assert torch.equal(a, b)
            idx, w, routed, dense, mixed, logits = out
            R.assert_within("experts", routed, *Q.experts(x, *copies, idx, w))
            R.assert_within("dense", dense, *R.forward(x, *shared)[:2])
            R.assert_within("logits", logits, *Q.linear(mixed, *head))
    assert ffn.status() == 0
