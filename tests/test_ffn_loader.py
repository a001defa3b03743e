"""Which modules the gated block's loader and swap take: those that compute what the operator computes."""

import copy

import pytest
import torch

from cernels_b200 import swaps, w4
from cernels_b200.registry import gated_ffn, moe_experts_w4
from tests import ffn_reference as R
from tests.test_ffn_modules import DeepseekV2Experts, DeepseekV2MLP


class Adapter(torch.nn.Module):  # a low-rank adapter that shows its base layer's weight and bias
    def __init__(self, base):
        super().__init__()
        self.base = base
        self.a = torch.nn.Parameter(torch.randn(4, base.in_features))
        self.b = torch.nn.Parameter(torch.randn(base.out_features, 4))

    weight = property(lambda self: self.base.weight)
    bias = property(lambda self: self.base.bias)

    def forward(self, x):
        return self.base(x) + x @ self.a.T @ self.b.T


class Wider(torch.nn.Linear):
    def forward(self, x):
        return 2.0 * super().forward(x)


def wrap(mlp, name):
    setattr(mlp, name, Adapter(getattr(mlp, name)))


def subclass(mlp, name):
    setattr(mlp, name, Wider(64, 96, bias=False))


def parametrised(mlp, name):
    torch.nn.utils.parametrize.register_parametrization(getattr(mlp, name), "weight", torch.nn.Identity())


def weight_norm(mlp, name):  # recomputes the weight in a hook before each call
    proj = getattr(mlp, name)
    proj.weight.data = proj.weight.data.float()
    torch.nn.utils.weight_norm(proj)


def forward_hook(mlp, name):
    getattr(mlp, name).register_forward_hook(lambda mod, args, out: 2 * out)


def pre_hook(mlp, name):
    getattr(mlp, name).register_forward_pre_hook(lambda mod, args: (args[0] + 1,))


def backward_hook(mlp, name):
    getattr(mlp, name).register_full_backward_hook(lambda mod, gi, go: None)


def own_forward(mlp, name):
    proj = getattr(mlp, name)
    proj.forward = lambda x: 3.0 * torch.nn.functional.linear(x, proj.weight)


@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj"])
@pytest.mark.parametrize("change", [wrap, subclass, parametrised, weight_norm, forward_hook, pre_hook, backward_hook,
                                    own_forward])
def test_changed_projections_are_refused(change, name):
    m = torch.nn.ModuleList([DeepseekV2MLP(), DeepseekV2MLP()])
    change(m[1], name)
    with pytest.raises(RuntimeError, match=name):
        gated_ffn.check_module(m[1])
    with pytest.raises(RuntimeError, match=name):
        swaps.SWAPS["deepseek_v2_mlp"][0](m, "custom")
    assert not any("forward" in vars(mod) for mod in m)


@pytest.mark.parametrize("change", [wrap, forward_hook])
def test_projections_changed_after_the_swap_are_refused_when_called(change):
    m = torch.nn.ModuleList([DeepseekV2MLP()])
    swaps.SWAPS["deepseek_v2_mlp"][0](m, "custom")
    change(m[0], "up_proj")
    with pytest.raises(RuntimeError, match="up_proj"):
        m[0](torch.zeros(1, 64, dtype=torch.bfloat16))


def test_activations():
    def silu(x):  # another function of that name
        return x

    class Scaled(torch.nn.SiLU):
        def forward(self, x):
            return 2.0 * super().forward(x)

    hooked = torch.nn.SiLU()
    hooked.register_forward_hook(lambda mod, args, out: -out)
    for act in (silu, Scaled(), hooked, torch.nn.GELU()):
        with pytest.raises(RuntimeError, match="silu"):
            gated_ffn.check_module(DeepseekV2MLP(act=act))
    without = DeepseekV2MLP()
    del without.act_fn
    with pytest.raises(RuntimeError, match="silu"):  # whatever it applies, it is not known to be silu
        gated_ffn.check_module(without)
    gated_ffn.check_module(DeepseekV2MLP(act=torch.nn.SiLU(inplace=True)))


def test_the_transformers_modules_are_taken():
    transformers = pytest.importorskip("transformers")
    from transformers.models.deepseek_v2.modeling_deepseek_v2 import DeepseekV2MLP as Deepseek
    from transformers.models.qwen3_next.modeling_qwen3_next import Qwen3NextMLP as Qwen

    small = dict(hidden_size=64, intermediate_size=96, hidden_act="silu")
    for mlp in (Deepseek(transformers.DeepseekV2Config(**small)), Qwen(transformers.Qwen3NextConfig(**small), 96)):
        gated_ffn.check_module(mlp)


def test_a_forward_that_something_else_set_is_kept():
    """Wrappers that move weights or time calls set an instance's forward: the swap neither replaces nor removes it."""
    apply = swaps.SWAPS["deepseek_v2_mlp"][0]
    m = torch.nn.ModuleList([DeepseekV2MLP(), DeepseekV2MLP()])
    plain = m[1].forward

    def timed(x):
        return plain(x)

    m[1].forward = timed
    with pytest.raises(RuntimeError, match="forward of its own"):
        apply(m, "custom")
    assert "forward" not in vars(m[0]) and m[1].forward is timed
    assert apply(m, "stock") == 2 and m[1].forward is timed
    del m[1].forward
    assert apply(m, "custom") == 2 and apply(m, "custom") == 2  # its own it does replace
    m[0].forward = timed  # set over the swap's
    assert apply(m, "stock") == 2
    assert m[0].forward is timed and "forward" not in vars(m[1])


def test_copies_of_swapped_models_compute_with_their_own_weights(monkeypatch):
    seen = []
    monkeypatch.setattr(gated_ffn, "kernel", lambda x, mlp: seen.append(mlp))
    monkeypatch.setattr(moe_experts_w4, "decode_kernel", lambda x, idx, w, experts: seen.append(experts))
    m = torch.nn.ModuleList([DeepseekV2MLP(), DeepseekV2Experts()])
    swaps.SWAPS["deepseek_v2_mlp"][0](m, "custom")
    swaps.SWAPS["deepseek_v2"][0](m, "custom_w4")
    c = copy.deepcopy(m)
    x, idx, w = torch.zeros(2, 64), torch.zeros(2, 2), torch.zeros(2, 2)
    for mod, args in zip(c, ((x,), (x, idx, w))):
        mod(*args)
    assert seen[0] is c[0] and seen[1] is c[1]
    assert c[1]._cernels_w4[0] is not m[1]._cernels_w4[0]
    for apply in (swaps.SWAPS["deepseek_v2_mlp"][0], swaps.SWAPS["deepseek_v2"][0]):
        assert apply(c, "stock") == 1
    assert not any("forward" in vars(mod) for mod in c) and all("forward" in vars(mod) for mod in m)


def odd_view(x):
    """The same values 2 bytes off a 16-byte boundary."""
    wide = torch.zeros(x.numel() + 9, dtype=x.dtype, device=x.device)
    off = (2 - wide.data_ptr()) % 16 // 2
    view = wide[off:off + x.numel()].view(x.shape)
    view.copy_(x)
    assert view.data_ptr() % 16 == 2
    return view


@pytest.mark.parametrize("make", [lambda x: x, odd_view, lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
                                  lambda x: x[:1].expand(3, 2, 64), lambda x: odd_view(x)[:, 1:]],
                         ids=["plain", "odd", "transposed", "expanded", "odd slice"])
def test_loaders_hand_over_rows_that_the_kernels_can_read(monkeypatch, make):
    x = make(torch.randn(3, 2, 64).to(torch.bfloat16))
    got = []

    def take(rows, *rest):
        got.append(rows)
        return rows

    monkeypatch.setattr(gated_ffn, "gated_ffn", take)
    monkeypatch.setattr(w4, "moe_experts_decode_w4", take)
    assert torch.equal(gated_ffn.kernel(x, DeepseekV2MLP()), x)
    e = DeepseekV2Experts()
    moe_experts_w4.prepare(e)
    flat = x[:, 0]
    moe_experts_w4.decode_kernel(flat, torch.zeros(3, 2), torch.zeros(3, 2), e)
    assert torch.equal(got[1], flat) and got[1].is_contiguous()
    assert all(t.data_ptr() % 16 == 0 and t.stride(1) == 1 for t in got)


@pytest.mark.gpu
def test_a_misaligned_x_through_the_swapped_modules():
    torch.manual_seed(3)
    m = torch.nn.ModuleList([DeepseekV2MLP(device="cuda"), DeepseekV2Experts(device="cuda")])
    swaps.SWAPS["deepseek_v2_mlp"][0](m, "custom")
    swaps.SWAPS["deepseek_v2"][0](m, "custom_w4")
    x = torch.randn(3, 64, device="cuda").to(torch.bfloat16)
    w, idx = torch.rand(3, 4, device="cuda").topk(2, -1)
    with torch.no_grad():
        assert torch.equal(m[0](odd_view(x)), m[0](x)) and torch.equal(m[1](odd_view(x), idx, w), m[1](x, idx, w))
    a, b = x.clone().requires_grad_(), odd_view(x).requires_grad_()
    dy = torch.randn_like(x)
    assert torch.equal(torch.autograd.grad(m[0](a), a, dy)[0], torch.autograd.grad(m[0](b), b, dy)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_autocast_casts_as_the_module_does(kind):
    """32-bit weights in training: the gradients of the cast weights, in 32 bits."""
    torch.manual_seed(4)
    mlp = DeepseekV2MLP(device="cuda").float()
    model = torch.nn.ModuleList([mlp])
    x = torch.randn(40, 64, device="cuda", dtype=kind).requires_grad_()
    dy = torch.randn(40, 64, device="cuda").to(torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        stock = mlp(x)
        swaps.SWAPS["deepseek_v2_mlp"][0](model, "custom")
        y = mlp(x)
    assert y.dtype == stock.dtype == torch.bfloat16
    weights = [mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight]
    cast = [v.detach().to(torch.bfloat16) for v in (x, *weights)]
    want, bound, state = R.forward(*cast)
    R.assert_within("y", y.detach(), want, bound)
    for t, g, (w, b) in zip((x, *weights), torch.autograd.grad(y, (x, *weights), dy), R.backward(state, dy)):
        assert g.dtype == t.dtype
        R.assert_within("gradient", g, w, b)
    with pytest.raises(RuntimeError, match="bf16"):  # no autocast, no cast
        mlp(x)
