"""gated_ffn loader — the dense MLP / shared expert modules beside the routed experts
(transformers' DeepseekV2MLP, Qwen3NextMLP and others with bias-free gate_proj, up_proj,
down_proj and SiLU), which the reference runs as they are
(src/kops/registry/qwen3_next_moe_experts.py:31-44).

``kernel(x, mlp)`` takes hidden states [..., H] and the module. Unlike the experts' loaders it is
differentiable, in x and the module's weights; under ``torch.autocast`` to bf16 x and weights of other
types are cast to it, as they are for the module.
"""

import torch

from ..ffn import gated_ffn, readable


_PROJECTIONS = ("gate_proj", "up_proj", "down_proj")
_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


def _altered(mod) -> bool:
    """Whether calling `mod` does more than its class's forward: hooks, or a forward of its own."""
    d = vars(mod)
    return "forward" in d or any(d.get(h) for h in _HOOKS)


def _is_silu(act) -> bool:
    if act is torch.nn.functional.silu:
        return True
    kind = type(act)
    known = kind is torch.nn.SiLU or (kind.__name__ == "SiLUActivation" and kind.__module__ == "transformers.activations")
    return known and not _altered(act)


def check_module(mlp) -> None:
    """Raises when `mlp` computes something else than down(silu(gate(x)) * up(x)) without biases, as far as its
    parts show: projections that are not torch.nn.Linear itself (adapters, parametrisations, quantised layers) or carry
    hooks, which the operator would pass by, and an activation that is not SiLU."""
    if mlp is None:
        raise RuntimeError("mlp module not available (meta device)")
    for name in _PROJECTIONS:
        proj = getattr(mlp, name)
        if type(proj) is not torch.nn.Linear:
            raise RuntimeError(f"gated_ffn takes plain torch.nn.Linear projections: {name} is {type(proj).__name__}")
        if proj.bias is not None:
            raise RuntimeError(f"gated_ffn has no bias: {name} has one")
        if _altered(proj):
            raise RuntimeError(f"gated_ffn does not call its projections: {name} has hooks or a forward of its own")
    act = getattr(mlp, "act_fn", None)
    if not _is_silu(act):
        raise RuntimeError(f"gated_ffn applies silu, the module {getattr(act, '__name__', type(act).__name__)}")


def kernel(x, mlp):
    check_module(mlp)
    t = x, mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") is torch.bfloat16:
        x, *w = (v.to(torch.bfloat16) for v in t)  # as autocast does for the module's linear layers
    else:
        x, *w = t
    return gated_ffn(readable(x.reshape(-1, x.shape[-1])), *w).reshape(x.shape)
