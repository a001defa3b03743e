"""gated_ffn loader — the dense MLP / shared expert modules beside the routed experts
(transformers' DeepseekV2MLP, Qwen3NextMLP and others with bias-free gate_proj, up_proj,
down_proj and SiLU), which the reference runs as they are
(src/kops/registry/qwen3_next_moe_experts.py:31-44).

``kernel(x, mlp)`` takes hidden states [..., H] and the module. Unlike the experts' loaders it is
differentiable, in x and the module's weights.
"""

import torch

from ..ffn import gated_ffn, rows_ok


def check_module(mlp) -> None:
    """Raises when `mlp` computes something else than down(silu(gate(x)) * up(x)) without biases."""
    if mlp is None:
        raise RuntimeError("mlp module not available (meta device)")
    for name in ("gate_proj", "up_proj", "down_proj"):
        if getattr(mlp, name).bias is not None:
            raise RuntimeError(f"gated_ffn has no bias: {name} has one")
    act = getattr(mlp, "act_fn", None)
    if act is not None and not isinstance(act, torch.nn.SiLU) and getattr(act, "__name__", "") != "silu":
        if type(act).__name__ not in ("SiLU", "SiLUActivation"):
            raise RuntimeError(f"gated_ffn applies silu, the module {type(act).__name__}")


def kernel(x, mlp):
    check_module(mlp)
    xf = x.reshape(-1, x.shape[-1])
    y = gated_ffn(xf if rows_ok(xf) else xf.contiguous(), mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight)
    return y.reshape(x.shape)
