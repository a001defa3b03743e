"""In-model swaps: replace the forward of every transformers experts module of a class with
this library's operators — the reference's swap point #2 (src/modeling/swaps.py).

As in the reference, the replacement is an instance attribute (``mod.forward``), so deleting it
("stock") restores the class method, and the forward picks the decode entry point at or below
DECODE_MAX_TOKENS tokens and the prefill entry point above (src/modeling/swaps.py:13,20-42).
The ops take no host synchronisation, so a swapped model can be captured in a CUDA graph.

SWAPS maps a model name to (apply(model, variant), variants), stock first.
"""

from __future__ import annotations

import functools
from typing import Callable

import torch

DECODE_MAX_TOKENS = 4  # at or below this many tokens the decode entry point handles the op


# Forwards are partial objects of the module: a copy of a swapped model (copy.deepcopy) gets ones of its own modules,
# where a closure would go on computing with the original's.
def _experts_forward(mod, kernel: Callable | None, decode_kernel: Callable | None, h, idx, w):
    op = decode_kernel if h.size(0) <= DECODE_MAX_TOKENS else kernel
    if op is None:  # this shape's entry point is not enabled in this variant
        return type(mod).forward(mod, h, idx, w)
    return op(h, idx, w, mod)


def swap_experts(model: torch.nn.Module, cls_name: str, kernel: Callable | None,
                 decode_kernel: Callable | None) -> int:
    """Sets (or, with both kernels None, restores) the forward of every `cls_name` instance.
    Returns the number of modules touched; raises when the model has none."""
    n = 0
    for mod in model.modules():
        if type(mod).__name__ != cls_name:
            continue
        n += 1
        if "forward" in vars(mod):
            del mod.forward
        if kernel is not None or decode_kernel is not None:
            mod.forward = functools.partial(_experts_forward, mod, kernel, decode_kernel)
    if not n:
        raise RuntimeError(f"no {cls_name} modules found — wrong model for this swap")
    return n


# ---------------------------------------------------------------- per-family kernels
def _linear_kernels():
    from .registry import cohere2_moe_experts as c2

    return c2.kernel, c2.decode_kernel


def _gpt_oss_kernels():
    """GptOssExperts.forward(hidden, router_indices, routing_weights) with its biases."""
    from . import ops
    from .registry import gpt_oss_moe_experts as go

    def prefill(h, idx, w, mod):
        w1, b1, w2, b2 = go._weights(mod)
        with torch.no_grad():
            return ops.gpt_oss_moe_experts(h.contiguous(), w1, b1, w2, b2, idx.to(torch.int32).contiguous(),
                                           w.float().contiguous(), int(idx.size(1)))

    def decode(h, idx, w, mod):
        w1, b1, w2, b2 = go._weights(mod)
        with torch.no_grad():
            return ops.gpt_oss_moe_experts_decode(h.contiguous(), w1, b1, w2, b2, idx.to(torch.int32).contiguous(),
                                                  w.float().contiguous(), int(idx.size(1)))

    return prefill, decode


def _family(cls_name: str, kernels: Callable):
    def apply(model, variant: str):
        if variant == "stock":
            return swap_experts(model, cls_name, None, None)
        kernel, decode_kernel = kernels()
        return swap_experts(model, cls_name, kernel, decode_kernel if variant == "custom" else None)

    return apply


def _linear_family(cls_name: str):
    """Experts of the LINEAR layout, with a variant that decodes on 4-bit copies of the weights (made
    here, once: apply it again after changing them) and prefills on the bf16 ones."""
    plain = _family(cls_name, _linear_kernels)

    def apply(model, variant: str):
        from .registry import moe_experts_w4

        if variant != "custom_w4":
            for mod in model.modules():
                if type(mod).__name__ == cls_name:
                    moe_experts_w4.release(mod)
            return plain(model, variant)
        mods = [m for m in model.modules() if type(m).__name__ == cls_name]
        for mod in mods:  # all of them or none
            moe_experts_w4.group_of(mod.gate_up_proj.shape[2], mod.down_proj.shape[2])
        for mod in mods:
            moe_experts_w4.prepare(mod)
        return swap_experts(model, cls_name, _linear_kernels()[0], moe_experts_w4.decode_kernel)

    return apply


def _mlp_forward(mlp, x):
    from .registry import gated_ffn

    return gated_ffn.kernel(x, mlp)


def swap_mlps(model: torch.nn.Module, cls_name: str, custom: bool) -> int:
    """Sets (or restores) the forward of every `cls_name` instance, a dense gated MLP (gate_proj, up_proj,
    down_proj), to the gated feed-forward operator, which is differentiable. A forward that something else has set on an
    instance is neither replaced (that raises, and leaves the model as it was) nor taken away. Returns the number of
    modules of the class; raises when the model has none."""
    from .registry import gated_ffn

    mods = [m for m in model.modules() if type(m).__name__ == cls_name]
    if not mods:
        raise RuntimeError(f"no {cls_name} modules found — wrong model for this swap")
    ours = [getattr(vars(m).get("forward"), "func", None) is _mlp_forward for m in mods]
    if custom:  # all of them or none
        for mod, mine in zip(mods, ours):
            if "forward" in vars(mod) and not mine:
                raise RuntimeError(f"a {cls_name} has a forward of its own, which this swap would replace")
            gated_ffn.check_module(mod)
    for mod, mine in zip(mods, ours):
        if mine:
            del mod.forward
        if custom:
            mod.forward = functools.partial(_mlp_forward, mod)
    return len(mods)


def _mlp_family(cls_name: str):
    return lambda model, variant: swap_mlps(model, cls_name, variant != "stock")


_LINEAR_VARIANTS = ("stock", "custom_prefill", "custom", "custom_w4")

SWAPS = {
    # the reference's two models (their experts classes need transformers >= 5.10)
    "north_mini_code": (_linear_family("Cohere2MoeExperts"), _LINEAR_VARIANTS),
    "deepseek_ocr_2": (_linear_family("DeepseekOcr2TextExperts"), _LINEAR_VARIANTS),
    # experts classes of the installed transformers with the same contracts
    "deepseek_v2": (_linear_family("DeepseekV2Experts"), _LINEAR_VARIANTS),
    "qwen3_next": (_linear_family("Qwen3NextExperts"), _LINEAR_VARIANTS),
    "gpt_oss": (_family("GptOssExperts", _gpt_oss_kernels), ("stock", "custom_prefill", "custom")),
    # the dense layers and shared experts beside them, for training and serving
    "deepseek_v2_mlp": (_mlp_family("DeepseekV2MLP"), ("stock", "custom")),
    "qwen3_next_mlp": (_mlp_family("Qwen3NextMLP"), ("stock", "custom")),
}
