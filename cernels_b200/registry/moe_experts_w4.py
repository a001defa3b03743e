"""Decode loader on 4-bit copies of the experts' weights.

``prepare(experts)`` quantises an experts module's gate_up_proj and down_proj and keeps the copies on
it, a quarter of their size; ``decode_kernel(x, top_k_index, top_k_weights, experts)`` then has the
contract of the ``decode_kernel`` of cohere2 / deepseek_ocr2
(src/kops/registry/cohere2_moe_experts.py), for every experts module of that layout. The copies
are made when ``prepare`` is called and not looked after: call it again when the weights change.
``release(experts)`` drops them.
"""

import torch

from .. import w4
from ..ffn import readable
from ._common import routing_tensors

_SLOT = "_cernels_w4"


def group_of(hidden: int, inter: int) -> int:
    """The largest group that divides both widths."""
    for group in sorted(w4.GROUPS, reverse=True):
        if hidden % group == 0 and inter % group == 0:
            return group
    raise RuntimeError(f"4-bit experts need widths that are multiples of {min(w4.GROUPS)}: got {hidden} and {inter}")


def prepare(experts, group: int | None = None):
    """Quantises the module's weights; returns and keeps (gate_up codes, gate_up scales, down codes,
    down scales)."""
    if experts is None:
        raise RuntimeError("experts module not available (meta device)")
    w1, w2 = experts.gate_up_proj, experts.down_proj
    group = group_of(w1.shape[2], w2.shape[2]) if group is None else group
    # one expert at a time: the quantiser works in fp32
    parts = [[w4.quantize_w4(w, group) for w in t.data] for t in (w1, w2)]
    copies = tuple(torch.stack([p[i] for p in side]) for side in parts for i in (0, 1))
    setattr(experts, _SLOT, copies)
    return copies


def release(experts) -> None:
    if hasattr(experts, _SLOT):
        delattr(experts, _SLOT)


def decode_kernel(x, top_k_index, top_k_weights, experts):
    copies = getattr(experts, _SLOT, None)
    if copies is None:
        raise RuntimeError("no 4-bit weights on this module: call moe_experts_w4.prepare(experts) first")
    with torch.no_grad():
        idx, w = routing_tensors(top_k_index, top_k_weights)
        return w4.moe_experts_decode_w4(readable(x.contiguous()), *copies, idx, w, int(top_k_index.size(1)))
