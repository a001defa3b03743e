"""Products with 4-bit weights and group scales, for the decode path.

A weight row of K values is stored as K / 2 bytes (two codes a byte, the even position in the low
half) and K / G bf16 scales, G 32, 64 or 128::

    W[n, k] = (q[n, k] - 8) * scale[n, k // G]

Weights are never rounded and sums are in 32 bits. A block of 128 values of x is taken as 14 bits and a sign below its
largest value if at least half of its nonzero values are exact that way (none is then off by more than 2^-8 of the
block's median); else, and with an infinity or a NaN in it, it is multiplied exactly in bf16.

``linear_w4`` is a linear layer for a few rows; ``moe_experts_decode_w4`` is the routed experts'
decode call (``*_moe_experts_decode``) on such weights, a quarter of the bytes that bound it;
``quantize_w4`` makes the codes and scales from bf16 weights. The first two are
``torch.ops.cernels_b200.*`` too. They are for inference: a call that would need a gradient raises.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .ffn import _call, below_autograd, int32_sizes, refuse_tangents, rows_ok, _stride, traced
from .ops import DECODE_MAX_PAIRS, _check

_BF16 = torch.bfloat16
GROUPS = (32, 64, 128)


def quantize_w4(weight: torch.Tensor, group: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes [..., K / 2] uint8, scales [..., K / group] bf16) of weight [..., K], each group scaled by
    its largest magnitude / 7 and rounded to the nearest code (a group of zeros gets scale 0)."""
    _check(group in GROUPS, f"group must be one of {GROUPS}")
    _check(weight.dim() >= 2 and weight.is_floating_point(), "weight must be a floating [..., N, K] tensor")
    _check(weight.shape[-1] % group == 0 and weight.shape[-1] > 0, "K must be a multiple of group")
    w = weight.detach().float().unflatten(-1, (-1, group))
    scale = (w.abs().amax(-1) / 7.0).to(_BF16)
    q = w / torch.where(scale == 0, torch.ones_like(scale), scale).float().unsqueeze(-1)
    q = (torch.round(q) + 8.0).clamp_(0.0, 15.0).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), scale


def _check_no_grad(*tensors: torch.Tensor) -> None:
    refuse_tangents("a 4-bit product", *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            _check(not t.requires_grad, "4-bit products have no gradient: call them under torch.no_grad()")


def _check_w4(name: str, q: torch.Tensor, s: torch.Tensor, lead: tuple, k: int, dev: torch.device) -> int:
    """The group size of codes q [*lead, k / 2] with scales s [*lead, k / G]."""
    if not (q.device == dev and s.device == dev and q.dtype is torch.uint8 and s.dtype is _BF16
            and q.is_contiguous() and s.is_contiguous()):
        raise RuntimeError(f"{name} must be contiguous uint8 codes and bf16 scales on {dev}")
    n_groups = s.shape[-1]
    if k % 2 or q.shape != (*lead, k // 2) or s.shape != (*lead, n_groups) or n_groups == 0:
        raise RuntimeError(f"{name}: codes must be {[*lead, k // 2]} and scales {[*lead, 'K / group']}")
    group = k // n_groups
    if group not in GROUPS or group * n_groups != k:
        raise RuntimeError(f"{name}: group must be one of {GROUPS} and divide K")
    return group


def _linear_w4(x, qweight, scales):
    _check(x.is_cuda, "x must be a CUDA tensor")
    _check(x.dim() == 2 and x.dtype is _BF16, "x must be [T, K] bf16")
    _check(qweight.dim() == 2, "qweight must be [N, K / 2]")
    T, K = x.shape
    N = qweight.shape[0]
    group = _check_w4("qweight", qweight, scales, (N,), K, x.device)
    _check(rows_ok(x), "x must have contiguous rows, a multiple of 8 elements (and at least K) apart")
    if scales.data_ptr() % 4:  # rows of a slice may start in the middle of the words that the kernel copies
        scales = scales.clone()
    int32_sizes(T, N, K)
    out = x.new_empty((T, N))
    if T and N:
        _call(x.device, "cernels_linear_w4", T, N, K, group, x.data_ptr(), _stride(x), qweight.data_ptr(),
              scales.data_ptr(), out.data_ptr())
    return out


def linear_w4(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """``x @ W.T`` for 4-bit W: x [T, K] bf16 (rows may lie apart), qweight [N, K / 2] uint8, scales
    [N, K / G] bf16. Made for a few rows, where the weights' bytes bound it: they are read once for as many rows as
    shared memory holds, at most 16 (16 up to K = 4864, 9 at 8192, 2 at 32768). More rows work."""
    if traced(x, qweight, scales):
        return _ops.linear_w4(x, qweight, scales)
    _check_no_grad(x, scales)
    return _linear_w4(x, qweight, scales)


def _linear_dispatched(x, qweight, scales):
    _check_no_grad(x, scales)
    t = x, qweight, scales
    return below_autograd(_ops.linear_w4, *t) if traced(*t) else _linear_w4(*t)


@functools.lru_cache(maxsize=1024)
def _moe_plan(tokens: int, hidden: int, experts: int, inter: int, topk: int, group: int):
    """The C ABI's shape (kept alive by the reference to it that is returned) and workspace bytes."""
    int32_sizes(tokens, hidden, experts, inter, topk)
    ref, n = ctypes.byref(_lib.MoeShape(tokens, hidden, experts, inter, topk, _lib.LAYOUT_LINEAR)), ctypes.c_size_t(0)
    _lib.check(_lib.load().cernels_moe_w4_workspace_bytes(ref, group, ctypes.byref(n)), "workspace query")
    return ref, n.value


def _moe_experts_decode_w4(x, gate_up_q, gate_up_scales, down_q, down_scales, indices, weights, topk):
    _check(x.is_cuda, "x must be a CUDA tensor")
    _check(x.dim() == 2 and x.dtype == _BF16 and x.is_contiguous(), "x must be contiguous [T, H] bf16")
    _check(gate_up_q.dim() == 3 and gate_up_q.shape[1] % 2 == 0, "gate_up_q must be [E, 2F, H / 2]")
    T, H = x.shape
    E, F = gate_up_q.shape[0], gate_up_q.shape[1] // 2
    group = _check_w4("gate_up_q", gate_up_q, gate_up_scales, (E, 2 * F), H, x.device)
    _check(_check_w4("down_q", down_q, down_scales, (E, H), F, x.device) == group,
           "gate_up and down weights must have the same group")
    for name, t, dtype in (("indices", indices, torch.int32), ("weights", weights, torch.float32)):
        _check(t.device == x.device and t.dtype == dtype and t.is_contiguous() and tuple(t.shape) == (T, topk),
               f"{name} must be contiguous [T, topk] {dtype} on {x.device}")
    _check(T * topk <= DECODE_MAX_PAIRS, f"at most {DECODE_MAX_PAIRS} (token, slot) pairs per call")
    out = x.new_empty((T, H))
    if T == 0:
        return out
    ref, n = _moe_plan(T, H, E, F, topk, group)
    ws = x.new_empty((n + 1) // 2)
    _call(x.device, "cernels_moe_experts_decode_w4", ref, group, x.data_ptr(), gate_up_q.data_ptr(),
          gate_up_scales.data_ptr(), down_q.data_ptr(), down_scales.data_ptr(), indices.data_ptr(), weights.data_ptr(),
          out.data_ptr(), ws.data_ptr(), n)
    return out


def moe_experts_decode_w4(x: torch.Tensor, gate_up_q: torch.Tensor, gate_up_scales: torch.Tensor, down_q: torch.Tensor,
                          down_scales: torch.Tensor, indices: torch.Tensor, weights: torch.Tensor,
                          topk: int) -> torch.Tensor:
    """``cohere2_moe_experts_decode`` (and the other experts of its layout) on 4-bit weights.

    x [T, H] bf16; gate_up_q [E, 2F, H / 2], down_q [E, H, F / 2] uint8 with their scales; indices
    [T, topk] int32 (ids outside [0, E) are skipped), weights [T, topk] fp32. At most 1024 pairs.
    """
    t = x, gate_up_q, gate_up_scales, down_q, down_scales, indices, weights
    if traced(*t):
        return _ops.moe_experts_decode_w4(*t, topk)
    _check_no_grad(x, gate_up_scales, down_scales, weights)
    return _moe_experts_decode_w4(*t, topk)


def _moe_dispatched(x, gate_up_q, gate_up_scales, down_q, down_scales, indices, weights, topk):
    _check_no_grad(x, gate_up_scales, down_scales, weights)
    t = x, gate_up_q, gate_up_scales, down_q, down_scales, indices, weights
    return below_autograd(_ops.moe_experts_decode_w4, *t, topk) if traced(*t) else _moe_experts_decode_w4(*t, topk)


_DEF = torch.library.Library("cernels_b200", "FRAGMENT")
_DEF.define("linear_w4(Tensor x, Tensor qweight, Tensor scales) -> Tensor")
_DEF.define("moe_experts_decode_w4(Tensor x, Tensor gate_up_q, Tensor gate_up_scales, Tensor down_q, "
            "Tensor down_scales, Tensor indices, Tensor weights, int topk) -> Tensor")
_DEF.impl("linear_w4", _linear_w4, "CUDA")
_DEF.impl("linear_w4", _linear_dispatched, "AutogradCUDA")
_DEF.impl("linear_w4", lambda x, qweight, scales: x.new_empty((x.shape[0], qweight.shape[0])), "Meta")
_DEF.impl("moe_experts_decode_w4", _moe_experts_decode_w4, "CUDA")
_DEF.impl("moe_experts_decode_w4", _moe_dispatched, "AutogradCUDA")
_DEF.impl("moe_experts_decode_w4", lambda x, *rest: torch.empty_like(x), "Meta")
_ops = torch.ops.cernels_b200
