"""The gated feed-forward block outside the routed experts, with its gradient.

``gated_ffn(x, gate_proj, up_proj, down_proj)`` computes ``(silu(x Wg^T) * (x Wu^T)) Wd^T``:
the dense MLP and the shared expert of the models in :mod:`cernels_b200.registry` (the
reference runs them as torch modules, src/kops/registry/qwen3_next_moe_experts.py:31-44).
It is ``torch.ops.cernels_b200.gated_ffn`` too, and differentiable in all four arguments;
gradients are deterministic. The backward pass keeps, per token, 2F values in 32 bits and F in
bf16. Like the experts operators it runs on the current stream, takes scratch from torch's
caching allocator and never synchronises.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _check

_BF16 = torch.bfloat16


def rows_ok(x: torch.Tensor) -> bool:
    """Whether the kernels can read the rows of x where they lie."""
    return x.stride(1) == 1 and (x.shape[0] <= 1 or (x.stride(0) >= x.shape[1] and x.stride(0) % 8 == 0))


def readable(x: torch.Tensor) -> torch.Tensor:
    """x, or a copy of it where the kernels cannot read its rows in place: for loaders, whose modules take any x."""
    if rows_ok(x) and (traced(x) or x.data_ptr() % 16 == 0):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def int32_sizes(*sizes: int) -> None:
    """Refuses sizes that the C ABI's 32-bit fields would wrap."""
    _check(max(sizes) < 1 << 31, "sizes must be below 2^31")


def refuse_tangents(name: str, *tensors: torch.Tensor) -> None:
    """Raises for forward-mode inputs: the operators have no such derivative, and a tangent must not get lost."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            _check(forward_ad.unpack_dual(t).tangent is None, f"{name} has no forward-mode derivative")


class _Plan(NamedTuple):
    shape: _lib.FfnShape
    ref: object  # ctypes.byref(shape)
    workspace: int  # bytes
    backward_workspace: int
    saved: int


@functools.lru_cache(maxsize=1024)
def _plan(tokens: int, hidden: int, intermediate: int) -> _Plan:
    """What the C ABI says about a call of these sizes (its queries are a few us of a 10 us call)."""
    int32_sizes(tokens, hidden, intermediate)
    shape = _lib.FfnShape(tokens, hidden, intermediate)
    ref, lib, n = ctypes.byref(shape), _lib.load(), ctypes.c_size_t(0)
    sizes = []
    for backward in (0, 1):
        _lib.check(lib.cernels_gated_ffn_workspace_bytes(ref, backward, ctypes.byref(n)), "workspace query")
        sizes.append(n.value)
    _lib.check(lib.cernels_gated_ffn_saved_bytes(ref, ctypes.byref(n)), "size query")
    return _Plan(shape, ref, *sizes, n.value)


def _validate(x, gate_proj, up_proj, down_proj) -> _Plan:
    _check(x.is_cuda, "x must be a CUDA tensor")
    _check(x.dim() == 2 and x.dtype is _BF16, "x must be [T, H] bf16")
    T, H = x.shape
    dev = x.device
    for w in (gate_proj, up_proj, down_proj):
        if not (w.device == dev and w.dtype is _BF16 and w.is_contiguous()):
            raise RuntimeError(f"gate_proj, up_proj and down_proj must be contiguous bf16 on {dev}")
    _check(gate_proj.dim() == 2, "gate_proj must be [F, H]")
    F = gate_proj.shape[0]
    _check(gate_proj.shape == (F, H) and up_proj.shape == (F, H), "gate_proj and up_proj must be [F, H]")
    _check(down_proj.shape == (H, F), "down_proj must be [H, F]")
    _check(H > 0 and F > 0 and H % 8 == 0 and F % 8 == 0, "H and F must be multiples of 8")
    _check(rows_ok(x), "x must have contiguous rows, a multiple of 8 elements (and at least H) apart")
    return _plan(T, H, F)


def _stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


# The current stream's handle; the public call builds a Stream object first, 2 us of a 10 us call.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device: torch.device, name: str, *args) -> None:
    """Calls a C-ABI entry, whose last argument is the stream, with `device` current."""
    fn = getattr(_lib.load(), name)
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter))
_compiling = torch.compiler.is_compiling
_modes = torch._C._len_torch_dispatch_stack
_transform = torch._C._functorch.peek_interpreter_stack
_jit = torch._C._get_tracing_state


def traced(*tensors: torch.Tensor) -> bool:
    """Whether a call has to go through torch's dispatcher: tensors that stand for others (fake ones of torch.compile and
    torch.export, wrappers), or a mode or transform that wants to see it. Else it launches at once: the way there and
    back is a few us of a 10 us call."""
    if _compiling() or _modes() or _transform() is not None or _jit() is not None:
        return True
    for t in tensors:
        if type(t) not in _PLAIN:
            return True
    return False


def below_autograd(op, *args):
    """Calls `op` at the implementations below autograd's: a device's, Meta, or a tracer."""
    with torch._C._AutoDispatchBelowAutograd():
        return op(*args)


def _forward(x, gate_proj, up_proj, down_proj) -> torch.Tensor:
    plan = _validate(x, gate_proj, up_proj, down_proj)
    out = x.new_empty(x.shape)
    if x.shape[0] == 0:
        return out
    ws = x.new_empty((plan.workspace + 1) // 2)
    _call(x.device, "cernels_gated_ffn", plan.ref, x.data_ptr(), _stride(x), gate_proj.data_ptr(),
          up_proj.data_ptr(), down_proj.data_ptr(), out.data_ptr(), ws.data_ptr(), plan.workspace)
    return out


def _train(x, gate_proj, up_proj, down_proj) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The result and what the backward pass reads: silu(g) * u in bf16, g and u in 32 bits (the kernels' order)."""
    plan = _validate(x, gate_proj, up_proj, down_proj)
    out = x.new_empty(x.shape)
    act = x.new_empty((plan.shape.tokens, plan.shape.intermediate))
    saved = x.new_empty(plan.saved // 4, dtype=torch.float32)
    if plan.shape.tokens:
        _call(x.device, "cernels_gated_ffn_forward", plan.ref, x.data_ptr(), _stride(x), gate_proj.data_ptr(),
              up_proj.data_ptr(), down_proj.data_ptr(), out.data_ptr(), act.data_ptr(), saved.data_ptr())
    return out, act, saved


def _grads(dout, x, gate_proj, up_proj, down_proj, act, saved, needs) -> tuple[torch.Tensor | None, ...]:
    """The gradients of the arguments that `needs` marks."""
    plan = _plan(x.shape[0], x.shape[1], gate_proj.shape[0])
    dout = dout.contiguous()
    if dout.data_ptr() % 16:
        dout = dout.clone()
    grads = [dout.new_empty(t.shape) if need else None for t, need in zip((x, gate_proj, up_proj, down_proj), needs)]
    ws = dout.new_empty((plan.backward_workspace + 1) // 2)
    _call(x.device, "cernels_gated_ffn_backward", plan.ref, x.data_ptr(), _stride(x), gate_proj.data_ptr(),
          up_proj.data_ptr(), down_proj.data_ptr(), act.data_ptr(), saved.data_ptr(), dout.data_ptr(),
          *(None if g is None else g.data_ptr() for g in grads), ws.data_ptr(), plan.backward_workspace)
    return tuple(grads)


def _grads_op(*args) -> list[torch.Tensor]:
    return [g for g in _grads(*args) if g is not None]


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_proj, up_proj, down_proj):
        out, act, saved = _train(x, gate_proj, up_proj, down_proj)
        ctx.save_for_backward(x, gate_proj, up_proj, down_proj, act, saved)
        return out

    @staticmethod
    def backward(ctx, dout):
        # Gradients of gradients are refused; the wrapper that sees to that is only needed, and only
        # paid for, where the caller records the backward pass.
        return (_backward_recorded if torch.is_grad_enabled() else _backward)(ctx, dout)


class _TracedGatedFfn(_GatedFfn):
    @staticmethod
    def forward(ctx, *t):
        out, act, saved = below_autograd(_ops.gated_ffn_train, *t)
        ctx.save_for_backward(*t, act, saved)
        return out


def _backward(ctx, dout):
    needs, saved = ctx.needs_input_grad, ctx.saved_tensors
    if not traced(dout):
        return _grads(dout, *saved, needs)
    grads = iter(below_autograd(_ops.gated_ffn_backward, dout, *saved, needs))
    return tuple(next(grads) if need else None for need in needs)


_backward_recorded = once_differentiable(_backward)


def gated_ffn(x: torch.Tensor, gate_proj: torch.Tensor, up_proj: torch.Tensor, down_proj: torch.Tensor) -> torch.Tensor:
    """``(silu(x @ gate_proj.T) * (x @ up_proj.T)) @ down_proj.T``.

    x [T, H] bf16 whose rows may lie apart (row stride a multiple of 8); gate_proj and up_proj
    [F, H], down_proj [H, F], contiguous bf16; H and F multiples of 8. Sums run in 32 bits; the
    product of the halves is rounded to bf16 once, as the second matrix product's operand.
    """
    if traced(x, gate_proj, up_proj, down_proj):
        return _ops.gated_ffn(x, gate_proj, up_proj, down_proj)
    if _records(x, gate_proj, up_proj, down_proj):
        return _GatedFfn.apply(x, gate_proj, up_proj, down_proj)
    return _forward(x, gate_proj, up_proj, down_proj)


def _records(x, gate_proj, up_proj, down_proj) -> bool:
    refuse_tangents("gated_ffn", x, gate_proj, up_proj, down_proj)
    return torch.is_grad_enabled() and (x.requires_grad or gate_proj.requires_grad or up_proj.requires_grad
                                        or down_proj.requires_grad)


def _dispatched(*t):
    if _records(*t):
        return (_TracedGatedFfn if traced(*t) else _GatedFfn).apply(*t)
    return below_autograd(_ops.gated_ffn, *t) if traced(*t) else _forward(*t)


def _meta(x, gate_proj, up_proj, down_proj):
    return x.new_empty((x.shape[0], down_proj.shape[0]))


def _meta_train(x, gate_proj, up_proj, down_proj):
    T, F = x.shape[0], gate_proj.shape[0]
    return (_meta(x, gate_proj, up_proj, down_proj), x.new_empty((T, F)),
            x.new_empty((T + 31) // 32 * 32 * 2 * F, dtype=torch.float32))


def _meta_grads(dout, x, gate_proj, up_proj, down_proj, act, saved, needs):
    return [t.new_empty(t.shape) for t, need in zip((x, gate_proj, up_proj, down_proj), needs) if need]


def status(device: torch.device | str | int | None = None) -> int:
    """0, or the code of a bounded wait that gave up in one of these kernels on `device` (default: the current one) since
    the last call, whoever made it; the results since then are not to be used. Synchronises the current stream."""
    code = ctypes.c_int(0)
    index = device if isinstance(device, int) else None
    if device is not None and index is None:
        dev = torch.device(device)
        _check(dev.type == "cuda", f"no such word on {dev}")
        index = dev.index
    index = torch.cuda.current_device() if index is None else index
    with torch.cuda.device(index):
        _lib.check(_lib.load().cernels_ffn_status(ctypes.byref(code), torch.cuda.current_stream(index).cuda_stream),
                   "cernels_ffn_status")
    return code.value


_DEF = torch.library.Library("cernels_b200", "FRAGMENT")
_ARGS = "Tensor x, Tensor gate_proj, Tensor up_proj, Tensor down_proj"
_DEF.define(f"gated_ffn({_ARGS}) -> Tensor")
_DEF.define(f"gated_ffn_train({_ARGS}) -> (Tensor, Tensor, Tensor)")
_DEF.define(f"gated_ffn_backward(Tensor dout, {_ARGS}, Tensor act, Tensor saved, bool[] needs) -> Tensor[]")
_DEF.impl("gated_ffn", _forward, "CUDA")
_DEF.impl("gated_ffn", _dispatched, "AutogradCUDA")
_DEF.impl("gated_ffn", _meta, "Meta")
# the halves of a training step, as a traced one records them
_DEF.impl("gated_ffn_train", _train, "CUDA")
_DEF.impl("gated_ffn_train", _meta_train, "Meta")
_DEF.impl("gated_ffn_backward", _grads_op, "CUDA")
_DEF.impl("gated_ffn_backward", _meta_grads, "Meta")
_ops = torch.ops.cernels_b200
