"""The gated feed-forward block and its gradient, against 64 bits (bounds: ffn_reference)."""

import threading

import pytest
import torch

import cernels_b200
from cernels_b200 import _lib, ffn
from tests import ffn_reference as R

gpu = pytest.mark.gpu
# one token, a token more or less than the tiles' 32 / 128 / 256 rows, widths that no tile or K block
# divides, widths under one K block, several tiles each way
SHAPES = [(1, 64, 64), (2, 8, 8), (5, 72, 40), (16, 256, 136), (17, 2048, 512), (31, 200, 264), (33, 64, 72), (48, 72, 520), (49, 72, 520),
          (20, 16384, 8), (20, 8, 16384), (3, 65536, 8),
          # more tiles than a CTA takes at once, at every number of columns that has a kernel of its own
          (1, 64, 40000), (4, 40000, 64), (3, 4096, 8192), (9, 72, 40000), (13, 2880, 2880), (16, 40000, 72), (33, 64, 20000),
          # rows of x that shared memory does not hold
          (2, 131072, 8), (1, 8, 131072), (127, 328, 128),
          (128, 64, 192), (129, 520, 384), (255, 136, 264), (257, 1024, 520), (512, 768, 256), (700, 2880, 328),
          (1300, 136, 1408)]


def leaves(args):
    return [a.clone().requires_grad_() for a in args]


# ---------------------------------------------------------------- CPU: refusals
def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_refuses_cpu_tensors():
    t = [torch.zeros(2, 8, dtype=torch.bfloat16)] * 3 + [torch.zeros(8, 2, dtype=torch.bfloat16)]
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        cernels_b200.gated_ffn(*t)


def test_meta_shape():
    y = torch.ops.cernels_b200.gated_ffn(meta(5, 64), meta(32, 64), meta(32, 64), meta(64, 32))
    assert y.shape == (5, 64) and y.dtype == torch.bfloat16


@pytest.mark.parametrize("bad,code", [((-1, 64, 64), 1), ((4, 0, 64), 1), ((4, 64, 0), 1), ((4, 60, 64), 2), ((4, 64, 4), 2),
                                      ((4, 1 << 21, 64), 5)])
def test_c_entry_refuses_shapes(bad, code):
    import ctypes

    s, n = _lib.FfnShape(*bad), ctypes.c_size_t(0)
    lib = _lib.load()
    assert lib.cernels_gated_ffn_workspace_bytes(ctypes.byref(s), 0, ctypes.byref(n)) == code
    assert lib.cernels_gated_ffn_saved_bytes(ctypes.byref(s), ctypes.byref(n)) == code


@pytest.mark.parametrize("sizes", [(2**32 + 1, 8, 8), (1, 2**31, 8), (1, 8, 2**32 + 8)])
def test_sizes_do_not_wrap(sizes):
    with pytest.raises(RuntimeError, match="2\\^31"):
        ffn._plan(*sizes)


def test_c_entry_refuses_pointers():
    import ctypes

    lib = _lib.load()
    s = _lib.FfnShape(4, 64, 64)
    ok, odd = 1 << 20, (1 << 20) + 8  # never read: refused before any launch
    call = lib.cernels_gated_ffn
    assert call(ctypes.byref(s), None, 64, ok, ok, ok, ok, ok, 1 << 20, None) == 6
    assert call(ctypes.byref(s), odd, 64, ok, ok, ok, ok, ok, 1 << 20, None) == 2
    assert call(ctypes.byref(s), ok, 60, ok, ok, ok, ok, ok, 1 << 20, None) == 2
    assert call(ctypes.byref(s), ok, 32, ok, ok, ok, ok, ok, 1 << 20, None) == 1
    assert lib.cernels_gated_ffn_workspace_bytes(ctypes.byref(s), 0, None) == 6
    assert call(None, ok, 64, ok, ok, ok, ok, ok, 1 << 20, None) == 6


# ---------------------------------------------------------------- GPU
@gpu
@pytest.mark.parametrize("T,H,F", SHAPES)
def test_forward(T, H, F):
    *args, _ = R.case(T, H, F, seed=T + H)
    want, bound, _ = R.forward(*args)
    R.assert_within("y", cernels_b200.gated_ffn(*args), want, bound)
    R.assert_within("op y", torch.ops.cernels_b200.gated_ffn(*args), want, bound)
    assert ffn.status() == 0


@gpu
@pytest.mark.parametrize("T,H,F", SHAPES)
def test_gradients(T, H, F):
    *args, dy = R.case(T, H, F, seed=T + F)
    want, bound, state = R.forward(*args)
    t = leaves(args)
    y = cernels_b200.gated_ffn(*t)
    R.assert_within("y", y.detach(), want, bound)
    got = torch.autograd.grad(y, t, dy)
    for name, g, (w, b) in zip(("dx", "dgate", "dup", "ddown"), got, R.backward(state, dy)):
        R.assert_within(name, g, w, b)
    assert ffn.status() == 0


@gpu
def test_gradients_against_differences():
    """The gradient along a direction equals the difference quotient of the 64-bit function: with a
    step of 2^-14 its truncation is under 1e-6 of the curvature terms, allowed for as 1e-5 of the sum
    of magnitudes."""
    *args, dy = R.case(40, 128, 96, seed=3)
    t = leaves(args)
    got = torch.autograd.grad(cernels_b200.gated_ffn(*t), t, dy)
    bounds = [b for _, b in R.backward(R.forward(*args)[2], dy)]
    step = 2.0 ** -14
    for i in range(4):
        v = torch.randn_like(args[i], dtype=torch.float32).double()
        hi, lo = ([a.double() + (sign * step * v if j == i else 0.0) for j, a in enumerate(args)] for sign in (1, -1))
        quotient = ((R.forward(*hi)[0] - R.forward(*lo)[0]) * dy.double()).sum() / (2 * step)
        along = (got[i].double() * v).sum()
        room = (bounds[i] * v.abs()).sum() + 1e-5 * (got[i].double() * v).abs().sum()
        assert (along - quotient).abs() <= room, (i, along.item(), quotient.item(), room.item())


@gpu
def test_more_than_2_31_stored_values():
    """So many tokens that what the backward pass stores is indexed past 32 bits; the last rows' results
    and input gradients, and weight gradients that only they feed."""
    T, H, F = 131_200, 64, 8192
    assert T * 2 * F > 2 ** 31
    x, wg, wu, wd, _ = R.case(T, H, F, seed=14)
    dy = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    tail = slice(T - 40, T)
    dy[tail] = R.case(40, H, 8, seed=15)[4]
    t = leaves((x, wg, wu, wd))
    y = cernels_b200.gated_ffn(*t)
    got = torch.autograd.grad(y, t, dy)
    want, bound, state = R.forward(x[tail], wg, wu, wd)
    R.assert_within("y", y.detach()[tail], want, bound)
    grads = R.backward(state, dy[tail])
    R.assert_within("dx", got[0][tail], *grads[0])
    assert not got[0][:T - 40].any()
    for g, (w, b) in zip(got[1:], grads[1:]):  # the other rows add products of zeros
        R.assert_within("dw", g, w, b)


@gpu
@pytest.mark.parametrize("T", [3, 70])
@pytest.mark.parametrize("need", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 0, 1), (0, 1, 1, 1)])
def test_partial_gradients_are_the_same(T, need):
    *args, dy = R.case(T, 192, 136, seed=4)
    t = leaves(args)
    full = torch.autograd.grad(cernels_b200.gated_ffn(*t), t, dy)
    t = [a.clone().requires_grad_(bool(n)) for a, n in zip(args, need)]
    part = torch.autograd.grad(cernels_b200.gated_ffn(*t), [a for a, n in zip(t, need) if n], dy)
    for g, f in zip(part, [f for f, n in zip(full, need) if n]):
        assert torch.equal(g, f)


@gpu
def test_repeats_bit_for_bit():
    *args, dy = R.case(700, 512, 264, seed=5)
    t = leaves(args)
    runs = [(cernels_b200.gated_ffn(*t), ) for _ in range(2)]
    grads = [torch.autograd.grad(y, t, dy) for y, in runs]
    assert torch.equal(runs[0][0], runs[1][0])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@gpu
@pytest.mark.parametrize("T", [1, 9, 40, 150])
def test_row_strides_and_views(T):
    """x as every other row of a wider buffer, weights as halves of a merged matrix."""
    H, F = 128, 72
    *args, dy = R.case(T, H, F, seed=6)
    wide = torch.full((2 * T, H + 24), 7.0, dtype=torch.bfloat16, device="cuda")
    x = wide[::2, 8:8 + H]
    x.copy_(args[0])
    merged = torch.cat((args[1], args[2]))
    t = [x.detach().requires_grad_(), merged[:F].requires_grad_(), merged[F:].requires_grad_(), args[3].requires_grad_()]
    y = cernels_b200.gated_ffn(*t)
    want, bound, state = R.forward(*args)
    R.assert_within("y", y.detach(), want, bound)
    with torch.no_grad():
        R.assert_within("y", cernels_b200.gated_ffn(*t), want, bound)
    for g, (w, b) in zip(torch.autograd.grad(y, t, dy), R.backward(state, dy)):
        R.assert_within("gradient", g, w, b)


@gpu
def test_broadcast_and_misaligned_output_gradients():
    *args, _ = R.case(20, 64, 40, seed=7)
    t = leaves(args)
    got = torch.autograd.grad(cernels_b200.gated_ffn(*t).sum(), t)  # an expanded gradient of ones
    ones = torch.ones(20, 64, dtype=torch.bfloat16, device="cuda")
    for g, (w, b) in zip(got, R.backward(R.forward(*args)[2], ones)):
        R.assert_within("gradient", g, w, b)
    odd = torch.ones(20 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(20, 64)
    again = torch.autograd.grad(cernels_b200.gated_ffn(*t), t, odd)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@gpu
def test_one_weight_for_both_halves():
    x, w, _, wd, dy = R.case(33, 64, 48, seed=8)
    x, w, wd = leaves((x, w, wd))
    got = torch.autograd.grad(cernels_b200.gated_ffn(x, w, w, wd), (x, w, wd), dy)
    (dx, ex), (dg, eg), (du, eu), (dd, ed) = R.backward(R.forward(x, w, w, wd)[2], dy)
    R.assert_within("dx", got[0], dx, ex)
    R.assert_within("dw", got[1], dg + du, eg + eu + R.HALF * ((dg + du).abs() + eg + eu))
    R.assert_within("dwd", got[2], dd, ed)


@gpu
def test_no_tokens():
    *args, dy = R.case(0, 64, 32)
    t = leaves(args)
    y = cernels_b200.gated_ffn(*t)
    assert y.shape == (0, 64)
    g = torch.autograd.grad(y, t, dy)
    assert g[0].shape == (0, 64) and all(not v.any() for v in g[1:])
    assert cernels_b200.gated_ffn(*args).shape == (0, 64)


@gpu
@pytest.mark.parametrize("T", [4, 200])
def test_saturated_and_special_values(T):
    """Gates far out on either side leave silu at 0 or at its argument; a token of infinities or NaN
    touches its own row only."""
    *args, _ = R.case(T, 64, 32, seed=9)
    args[0][0] *= 1000.0
    args[0][1] = 0.0
    want, bound, _ = R.forward(*args)
    R.assert_within("y", cernels_b200.gated_ffn(*args), want, bound)
    args[0][2] = float("inf")
    args[0][3] = float("nan")
    y = cernels_b200.gated_ffn(*args)
    keep = [i for i in range(T) if i not in (2, 3)]
    R.assert_within("y", y[keep], want[keep], bound[keep])
    assert y[3].isnan().all() and not torch.isfinite(y[2]).any()


@gpu
def test_refusals_on_cuda():
    x, wg, wu, wd, _ = R.case(4, 64, 32)
    call = cernels_b200.gated_ffn
    bad = [(x.float(), wg, wu, wd), (x, wg.half(), wu, wd), (x, wg[:, :32], wu, wd), (x, wg, wu[:16], wd),
           (x, wg, wu, wd.t()), (x, wg, wu, wd[:, :16]), (x[None], wg, wu, wd), (x, wg.cpu(), wu, wd),
           (x.expand(4, 64).t(), wg, wu, wd), (x[:1].expand(4, 64), wg, wu, wd),
           (x[:, :60].contiguous(), wg[:, :60].contiguous(), wu[:, :60].contiguous(), wd[:60])]
    for args in bad:
        with pytest.raises(RuntimeError):
            call(*args)
    odd = torch.zeros(4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 64)
    with pytest.raises(RuntimeError, match="aligned"):
        call(odd, wg, wu, wd)
    t = leaves((x, wg, wu, wd))
    with pytest.raises(RuntimeError):  # no second derivative
        g, = torch.autograd.grad(call(*t), t[:1], torch.ones_like(x), create_graph=True)
        torch.autograd.grad(g.sum(), t[1])


@gpu
def test_other_stream_and_first_call_of_a_thread():
    *args, dy = R.case(130, 64, 48, seed=10)
    want = cernels_b200.gated_ffn(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = cernels_b200.gated_ffn(*args)
    side.synchronize()
    assert torch.equal(y, want)
    got = []
    torch.cuda.synchronize()
    th = threading.Thread(target=lambda: got.append(cernels_b200.gated_ffn(*args)))
    th.start()
    th.join()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want)


@gpu
@pytest.mark.parametrize("T", [2, 150])
def test_two_graphs_replay_with_new_inputs(T):
    """A forward graph and a training graph, captured apart and replayed in turn on changed inputs."""
    a, b = R.case(T, 64, 48, seed=11), R.case(T, 64, 48, seed=12)
    fixed = [v.clone() for v in a]
    t = [v.requires_grad_() for v in fixed[:4]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.no_grad():
            cernels_b200.gated_ffn(*t)
        torch.autograd.grad(cernels_b200.gated_ffn(*t), t, fixed[4])
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1), torch.no_grad():
        y = cernels_b200.gated_ffn(*t)
    with torch.cuda.graph(g2):
        z = cernels_b200.gated_ffn(*t)
        grads = torch.autograd.grad(z, t, fixed[4])
    for values in (b, a, b):
        with torch.no_grad():
            for f, v in zip(fixed, values):
                f.copy_(v)
        g1.replay()
        g2.replay()
        want, bound, state = R.forward(*values[:4])
        R.assert_within("y", y, want, bound)
        R.assert_within("z", z.detach(), want, bound)
        for g, (w, e) in zip(grads, R.backward(state, values[4])):
            R.assert_within("gradient", g, w, e)


@gpu
def test_training_a_small_block():
    """A few optimiser steps through the operator run, with finite gradients of the weights' type."""
    x, *w, target = R.case(64, 64, 48, seed=13)
    params = [torch.nn.Parameter(v) for v in w]
    opt = torch.optim.SGD(params, lr=1e-3)
    for _ in range(3):
        opt.zero_grad()
        loss = ((cernels_b200.gated_ffn(x, *params).float() - target.float()) ** 2).mean()
        loss.backward()
        assert all(torch.isfinite(p.grad).all() and p.grad.dtype == torch.bfloat16 for p in params)
        opt.step()
