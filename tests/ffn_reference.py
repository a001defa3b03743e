"""The gated feed-forward block in 64 bits, with a bound for each output's error.

The bounds follow the operator's roundings, nothing measured: a bf16 rounding moves a value by at
most eps/2 = 2^-8 of it (the halved product and the gradients at it are rounded once as operands,
every output once), and a 32-bit sum of n products by at most n * 2^-23 of the sum of their
magnitudes (2^-23, not 2^-24: a tensor core may truncate). SIG is the relative error allowed to the
32-bit sigmoid: the exponential's and the division's few units of 2^-24, with its argument's
rounding |g| * 2^-24 for |g| up to 64 (beyond, the factor itself is below 1e-27).
"""

import torch

HALF = 2.0 ** -8
ADD = 2.0 ** -23
SIG = 2.0 ** -16
TINY = 1e-30  # results under the normal range


def _acc(a, b_t):
    """Bound of the 32-bit sum a @ b_t: terms * 2^-23 * sum of magnitudes."""
    return a.shape[1] * ADD * (a.abs() @ b_t.abs())


def forward(x, wg, wu, wd):
    """(y, bound of y's error, what the backward pass needs)."""
    x, wg, wu, wd = (t.detach().double() for t in (x, wg, wu, wd))
    g, u = x @ wg.T, x @ wu.T
    eg, eu = _acc(x, wg.T), _acc(x, wu.T)
    s = torch.sigmoid(g)
    a = g * s
    h = a * u
    # |silu'| <= 1.1
    eh = u.abs() * (1.1 * eg + SIG * a.abs()) + a.abs() * eu + 1.1 * eg * eu
    eh = eh + HALF * (h.abs() + eh)
    y = h @ wd.T
    ey = eh @ wd.abs().T + _acc(h.abs() + eh, wd.T)
    ey = ey + HALF * (y.abs() + ey) + TINY
    return y, ey, (x, wg, wu, wd, g, u, s, a, h, eg, eu, eh)


def backward(state, dy):
    """[(gradient, bound)] for x, gate_proj, up_proj, down_proj."""
    x, wg, wu, wd, g, u, s, a, h, eg, eu, eh = state
    dy = dy.detach().double()
    dh = dy @ wd
    edh = _acc(dy, wd)
    slope = s * (1.0 + g * (1.0 - s))
    # |silu''| <= 0.5; the 32-bit slope is off by SIG of its terms
    eslope = 0.5 * eg + SIG * (s + (g * s * (1.0 - s)).abs()) + SIG * a.abs()
    du = dh * a
    edu = edh * a.abs() + (dh.abs() + edh) * (1.1 * eg + SIG * a.abs())
    edu = edu + HALF * (du.abs() + edu)
    dg = dh * u * slope
    edg = (edh * (u * slope).abs() + (dh.abs() + edh) * (eu * slope.abs() + (u.abs() + eu) * eslope))
    edg = edg + HALF * (dg.abs() + edg)

    def out(v, e):
        return v, e + HALF * (v.abs() + e) + TINY

    dx = dg @ wg + du @ wu
    edx = edg @ wg.abs() + edu @ wu.abs() + _acc(torch.cat((dg.abs() + edg, du.abs() + edu), 1), torch.cat((wg, wu)))
    dwg, edwg = dg.T @ x, edg.T @ x.abs() + _acc((dg.abs() + edg).T, x)
    dwu, edwu = du.T @ x, edu.T @ x.abs() + _acc((du.abs() + edu).T, x)
    dwd, edwd = dy.T @ h, dy.abs().T @ eh + _acc(dy.T, h.abs() + eh)
    return [out(dx, edx), out(dwg, edwg), out(dwu, edwu), out(dwd, edwd)]


def case(T, H, F, seed=0, device="cuda", std=0.05):
    gen = torch.Generator(device=device).manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=device) * scale).to(torch.bfloat16)

    return rnd(T, H), rnd(F, H, scale=std), rnd(F, H, scale=std), rnd(H, F, scale=std), rnd(T, H)


def assert_within(name, got, want, bound):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"
