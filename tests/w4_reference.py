"""4-bit products in 64 bits, with bounds of their errors (the constants of ffn_reference).

Codes and scales are exact in 64 bits and never rounded by the operator. It takes x as 14 bits and a
sign below the largest value of each block of 128, rounding it by at most 2^-14 of that value; sums
within a group are exact integers, and each group's sum then meets seven 32-bit roundings on its way
into its block's and the row's sum (conversion, two for its parts, scale, unit, two additions), which add up with
the number of groups. The experts' call adds the rounding of the halved product, as an operand.
"""

import torch

from tests.ffn_reference import ADD, HALF, SIG, TINY


def codes(shape, group, seed, device="cuda"):
    """Random codes over the whole range and scales of both signs, tiny to large."""
    gen = torch.Generator(device=device).manual_seed(seed)
    q = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), generator=gen, device=device, dtype=torch.uint8)
    s = torch.randn(*shape[:-1], shape[-1] // group, generator=gen, device=device) * 0.01
    return q, s.to(torch.bfloat16)


def values(q, s):
    low, high = (q & 15).double() - 8.0, (q >> 4).double() - 8.0
    v = torch.stack((low, high), -1).flatten(-2)
    return v * s.double().repeat_interleave(v.shape[-1] // s.shape[-1], -1)


def _sum_bound(x, q, s):
    """Bound of the operator's sums of |x| [T, K] with the weights of (q, s) [N, ..]."""
    w = values(q, s).abs()
    pad = -x.shape[1] % 128
    xb, wb = (torch.nn.functional.pad(v, (0, pad)).unflatten(1, (-1, 128)) for v in (x, w))
    rounded = 2.0 ** -14 * (xb.amax(-1) @ wb.sum(-1).T)
    return rounded + (s.shape[-1] + 7) * ADD * (x @ w.T + rounded)


def linear(x, q, s):
    x, w = x.double(), values(q, s)
    y = x @ w.T
    e = _sum_bound(x.abs(), q, s)
    return y, e + HALF * (y.abs() + e) + TINY


def experts(x, q1, s1, q2, s2, indices, weights):
    E, F = q1.shape[0], q1.shape[1] // 2
    x = x.double()
    y = torch.zeros_like(x)
    bound = torch.zeros_like(x)
    mag = torch.zeros_like(x)
    for t in range(indices.shape[0]):
        for j in range(indices.shape[1]):
            e = int(indices[t, j])
            if not 0 <= e < E:
                continue
            w1, w2, p = values(q1[e], s1[e]), values(q2[e], s2[e]), float(weights[t, j])
            gu, egu = w1 @ x[t], _sum_bound(x[t:t + 1].abs(), q1[e], s1[e])[0]
            g, u, eg, eu = gu[:F], gu[F:], egu[:F], egu[F:]
            a = g * torch.sigmoid(g)
            h = a * u
            eh = u.abs() * (1.1 * eg + SIG * a.abs()) + a.abs() * eu + 1.1 * eg * eu
            eh = eh + HALF * (h.abs() + eh)
            r = w2 @ h
            er = w2.abs() @ eh + _sum_bound((h.abs() + eh)[None], q2[e], s2[e])[0]
            y[t] += p * r
            bound[t] += abs(p) * er
            mag[t] += abs(p) * (r.abs() + er)
    bound = bound + (indices.shape[1] + 1) * ADD * mag
    return y, bound + HALF * (y.abs() + bound) + TINY
