"""Cases of the feed-forward operators: the gated block with its gradient, and products with
4-bit weights (a linear layer and the routed experts' decode call).

``run`` computes them in plain torch (32-bit) or, with ``own``, through this package's entry
points; ``exact`` gives the same results in 64 bits.
"""

import math

import torch

own = False

LISTED = [
    # One token through a dense layer in serving: bound by the weights' bytes and by latency.
    {"name": "ffn_t1", "op": "ffn", "train": False, "T": 1, "H": 2048, "F": 1408},
    # A small batch of streams being decoded, wide layer.
    {"name": "ffn_t13", "op": "ffn", "train": False, "T": 13, "H": 2880, "F": 2880},
    # A short prompt, odd length.
    {"name": "ffn_t301", "op": "ffn", "train": False, "T": 301, "H": 2048, "F": 768},
    # A long prompt through a large dense layer.
    {"name": "ffn_t8192", "op": "ffn", "train": False, "T": 8192, "H": 4096, "F": 8192},
    # A training step on a short ragged batch through a small shared expert.
    {"name": "train_t509", "op": "ffn", "train": True, "T": 509, "H": 2048, "F": 512},
    # A training step of ordinary size.
    {"name": "train_t4096", "op": "ffn", "train": True, "T": 4096, "H": 2048, "F": 1408},
    # A training step on a large batch, sizes that no tile divides.
    {"name": "train_t8191", "op": "ffn", "train": True, "T": 8191, "H": 2880, "F": 2880},
    # The smallest 4-bit projection of one token: latency.
    {"name": "w4_t1", "op": "w4", "T": 1, "N": 2048, "K": 2048, "G": 32},
    # A wide 4-bit projection for a few streams.
    {"name": "w4_t7", "op": "w4", "T": 7, "N": 16384, "K": 8192, "G": 128},
    # One token through 4-bit experts.
    {"name": "moe_w4_t1", "op": "moe_w4", "T": 1, "H": 2048, "F": 1408, "E": 64, "k": 6, "G": 128, "masked": False},
    # Eight streams through wide 4-bit experts.
    {"name": "moe_w4_t8", "op": "moe_w4", "T": 8, "H": 2880, "F": 2880, "E": 32, "k": 4, "G": 32, "masked": False},
    # A padded batch: some tokens have no expert at all.
    {"name": "moe_w4_t29", "op": "moe_w4", "T": 29, "H": 2048, "F": 768, "E": 128, "k": 8, "G": 64, "masked": True},
]


def listed():
    return [dict(c) for c in LISTED]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "train", "train", "w4", "moe_w4"])
    if op in ("ffn", "train"):
        H, F = _log(rng, 128, 6144, 8), _log(rng, 128, 8192, 8)
        top = 8192 * 4096 * 8192 // (3 if op == "train" else 1)
        T = _log(rng, 1 if op == "ffn" else 16, max(32, min(16384, top // (H * F))))
        return {"op": "ffn", "train": op == "train", "T": T, "H": H, "F": F}
    G = rng.choice([32, 64, 128])
    if op == "w4":
        return {"op": "w4", "T": _log(rng, 1, 24), "N": _log(rng, 64, 16384), "K": _log(rng, 2 * G, 8192, G), "G": G}
    E, T = _log(rng, 4, 128), _log(rng, 1, 32)
    return {"op": "moe_w4", "T": T, "H": _log(rng, 512, 2880 // G * G, G), "F": _log(rng, 256, 2048, G), "E": E,
            "k": min(E, rng.randint(1, 8)), "G": G, "masked": T >= 8 and rng.random() < 0.7}


def _normal(gen, shape, std):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen).to(torch.bfloat16)


def _quantised(gen, shape, group):
    """Codes of 4 bits, two a byte (even position in the low half), and their groups' scales."""
    w = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, 0.02, generator=gen)
    w = w.view(*shape[:-1], shape[-1] // group, group)
    scale = (w.abs().amax(-1) / 7.0).to(torch.bfloat16)
    q = torch.clamp(torch.round(w / scale.float().unsqueeze(-1)) + 8.0, 0.0, 15.0).to(torch.uint8).view(*shape)
    return q[..., 0::2] | (q[..., 1::2] << 4), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T = case["T"]
    if case["op"] == "ffn":
        H, F = case["H"], case["F"]
        t = [_normal(gen, (T, H), 1.0), _normal(gen, (F, H), 0.02), _normal(gen, (F, H), 0.02),
             _normal(gen, (H, F), 0.02)]
        if not case["train"]:
            return {"case": case, "in": t}
        return {"case": case, "in": [v.requires_grad_() for v in t], "dy": _normal(gen, (T, H), 1.0)}
    if case["op"] == "w4":
        q, s = _quantised(gen, (case["N"], case["K"]), case["G"])
        return {"case": case, "in": [_normal(gen, (T, case["K"]), 1.0), q, s]}
    H, F, E, k, G = (case[n] for n in ("H", "F", "E", "k", "G"))
    q1, s1 = _quantised(gen, (E, 2 * F, H), G)
    q2, s2 = _quantised(gen, (E, H, F), G)
    logits = torch.empty((T, E), dtype=torch.float32, device="cuda").normal_(0.0, 1.0, generator=gen)
    weights, indices = torch.softmax(logits, -1).topk(k, -1)
    indices = indices.to(torch.int32)
    if case["masked"]:
        indices = torch.where(torch.rand((T, 1), device="cuda", generator=gen) < 0.3, -1, indices).to(torch.int32)
    return {"case": case, "in": [_normal(gen, (T, H), 1.0), q1, s1, q2, s2, indices.contiguous(), weights.contiguous()]}


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        if case["op"] == "ffn":
            return _plain_ffn(*state["in"], state.get("dy"))
        if case["op"] == "w4":
            x, q, s = state["in"]
            return torch.matmul(x.float(), _values(q, s).t()).to(x.dtype)
        return _plain_moe(*state["in"])


def _run_own(case, state):
    import cernels_b200

    if case["op"] == "ffn":
        y = cernels_b200.gated_ffn(*state["in"])
        return (y, *torch.autograd.grad(y, state["in"], state["dy"])) if case["train"] else (y,)
    if case["op"] == "w4":
        return cernels_b200.linear_w4(*state["in"])
    return cernels_b200.moe_experts_decode_w4(*state["in"], case["k"])


def _plain_ffn(x, wg, wu, wd, dy):
    kind = x.dtype
    x, wg, wu, wd = x.float(), wg.float(), wu.float(), wd.float()
    g, u = torch.matmul(x, wg.t()), torch.matmul(x, wu.t())
    s = 1.0 / (1.0 + torch.exp(-g))
    h = g * s * u
    y = torch.matmul(h, wd.t()).to(kind)
    if dy is None:
        return (y,)
    dy = dy.float()
    dh = torch.matmul(dy, wd)
    du = dh * g * s
    dg = dh * u * s * (1.0 + g * (1.0 - s))
    dx = torch.matmul(dg, wg) + torch.matmul(du, wu)
    return (y, dx.to(kind), torch.matmul(dg.t(), x).to(kind), torch.matmul(du.t(), x).to(kind),
            torch.matmul(dy.t(), h).to(kind))


def _values(q, s):
    """The numbers that packed codes and their groups' scales stand for, in 32 bits."""
    v = torch.stack((q & 15, q >> 4), -1).to(torch.float32) - 8.0
    v = v.reshape(*s.shape, -1) * s.float().unsqueeze(-1)
    return v.reshape(*q.shape[:-1], -1)


def _plain_moe(x, q1, s1, q2, s2, indices, weights):
    T, k = indices.shape
    E, F = q1.shape[0], q1.shape[1] // 2
    flat = indices.reshape(-1).long()
    live = (flat >= 0) & (flat < E)
    e = torch.where(live, flat, 0)
    rows = x.float().repeat_interleave(k, 0).unsqueeze(-1)
    gu = torch.matmul(_values(q1[e], s1[e]), rows).squeeze(-1)
    g, u = gu[:, :F], gu[:, F:]
    h = g / (1.0 + torch.exp(-g)) * u
    y = torch.matmul(_values(q2[e], s2[e]), h.unsqueeze(-1)).squeeze(-1)
    y = torch.where(live.unsqueeze(-1), y * weights.reshape(-1, 1), 0.0)
    return y.reshape(T, k, -1).sum(1).to(x.dtype)


def work(case):
    T = case["T"]
    if case["op"] == "ffn":
        H, F = case["H"], case["F"]
        matrices, rows = 3 * H * F, T * H
        if case["train"]:  # x, dy and the weights in; y, dx and the weights' gradients out
            return {"bytes": 2 * (4 * rows + 2 * matrices), "flops": 18 * T * H * F}
        return {"bytes": 2 * (2 * rows + matrices), "flops": 6 * T * H * F}
    G = case["G"]
    if case["op"] == "w4":
        N, K = case["N"], case["K"]
        return {"bytes": N * K // 2 + 2 * N * (K // G) + 2 * T * (K + N), "flops": 2 * T * N * K}
    H, F, E, k = (case[n] for n in ("H", "F", "E", "k"))
    live = T * (0.7 if case["masked"] else 1.0)
    touched = E * (1.0 - (1.0 - k / E) ** live)  # expected number of experts that any token chose
    return {"bytes": touched * 3 * H * F * (0.5 + 2.0 / G) + 4 * T * H + 8 * T * k, "flops": 6 * live * k * H * F}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "ffn":
            x, w1, w3, w2 = (v.detach().double() for v in state["in"])
            a, b = x @ w1.T, x @ w3.T
            act = a * torch.sigmoid(a)
            mid = act * b
            out = [mid @ w2.T]
            if case["train"]:
                up = state["dy"].double()
                back = up @ w2
                slope = torch.sigmoid(a) * (1.0 + a * torch.sigmoid(-a))
                da, db = back * b * slope, back * act
                out += [da @ w1 + db @ w3, da.T @ x, db.T @ x, up.T @ mid]
            return tuple(out)
        if case["op"] == "w4":
            x, q, s = state["in"]
            return x.double() @ _exact_values(q, s).T
        x, q1, s1, q2, s2, indices, weights = state["in"]
        E, F = q1.shape[0], q1.shape[1] // 2
        out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
        for e in range(E):
            token, slot = torch.nonzero(indices == e, as_tuple=True)
            if token.numel():
                both = x[token].double() @ _exact_values(q1[e], s1[e]).T
                mid = both[:, :F] * torch.sigmoid(both[:, :F]) * both[:, F:]
                part = mid @ _exact_values(q2[e], s2[e]).T * weights[token, slot].double().unsqueeze(-1)
                out.index_add_(0, token, part)
        return out


def _exact_values(q, s):
    group = q.shape[-1] * 2 // s.shape[-1]
    v = torch.empty(q.shape[0], q.shape[1] * 2, dtype=torch.float64, device=q.device)
    v[:, 0::2] = (q % 16).double() - 8.0
    v[:, 1::2] = torch.div(q, 16, rounding_mode="floor").double() - 8.0
    return v * s.double().repeat_interleave(group, 1)
