"""Products with 4-bit weights, against 64 bits (bounds: w4_reference)."""

import ctypes

import pytest
import torch

import cernels_b200
from cernels_b200 import _lib, w4
from tests import w4_reference as R
from tests.ffn_reference import assert_within

gpu = pytest.mark.gpu


def rows(T, K, seed, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(T, K, generator=gen, device=device).to(torch.bfloat16)


def routing(T, k, E, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w, i = torch.softmax(torch.randn(T, E, generator=gen, device="cuda"), -1).topk(min(k, E), -1)
    return i.to(torch.int32).contiguous(), w.contiguous()


def experts(E, H, F, G, seed):
    return (*R.codes((E, 2 * F, H), G, seed), *R.codes((E, H, F), G, seed + 1))


# ---------------------------------------------------------------- CPU
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_rounds_to_the_nearest_code(group):
    gen = torch.Generator().manual_seed(group)
    w = (torch.randn(3, 5, 384, generator=gen) * 0.02).to(torch.bfloat16)
    w[0, 1] = 0.0
    w[1, 2, :group] = 1.5
    q, s = cernels_b200.quantize_w4(w, group)
    assert q.shape == (3, 5, 192) and q.dtype == torch.uint8 and s.shape == (3, 5, 384 // group)
    v = R.values(q, s)
    step = s.double().repeat_interleave(group, -1)
    # half a step; the largest magnitude is 7 scales up to the scale's own rounding (7 * 2^-8 steps)
    assert ((v - w.double()).abs() <= step * (0.5 + 7 * R.HALF)).all()
    assert not v[0, 1].any()
    nearest = torch.round(w.double() / torch.where(step == 0, 1.0, step)).clamp(-8, 7)
    assert torch.equal(torch.where(step == 0, 0.0, v / torch.where(step == 0, 1.0, step)).round(),
                       torch.where(step == 0, 0.0, nearest))


def test_quantize_refusals():
    for w, g in ((torch.zeros(4, 96), 64), (torch.zeros(4, 128), 16), (torch.zeros(128), 32),
                 (torch.zeros(4, 128, dtype=torch.int32), 32), (torch.zeros(4, 0), 32)):
        with pytest.raises(RuntimeError):
            cernels_b200.quantize_w4(w, g)


def test_refuses_cpu_tensors_and_gradients():
    q, s = R.codes((8, 64), 32, 0, "cpu")
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        cernels_b200.linear_w4(torch.zeros(1, 64, dtype=torch.bfloat16), q, s)
    with pytest.raises(RuntimeError, match="no gradient"):
        cernels_b200.linear_w4(torch.zeros(1, 64, dtype=torch.bfloat16, requires_grad=True), q, s)


def test_meta_shapes():
    def m(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")

    o = torch.ops.cernels_b200
    assert o.linear_w4(m(3, 64), m(10, 32, dtype=torch.uint8), m(10, 2)).shape == (3, 10)
    y = o.moe_experts_decode_w4(m(3, 64), m(4, 64, 32, dtype=torch.uint8), m(4, 64, 2), m(4, 64, 16, dtype=torch.uint8),
                                m(4, 64, 1), m(3, 2, dtype=torch.int32), m(3, 2, dtype=torch.float32), 2)
    assert y.shape == (3, 64)


@pytest.mark.parametrize("args,code", [((-1, 8, 64, 32), 1), ((1, 0, 64, 32), 1), ((1, 8, 0, 32), 1), ((1, 8, 96, 64), 1),
                                       ((1, 8, 64, 16), 5), ((1, 8, 1 << 16, 32), 5)])
def test_c_linear_refuses_shapes(args, code):
    ok = 1 << 20
    assert _lib.load().cernels_linear_w4(*args, ok, args[2], ok, ok, ok, None) == code


def test_c_linear_refuses_pointers():
    call, ok = _lib.load().cernels_linear_w4, 1 << 20  # never read: refused before any launch
    assert call(1, 8, 64, 32, None, 64, ok, ok, ok, None) == 6
    assert call(1, 8, 64, 32, ok + 8, 64, ok, ok, ok, None) == 2
    assert call(1, 8, 64, 32, ok, 64, ok + 4, ok, ok, None) == 2
    assert call(1, 8, 64, 32, ok, 64, ok, ok + 1, ok, None) == 2
    assert call(1, 8, 64, 32, ok, 68, ok, ok, ok, None) == 2
    assert call(1, 8, 64, 32, ok, 32, ok, ok, ok, None) == 1
    assert call(0, 8, 64, 32, None, 64, None, None, None, None) == 0


@pytest.mark.parametrize("shape,group,code", [((1, 64, 4, 64, 2, 1), 32, 5), ((1, 64, 4096, 64, 2, 0), 32, 5),
                                              ((513, 64, 4, 64, 2, 0), 32, 5), ((1, 96, 4, 64, 2, 0), 64, 1),
                                              ((1, 64, 4, 64, 2, 0), 48, 5), ((1, 64, 0, 64, 2, 0), 32, 1)])
def test_c_experts_refuse_shapes(shape, group, code):
    s, n = _lib.MoeShape(*shape), ctypes.c_size_t(0)
    assert _lib.load().cernels_moe_w4_workspace_bytes(ctypes.byref(s), group, ctypes.byref(n)) == code


@pytest.mark.parametrize("sizes", [(2**32 + 1, 64, 4, 32, 2), (1, 64, 4, 2**32 + 32, 2), (1, 64, 2**32 + 4, 32, 2)])
def test_sizes_do_not_wrap(sizes):
    with pytest.raises(RuntimeError, match="2\\^31"):
        w4._moe_plan(*sizes, 32)


# ---------------------------------------------------------------- GPU: linear
@gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,N,groups", [(1, 1, 1), (1, 16, 4), (2, 17, 3), (3, 100, 9), (7, 250, 16), (8, 64, 33), (9, 33, 5),
                                        (16, 130, 8), (17, 40, 7), (33, 31, 2), (1, 5000, 8), (5, 9000, 3),
                                        # more tiles than a CTA takes at once, for each kernel by columns
                                        (1, 90000, 2), (4, 50001, 3), (7, 60000, 2), (13, 50000, 2), (20, 30000, 2)])
def test_linear(T, N, groups, group):
    K = groups * group
    x = rows(T, K, T + N)
    q, s = R.codes((N, K), group, groups)
    want, bound = R.linear(x, q, s)
    y = cernels_b200.linear_w4(x, q, s)
    assert y.shape == (T, N)
    assert_within("y", y, want, bound)
    assert torch.equal(y, torch.ops.cernels_b200.linear_w4(x, q, s))


@gpu
def test_linear_every_code_at_every_place():
    """x as unit rows reads single weights back: every code at every position of a group, exactly
    (a code times its scale has at most 12 bits; the scale here is a power of two, so bf16 holds it)."""
    for group in (32, 64, 128):
        K, N = 2 * group, 16
        q = torch.empty(N, K // 2, dtype=torch.uint8, device="cuda")
        for n in range(N):
            c = (torch.arange(K, device="cuda") * 7 + n) % 16
            q[n] = (c[0::2] | (c[1::2] << 4)).to(torch.uint8)
        s = torch.full((N, 2), 0.5, dtype=torch.bfloat16, device="cuda")
        s[:, 1] = -4.0
        x = torch.eye(K, dtype=torch.bfloat16, device="cuda")
        assert torch.equal(cernels_b200.linear_w4(x, q, s).double(), R.values(q, s).T)


@gpu
def test_linear_long_reduction_and_many_columns():
    """The longest rows (shared memory holds x one or a few columns at a time)."""
    for T, K, group in ((16, 16384, 128), (3, 32768, 32), (1, 32768, 64)):
        x = rows(T, K, T)
        q, s = R.codes((48, K), group, T)
        assert_within("y", cernels_b200.linear_w4(x, q, s), *R.linear(x, q, s))


@gpu
def test_linear_row_strides_empty_and_repeats():
    x = rows(5, 128, 0)
    q, s = R.codes((24, 128), 64, 1)
    wide = torch.full((10, 160), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[::2, 16:144] = x
    y = cernels_b200.linear_w4(x, q, s)
    assert torch.equal(y, cernels_b200.linear_w4(wide[::2, 16:144], q, s))
    assert torch.equal(y, cernels_b200.linear_w4(x, q, s))
    q3, s3 = R.codes((24, 128), 128, 2)  # one scale a row: the slice's start is 2 bytes off a word
    assert torch.equal(cernels_b200.linear_w4(x, q3[5:], s3[5:]), cernels_b200.linear_w4(x, q3, s3)[:, 5:])
    assert cernels_b200.linear_w4(x[:0], q, s).shape == (0, 24)
    assert cernels_b200.linear_w4(x, q[:0], s[:0]).shape == (5, 0)


@gpu
@pytest.mark.parametrize("T", [4, 12])
def test_linear_special_values_stay_in_their_row(T):
    x = rows(T, 64, 2)
    q, s = R.codes((40, 64), 32, 3)
    want, bound = R.linear(x, q, s)
    x[1], x[2, 5] = float("nan"), float("inf")
    s[7, 0] = float("inf")
    y = cernels_b200.linear_w4(x, q, s)
    keep_t = [t for t in range(T) if t not in (1, 2)]
    keep_n = [n for n in range(40) if n != 7]
    assert_within("y", y[keep_t][:, keep_n], want[keep_t][:, keep_n], bound[keep_t][:, keep_n])
    assert y[1].isnan().all() and not torch.isfinite(y[:, 7]).any()


@gpu
def test_linear_refusals():
    x = rows(4, 128, 0)
    q, s = R.codes((24, 128), 64, 1)
    bad = [(x.float(), q, s), (x, q.char(), s), (x, q, s.float()), (x, q[:, :32], s), (x, q, s[:, :1].expand(24, 3)),
           (x, q, s[:12]), (x[0], q, s), (x[:, :64], q, s), (x, q.cpu(), s), (x, q.t().contiguous().t(), s),
           (x[:1].expand(4, 128), q, s), (x, q, R.codes((24, 128), 16, 0)[1])]
    for args in bad:
        with pytest.raises(RuntimeError):
            cernels_b200.linear_w4(*args)
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.ops.cernels_b200.linear_w4(x.clone().requires_grad_(), q, s)


# ---------------------------------------------------------------- GPU: experts
@gpu
@pytest.mark.parametrize("T,H,E,F,k,group", [
    (1, 64, 4, 32, 2, 32), (1, 128, 1, 64, 1, 64), (2, 256, 8, 128, 3, 128), (5, 96, 3, 160, 3, 32), (8, 192, 16, 64, 4, 64),
    (9, 128, 2, 128, 1, 128), (16, 256, 64, 384, 6, 128), (29, 64, 7, 96, 2, 32), (64, 128, 300, 64, 8, 64),
    (40, 64, 2, 32, 2, 32), (1, 2048, 64, 1408, 6, 128), (12, 256, 6, 8192, 2, 64), (3, 8192, 4, 128, 2, 32),
    (40, 128, 3, 4096, 2, 128)])
def test_experts(T, H, E, F, k, group):
    x = rows(T, H, T + H)
    w = experts(E, H, F, group, T + E)
    idx, p = routing(T, k, E, T)
    k = idx.shape[1]
    y = cernels_b200.moe_experts_decode_w4(x, *w, idx, p, k)
    assert_within("y", y, *R.experts(x, *w, idx, p))
    assert torch.equal(y, torch.ops.cernels_b200.moe_experts_decode_w4(x, *w, idx, p, k))


@gpu
def test_experts_skipped_ids_repeated_ids_and_empty_tokens():
    T, H, E, F, k = 21, 128, 5, 64, 4
    x, w = rows(T, H, 1), experts(E, H, F, 32, 2)
    gen = torch.Generator(device="cuda").manual_seed(3)
    idx = torch.randint(-2, E + 2, (T, k), generator=gen, device="cuda").to(torch.int32)  # repeats among them
    idx[4] = -1
    idx[5] = E
    idx[6] = 2
    idx[7] = torch.tensor([2 ** 31 - 1, -2 ** 31, 1, 1], device="cuda")
    p = torch.rand(T, k, generator=gen, device="cuda") - 0.3
    p[idx < 0] = float("nan")  # the weight of a skipped slot is not used
    y = cernels_b200.moe_experts_decode_w4(x, *w, idx, p, k)
    assert_within("y", y, *R.experts(x, *w, idx, p))
    assert not y[4].any() and not y[5].any()
    none = torch.full_like(idx, -1)
    assert not cernels_b200.moe_experts_decode_w4(x, *w, none, p, k).any()


@gpu
def test_experts_most_pairs_and_repeats_bit_for_bit():
    T, H, E, F, k = 128, 64, 2048, 32, 8
    x, w = rows(T, H, 4), experts(E, H, F, 32, 5)
    idx, p = routing(T, k, E, 6)
    a = cernels_b200.moe_experts_decode_w4(x, *w, idx, p, k)
    assert torch.equal(a, cernels_b200.moe_experts_decode_w4(x, *w, idx, p, k))
    some = [0, 1, 63, 64, 127]
    assert_within("y", a[some], *R.experts(x[some], *w, idx[some], p[some]))
    one = torch.zeros_like(idx)  # every pair on one expert
    y = cernels_b200.moe_experts_decode_w4(x, *w, one, p, k)
    assert_within("y", y[some], *R.experts(x[some], *w, one[some], p[some]))


@gpu
def test_experts_wide_rows():
    """Rows so long that an item holds fewer than 8 columns of x."""
    T, H, E, F, k = 6, 32768, 2, 64, 2
    x, w = rows(T, H, 7), experts(E, H, F, 64, 8)
    idx, p = routing(T, k, E, 9)
    assert_within("y", cernels_b200.moe_experts_decode_w4(x, *w, idx, p, k), *R.experts(x, *w, idx, p))
    T, H, E, F, k = 7, 64, 2, 16384, 1
    x, w = rows(T, H, 7), experts(E, H, F, 64, 8)
    idx, p = routing(T, k, E, 9)
    assert_within("y", cernels_b200.moe_experts_decode_w4(x, *w, idx, p, k), *R.experts(x, *w, idx, p))


@gpu
def test_experts_beyond_32_bit_offsets():
    """The last of so many experts that its codes start 2^31 bytes and more into the tensor."""
    T, H, E, F = 2, 4096, 70, 8192
    assert (E - 1) * 2 * F * (H // 2) > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(0)
    q1 = torch.zeros(E, 2 * F, H // 2, dtype=torch.uint8, device="cuda")
    q2 = torch.zeros(E, H, F // 2, dtype=torch.uint8, device="cuda")
    s1 = torch.zeros(E, 2 * F, H // 128, dtype=torch.bfloat16, device="cuda")
    s2 = torch.zeros(E, H, F // 128, dtype=torch.bfloat16, device="cuda")
    last = experts(1, H, F, 128, 3)
    for t, v in zip((q1, s1, q2, s2), last):
        t[E - 1] = v[0]
    x = rows(T, H, 4)
    idx = torch.full((T, 1), E - 1, dtype=torch.int32, device="cuda")
    p = torch.rand(T, 1, generator=gen, device="cuda")
    want, bound = R.experts(x, *last, torch.zeros_like(idx), p)
    assert_within("y", cernels_b200.moe_experts_decode_w4(x, q1, s1, q2, s2, idx, p, 1), want, bound)


@gpu
def test_experts_refusals():
    x, w = rows(4, 64, 0), experts(4, 64, 32, 32, 1)
    idx, p = routing(4, 2, 4, 2)
    call = cernels_b200.moe_experts_decode_w4
    other = R.codes((4, 64, 64), 64, 0)
    bad = [(x.float(), *w, idx, p, 2), (x, *w, idx.long(), p, 2), (x, *w, idx, p.half(), 2), (x, *w, idx, p, 3),
           (x, *w[:2], *w[:2], idx, p, 2), (x[:, :32], *w, idx, p, 2), (x, *w, idx[:2], p, 2), (x, w[0], w[1], *other, idx, p, 2),
           (x, w[0][:, :31], w[1][:, :31], *w[2:], idx, p, 2), (torch.cat([x] * 129), *w, torch.cat([idx] * 129), torch.cat([p] * 129), 2)]
    for args in bad:
        with pytest.raises(RuntimeError):
            call(*args)
    with pytest.raises(RuntimeError, match="no gradient"):
        call(x, *w, idx, p.clone().requires_grad_(), 2)
    assert call(x[:0], *w, idx[:0], p[:0], 2).shape == (0, 64)


@gpu
def test_other_stream_and_two_graphs():
    x, w = rows(3, 128, 0), experts(6, 128, 64, 64, 1)
    idx, p = routing(3, 2, 6, 2)
    q, s = R.codes((72, 128), 64, 3)
    want = cernels_b200.moe_experts_decode_w4(x, *w, idx, p, 2), cernels_b200.linear_w4(x, q, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cernels_b200.moe_experts_decode_w4(x, *w, idx, p, 2), cernels_b200.linear_w4(x, q, s)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = cernels_b200.moe_experts_decode_w4(x, *w, idx, p, 2)
    with torch.cuda.graph(g2):
        y2 = cernels_b200.moe_experts_decode_w4(x, *w, idx, p, 2)
        z = cernels_b200.linear_w4(y2, q, s)
    for seed in (4, 5):
        x.copy_(rows(3, 128, seed))
        i, v = routing(3, 2, 6, seed)
        idx.copy_(i)
        p.copy_(v)
        g1.replay()
        g2.replay()
        assert_within("y", y1, *R.experts(x, *w, idx, p))
        assert torch.equal(y1, y2)
        assert_within("z", z, *R.linear(y2, q, s))


@gpu
def test_decode_in_4_bits_follows_the_bf16_experts():
    """Quantised experts against the bf16 decode operator on the very values they stand for: both are
    within their own bounds of the same 64-bit result (the bf16 one rounds the values once more)."""
    T, H, E, F, k = 4, 256, 8, 128, 2
    gen = torch.Generator(device="cuda").manual_seed(0)
    w1 = (torch.randn(E, 2 * F, H, generator=gen, device="cuda") * 0.05).to(torch.bfloat16)
    w2 = (torch.randn(E, H, F, generator=gen, device="cuda") * 0.05).to(torch.bfloat16)
    q = (*cernels_b200.quantize_w4(w1, 64), *cernels_b200.quantize_w4(w2, 64))
    x = rows(T, H, 1)
    idx, p = routing(T, k, E, 2)
    got = cernels_b200.moe_experts_decode_w4(x, *q, idx, p, k)
    near = cernels_b200.cohere2_moe_experts_decode(x, R.values(q[0], q[1]).to(torch.bfloat16).contiguous(),
                                                   R.values(q[2], q[3]).to(torch.bfloat16).contiguous(), idx, p, k)
    want, bound = R.experts(x, *q, idx, p)
    assert_within("y", got, want, bound)
    assert ((near.double() - want).norm() / want.norm()) < 4 * R.HALF
