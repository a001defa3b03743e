"""4-bit products of x whose values differ widely within a block of 128: a few large ones, which an output
may not see because its codes are 0 (8 as stored) there, must not cost the others their bits.

Blocks in which more than half of the nonzero values are under 2^-7 of the largest are multiplied exactly; for rows of
x that have no other blocks the bound below holds: products are exact, a group's sum has at most G 32-bit
roundings, its scale and its way into the row's sum one each a group, and at most 16 warps' sums are added.
"""

import pytest
import torch

import cernels_b200
from tests import w4_reference as R
from tests.ffn_reference import ADD, assert_within

pytestmark = pytest.mark.gpu


def exact_bound(x, q, s):
    group = q.shape[1] * 2 // s.shape[1]
    return (group + s.shape[1] + 16) * ADD * (x @ R.values(q, s).abs().T)


def spread(T, K, large, size, seed, every=1):
    """x of rows 0.05 times normal values with `large` values of +-size in each block of 128, in the same places in every
    `every`-th row, and those places [K] as truth values."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, K, generator=gen, device="cuda") * 0.05
    place = torch.zeros(K, dtype=torch.bool, device="cuda")
    for b in range(0, K, 128):
        n = min(128, K - b)
        place[b + torch.randperm(n, generator=gen, device="cuda")[:max(1, large * n // 128)]] = True
    sign = torch.randint(0, 2, (T, K), generator=gen, device="cuda") * 2.0 - 1.0
    rows = (torch.arange(T, device="cuda") % every == 0).unsqueeze(1)
    return torch.where(place & rows, sign * size, x).to(torch.bfloat16), place


def hide(q, place, rows):
    """The codes q [.., N, K / 2] with value 0 at `place` in the given rows."""
    q = q.clone()
    part = q[..., rows, :]
    low = torch.where(place[0::2], 8, part & 15)
    high = torch.where(place[1::2], 8, part >> 4)
    q[..., rows, :] = (low | high << 4).to(torch.uint8)
    return q


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("large,size", [(1, 100.0), (1, 3000.0), (5, 1000.0), (40, 1e6), (60, 100.0), (1, 1e38)])
@pytest.mark.parametrize("T,N,groups", [(1, 100, 8), (3, 33, 13), (4, 5000, 4), (7, 250, 16), (8, 17, 33), (16, 130, 8), (29, 40, 7)])
def test_linear(T, N, groups, large, size, group, monkeypatch):
    K = groups * group
    x, place = spread(T, K, large, size, seed=T + N)
    q, s = R.codes((N, K), group, groups)
    q = hide(q, place, slice(0, N - N // 4))  # the other outputs see the large values
    monkeypatch.setattr(R, "_sum_bound", exact_bound)
    if size == 1e38:  # their sums may pass the range
        q = hide(q, place, slice(0, N))
    want, bound = R.linear(x, q, s)
    y = cernels_b200.linear_w4(x, q, s)
    assert_within("y", y, want, bound)
    assert torch.equal(y, cernels_b200.linear_w4(x, q, s))


@pytest.mark.parametrize("T", [2, 4, 7, 16, 20])
def test_ordinary_rows_beside_mixed_ones(T, monkeypatch):
    """Rows share tiles; an ordinary row's result does not depend on its neighbours."""
    x, place = spread(T, 640, 3, 500.0, seed=T, every=3)
    q, s = R.codes((90, 640), 64, 1)
    q = hide(q, place, slice(0, 90))
    y = cernels_b200.linear_w4(x, q, s)
    plain = [t for t in range(T) if t % 3]
    assert_within("ordinary", y[plain], *(v[plain] for v in R.linear(x, q, s)))
    z = x.clone()
    z[::3] = x[1 if T > 1 else 0]
    assert torch.equal(y[plain], cernels_b200.linear_w4(z, q, s)[plain])
    monkeypatch.setattr(R, "_sum_bound", exact_bound)
    assert_within("mixed", y[::3], *(v[::3] for v in R.linear(x, q, s)))


def test_blocks_of_mostly_zeros_and_of_different_kinds():
    """Zeros do not count; a row may have both kinds of blocks, empty ones and a last one cut off."""
    x, place = spread(5, 32 * 21, 2, 300.0, seed=3)
    x[1, 128:256] = 0.0
    x[2, :128] = torch.randn(128, device="cuda")
    x[3] = torch.where(torch.arange(672, device="cuda") % 9 == 0, x[3], 0.0)
    x[4] = 0.0
    q, s = R.codes((70, 672), 32, 4)
    q = hide(q, place, slice(0, 70))
    y = cernels_b200.linear_w4(x, q, s)
    assert_within("y", y, *R.linear(x, q, s))
    assert not y[4].any()


@pytest.mark.parametrize("T", [1, 4, 7, 16])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_infinities_and_nan_follow_the_definition(T, value):
    x = torch.randn(T, 256, device="cuda").to(torch.bfloat16)
    x[T // 2, 131] = value
    q, s = R.codes((600, 256), 64, 5)
    y = cernels_b200.linear_w4(x, q, s)
    want, bound = R.linear(x, q, s)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf())
    assert torch.equal(y.double()[y.isinf()], want[want.isinf()])
    keep = [t for t in range(T) if t != T // 2]
    assert_within("y", y[keep], want[keep], bound[keep])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,k,E", [(1, 2, 4), (6, 2, 5), (24, 3, 4)])
def test_experts(T, k, E, group, monkeypatch):
    """Both products of the experts: x with large values that no code sees, and gates and ups that make large
    values of the down product's x, seen by a quarter of its outputs."""
    H, F = 384, 256
    x, place = spread(T, H, 2, 400.0, seed=T)
    q1, s1 = R.codes((E, 2 * F, H), group, 1)
    q2, s2 = R.codes((E, H, F), group, 2)
    q1 = hide(q1, place, slice(0, 2 * F))
    big = torch.zeros(F, dtype=torch.bool, device="cuda")
    big[[5, 77, 130, 255]] = True
    s1 = torch.where(torch.cat((big, big))[:, None], s1.sign() * 8.0, s1.clamp(-0.02, 0.02)).to(torch.bfloat16)
    q1[:, :F][:, big] = q1[:, F:][:, big]  # gate = up there: large and positive or small
    s1[:, :F][:, big] = s1[:, F:][:, big]
    q2 = hide(q2, big, slice(0, H - H // 4))
    gen = torch.Generator(device="cuda").manual_seed(3)
    idx = torch.randint(0, E, (T, k), generator=gen, device="cuda").to(torch.int32)
    p = torch.rand(T, k, generator=gen, device="cuda")
    y = cernels_b200.moe_experts_decode_w4(x, q1, s1, q2, s2, idx, p, k)
    assert_within("y", y, *R.experts(x, q1, s1, q2, s2, idx, p))
    assert torch.equal(y, cernels_b200.moe_experts_decode_w4(x, q1, s1, q2, s2, idx, p, k))
    # the gate and up products alone, through a down product that reads single values back
    q3 = torch.full((E, H, F // 2), 0x88, dtype=torch.uint8, device="cuda")
    s3 = torch.ones(E, H, F // group, dtype=torch.bfloat16, device="cuda")
    for f in range(F):
        q3[:, f, f // 2] = 0x98 if f % 2 else 0x89
    monkeypatch.setattr(R, "_sum_bound", exact_bound)
    one = torch.ones_like(p[:, :1])
    z = cernels_b200.moe_experts_decode_w4(x, q1, s1, q3, s3, idx[:, :1].contiguous(), one, 1)
    want, bound = R.experts(x, q1, s1, q3, s3, idx[:, :1], one)
    # values under 2^-14 of the largest of a block that is not mixed may be rounded: the reader sees each alone
    lost = 2.0 ** -14 * torch.nn.functional.pad(want[:, :F].abs().unflatten(1, (-1, 128)).amax(-1).repeat_interleave(128, 1), (0, H - F))
    assert_within("h", z, want, bound + (1 + 2.0 ** -7) * lost)
