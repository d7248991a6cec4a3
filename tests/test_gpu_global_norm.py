"""Global norm and clipping by it against 64-bit sums.

Bounds: the sum of squares is held in double (half data: groups of eight squares in float, 8 u), so the norm is off by
its one rounding (and 4 u for half); a clipped value by the rounding of the factor, of the product and of the result."""
import pytest
import torch

from tests.lm_cases import KIND, NAMES, STORE, TINY, TYPES, U, WIDE, randn, within

pytestmark = pytest.mark.gpu


def truth(x):
    return sum((t.double() ** 2).sum() for t in x).sqrt() if x else torch.zeros((), device="cuda", dtype=torch.float64)


def norm_bound(dt, norm, count=1):
    if dt == 1:
        # Here the sums themselves are held in the type of the result, on both sides. A sum of squares (all of one sign) is
        # off by at most its longest chain of additions times u, relative, and its root by half of that. The kernel's
        # chain: 8 values per thread and chunk, at most 16 chunks here, 5 + 16 steps of the CTA and 2 + 5 + 16 of the
        # fold, below 180; the other side adds `count` tensors one by one, each summed in a tree, below count + 60.
        return norm * (0.5 * (240 + count) + 2) * U[dt]
    return norm * (6 * U[dt] if dt == 2 else 2 * U[dt])


def tensors(dt, lengths, seed=1, scale=1.0):
    return [(scale * randn(seed + i, n)).to(KIND[dt]) for i, n in enumerate(lengths)]


LISTS = [[], [1], [0], [7], [4096], [0, 5, 0, 3], [1, 2, 3, 4, 5, 6, 7, 8, 9], [100003], [8192, 1, 8192, 30000], [64] * 300, [5] * 700,
         [16384 * 3 + 1, 2047, 16384]]


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("lengths", LISTS, ids=lambda l: "%d_%d" % (len(l), sum(l)))
def test_norm_and_clip(ops, dt, lengths):
    x = tensors(dt, lengths)
    norm = torch.full((1,), 9, dtype=WIDE[dt], device="cuda")
    want = truth(x)
    ops.execGlobalNorm(dt, None, x, lengths, len(x), norm)
    within(norm[0], want, norm_bound(dt, want, len(x)))
    for most in (0.25 * float(want), 4 * float(want) + 1, 0.0):
        z = [torch.full_like(t, 3) for t in x]
        norm.fill_(9)
        ops.execClipByGlobalNorm(dt, None, x, z, lengths, len(x), most, norm)
        within(norm[0], want, norm_bound(dt, want, len(x)))
        factor = min(1.0, most / float(want)) if float(want) > 0 else 1.0
        for a, b in zip(x, z):
            if factor == 1.0:
                assert torch.equal(a, b)
            else:
                e = a.double() * factor
                within(b, e, e.abs() * (10 * U[dt] + STORE[dt]) + TINY[dt])
        keep = [t.clone() for t in x]
        ops.execClipByGlobalNorm(dt, None, keep, None, lengths, len(x), most, norm)
        assert all(torch.equal(a, b) for a, b in zip(keep, z))


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("xs,zs", [(0, 0), (1, 1), (1, 0), (3, 1), (2, 3)])
def test_unaligned_tensors(ops, dt, xs, zs):
    n = 20011
    xb, zb = randn(1, n + 8, dtype=KIND[dt]), torch.full((n + 8,), 3, dtype=KIND[dt], device="cuda")
    x, z = xb[xs:xs + n], zb[zs:zs + n]
    norm = torch.empty(1, dtype=WIDE[dt], device="cuda")
    want = truth([x])
    ops.execClipByGlobalNorm(dt, None, [x], [z], [n], 1, 0.5 * float(want), norm)
    within(norm[0], want, norm_bound(dt, want))
    e = x.double() * 0.5
    within(z, e, e.abs() * (10 * U[dt] + STORE[dt]) + TINY[dt])
    assert (zb[:zs] == 3).all() and (zb[zs + n:] == 3).all()


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
def test_norms_that_are_not_finite_scale_nothing(ops, dt):
    for value in (float("nan"), float("inf"), float("-inf")):
        x = tensors(dt, [1000, 50])
        x[1][20] = value
        z = [torch.zeros_like(t) for t in x]
        norm = torch.empty(1, dtype=WIDE[dt], device="cuda")
        ops.execClipByGlobalNorm(dt, None, x, z, [1000, 50], 2, 1e-3, norm)
        assert not norm.isfinite().any()
        assert all(torch.equal(a.nan_to_num(5), b.nan_to_num(5)) for a, b in zip(x, z))


def test_squares_beyond_the_range_of_a_float(ops):
    for size in (1e25, 1e-25):
        x = tensors(0, [5000, 3], scale=size)
        norm = torch.empty(1, device="cuda")
        want = truth(x)
        ops.execGlobalNorm(0, None, x, [5000, 3], 2, norm)
        within(norm[0], want, norm_bound(0, want))


def test_the_same_tensor_twice_counts_twice(ops):
    x = randn(1, 1000).float()
    norm = torch.empty(1, device="cuda")
    ops.execGlobalNorm(0, None, [x, x], [1000, 1000], 2, norm)
    want = truth([x, x])
    within(norm[0], want, norm_bound(0, want))


def test_many_values_are_summed_the_same_way_each_time(ops):
    x = tensors(0, [3000001, 5, 4000000])
    norms = [torch.empty(1, device="cuda") for _ in range(4)]
    for n in norms:
        ops.execGlobalNorm(0, None, x, [3000001, 5, 4000000], 3, n)
    assert all(torch.equal(n, norms[0]) for n in norms)
    want = truth(x)
    within(norms[0][0], want, norm_bound(0, want))


@pytest.mark.parametrize("dt,size,most", [(0, 1e34, 1e-6), (0, 1e35, 1e-25), (0, 1e30, 1e-30), (1, 1e150, 1e-170), (1, 1e140, 1e-150)])
@pytest.mark.parametrize("lengths", [[900, 31], [200003, 17]])
def test_factors_below_the_range_of_the_type(ops, dt, size, most, lengths):
    # the factor maxNorm / norm has no (normal) value in the type; the products with the large values that need it do
    x = tensors(dt, lengths, scale=size)
    for t in x:
        t[::3] *= 1e-3
    norm = torch.empty(1, dtype=WIDE[dt], device="cuda")
    want = truth(x)
    z = [torch.full_like(t, 3) for t in x]
    ops.execClipByGlobalNorm(dt, None, x, z, lengths, 2, most, norm)
    within(norm[0], want, norm_bound(dt, want, 2))
    for a, b in zip(x, z):
        e = a.double() / want * most
        slack = 0.5 * (240 + 2) + 2 if dt == 1 else 0           # of the norm itself, which is held in the type
        within(b, e, e.abs() * ((10 + slack) * U[dt] + STORE[dt]) + TINY[dt])
