"""Layer norm and its gradients against the formulas in 64 bits.

Bounds: u is the unit roundoff of the type that sums are held in. A sum that no thread takes more than D terms of (and
that is folded in fewer than D steps after) is off by at most D u times the sum of the magnitudes. Forward, the mean is
off by D u mean|x|, so h by that times invStd plus (D + 4) u |h|; every result adds one rounding to the stored type."""
import pytest
import torch

from tests.lm_cases import KIND, LAYOUTS, NAMES, STORE, TINY, TYPES, U, WIDE, between, info, place, randn, within

pytestmark = pytest.mark.gpu
D = 160          # at most 32 values per thread and 32 + 5 steps of folding; the sweeping kernels: 512 threads, 40000 values


def forward_truth(x, gain, bias, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    inv = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    h = (x - mean) * inv
    z = h if gain is None else h * gain.double()
    return (z if bias is None else z + bias.double()), mean[:, 0], inv[:, 0], h


def check_forward(dt, x, gain, bias, eps, z, mean, inv):
    want, m, i, h = forward_truth(x, gain, bias, eps)
    u = U[dt]
    size = x.double().abs()
    em = D * u * size.mean(1) + u * m.abs()
    eh = i[:, None] * (em[:, None] + u * (size + m.abs()[:, None])) + (D + 4) * u * h.abs()
    g = 1.0 if gain is None else gain.double().abs()
    within(z, want, eh * g + 2 * u * (h.abs() * g + want.abs()) + STORE[dt] * want.abs() + TINY[dt])
    if mean is not None:
        within(mean, m, em)
        # the variance moves by the square of the mean's error, and by the roundings of x - mean
        within(inv, i, i * ((D + 4) * u + 2 * u * i * size.max(1).values + (i * em) ** 2))


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 4096), (5, 31), (7, 64), (33, 257), (130, 1000), (9, 1024), (9, 1025),
                                       (4, 2047), (3, 4096), (2, 8191), (2, 16384), (2, 20001), (2, 33000), (1, 40000), (2500, 16)])
def test_forward(ops, dt, rows, cols):
    x = (randn(cols, rows, cols) * 1.5 + randn(cols + 1, rows, 1)).to(KIND[dt])
    gain, bias = (1 + 0.3 * randn(2, cols)).to(KIND[dt]), (0.2 * randn(3, cols)).to(KIND[dt])
    z = torch.full_like(x, 5)
    mean, inv = torch.empty(rows, dtype=WIDE[dt], device="cuda"), torch.empty(rows, dtype=WIDE[dt], device="cuda")
    ops.execLayerNorm(dt, None, x, info(x), gain, bias, 1e-5, z, info(z), mean, inv, [1], 1)
    check_forward(dt, x, gain, bias, 1e-5, z, mean, inv)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("xl", LAYOUTS)
@pytest.mark.parametrize("zl", ["dense", "apart", "every second"])
@pytest.mark.parametrize("rows,cols", [(6, 96), (3, 1500)])
def test_forward_layouts(ops, dt, xl, zl, rows, cols):
    x = place(randn(5, rows, cols, dtype=KIND[dt]), xl)
    z = place(torch.full((rows, cols), 5.0, dtype=KIND[dt], device="cuda"), zl)
    ops.execLayerNorm(dt, None, x, info(x), None, None, 1e-3, z, info(z), None, None, [1], 1)
    check_forward(dt, x, None, None, 1e-3, z, None, None)
    assert between(z) or zl == "dense"


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape,dims", [((4, 5, 6), [2]), ((4, 5, 6), [1, 2]), ((4, 5, 6), [0]), ((4, 5, 6), [0, 2]), ((4, 5, 6), [0, 1, 2]),
                                        ((1, 9), [1]), ((7, 1), [1])])
def test_dimension_lists(ops, dt, shape, dims):
    x = randn(11, *shape, dtype=KIND[dt])
    keep = [ax for ax in range(len(shape)) if ax not in dims]
    order = keep + dims
    rows = 1
    for ax in keep:
        rows *= shape[ax]
    flat = x.permute(order).reshape(rows, -1)
    gain, bias = randn(12, flat.shape[1], dtype=KIND[dt]), randn(13, flat.shape[1], dtype=KIND[dt])
    z = torch.empty_like(x)
    mean, inv = torch.empty(rows, dtype=WIDE[dt], device="cuda"), torch.empty(rows, dtype=WIDE[dt], device="cuda")
    ops.execLayerNorm(dt, None, x, info(x), gain, bias, 1e-2, z, info(z), mean, inv, dims, len(dims))
    check_forward(dt, flat, gain, bias, 1e-2, z.permute(order).reshape(rows, -1), mean, inv)


def test_values_far_from_zero_keep_their_variance(ops):
    # mean 1000, deviation 1: sum(x^2) - n mean^2 would lose the variance in float
    x = (1000 + randn(1, 8, 3000)).float()
    z = torch.empty_like(x)
    ops.execLayerNorm(0, None, x, info(x), None, None, 1e-5, z, info(z), None, None, [1], 1)
    check_forward(0, x, None, None, 1e-5, z, None, None)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
def test_in_place_and_special_values(ops, dt):
    x = randn(3, 12, 700, dtype=KIND[dt])
    x[3] = 2.5                                       # no variance at all
    x[5, 17], x[7, 20], x[9] = float("nan"), float("inf"), 0
    want = forward_truth(x, None, None, 1e-5)[0]
    z = x.clone()
    ops.execLayerNorm(dt, None, z, info(z), None, None, 1e-5, z, info(z), None, None, [1], 1)
    ok = [r for r in range(12) if r not in (5, 7)]
    check_forward(dt, x[ok], None, None, 1e-5, z[ok], None, None)
    assert z[5].isnan().all() and z[7].isnan().all() and want[5].isnan().all()
    assert (z[9] == 0).all()


def backward_truth(x, gain, mean, inv, dz):
    x, dz, mean, inv = x.double(), dz.double(), mean.double()[:, None], inv.double()[:, None]
    h = (x - mean) * inv
    d = dz if gain is None else dz * gain.double()
    n = x.shape[1]
    a, b = d.sum(1, keepdim=True) / n, (d * h).sum(1, keepdim=True) / n
    return inv * (d - a - h * b), (dz * h).sum(0), dz.sum(0), h, d


def check_backward(dt, x, gain, mean, inv, dz, dx, dgain, dbias):
    wx, wg, wb, h, d = backward_truth(x, gain, mean, inv, dz)
    u, n, rows = U[dt], x.shape[1], x.shape[0]
    i = inv.double()[:, None]
    sa, sb = d.abs().sum(1, keepdim=True) / n, (d * h).abs().sum(1, keepdim=True) / n
    if dx is not None:
        bound = i * u * (4 * d.abs() + (D + 6) * sa + (D + 10) * h.abs() * sb)
        within(dx, wx, bound + 4 * u * wx.abs() + STORE[dt] * wx.abs() + TINY[dt])
    deep = rows / 148 + 48                        # rows that one thread sums up, and the fold after
    if dgain is not None:
        within(dgain, wg, (deep + 4) * u * (dz.double() * h).abs().sum(0) + STORE[dt] * wg.abs() + TINY[dt])
    if dbias is not None:
        within(dbias, wb, deep * u * dz.double().abs().sum(0) + STORE[dt] * wb.abs() + TINY[dt])


def statistics(dt, x, eps=1e-5):
    _, m, i, _ = forward_truth(x, None, None, eps)
    return m.to(WIDE[dt]), i.to(WIDE[dt])


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 4096), (5, 31), (700, 64), (33, 257), (1300, 1000), (900, 1024), (40, 1025),
                                       (301, 2047), (30, 4096), (8, 4097), (5, 8192), (6, 8193), (3, 20001), (2500, 16), (5000, 7)])
def test_backward(ops, dt, rows, cols):
    x = (randn(cols, rows, cols) * 1.5 + randn(cols + 1, rows, 1)).to(KIND[dt])
    dz = randn(cols + 2, rows, cols, dtype=KIND[dt])
    gain = (1 + 0.3 * randn(2, cols)).to(KIND[dt])
    mean, inv = statistics(dt, x)
    dx = torch.full_like(x, 5)
    dgain, dbias = torch.full_like(gain, 5), torch.full_like(gain, 5)
    ops.execLayerNormGrad(dt, None, x, info(x), gain, mean, inv, dz, info(dz), dx, info(dx), dgain, dbias, [1], 1)
    check_backward(dt, x, gain, mean, inv, dz, dx, dgain, dbias)
    again = torch.empty_like(x), torch.empty_like(gain), torch.empty_like(gain)
    ops.execLayerNormGrad(dt, None, x, info(x), gain, mean, inv, dz, info(dz), again[0], info(dx), again[1], again[2], [1], 1)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dgain) and torch.equal(again[2], dbias)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("xl", LAYOUTS)
@pytest.mark.parametrize("dl", ["dense", "apart", "columns"])
@pytest.mark.parametrize("rows,cols", [(6, 96), (40, 1500)])
def test_backward_layouts(ops, dt, xl, dl, rows, cols):
    x = place(randn(5, rows, cols, dtype=KIND[dt]), xl)
    dz = place(randn(6, rows, cols, dtype=KIND[dt]), dl)
    dx = place(torch.full((rows, cols), 5.0, dtype=KIND[dt], device="cuda"), xl)
    mean, inv = statistics(dt, x)
    dgain, dbias = torch.empty(cols, dtype=KIND[dt], device="cuda"), torch.empty(cols, dtype=KIND[dt], device="cuda")
    ops.execLayerNormGrad(dt, None, x, info(x), None, mean, inv, dz, info(dz), dx, info(dx), dgain, dbias, [1], 1)
    check_backward(dt, x, None, mean, inv, dz, dx, dgain, dbias)
    assert between(dx) or xl == "dense"


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("layout", ["dense", "columns"])
@pytest.mark.parametrize("over", ["x", "dz"])
def test_backward_in_place(ops, dt, layout, over):
    rows, cols = 300, 200
    x, dz = place(randn(1, rows, cols, dtype=KIND[dt]), layout), place(randn(2, rows, cols, dtype=KIND[dt]), layout)
    gain = randn(3, cols, dtype=KIND[dt])
    mean, inv = statistics(dt, x)
    keep = x.clone(), dz.clone()
    dgain, dbias = torch.empty_like(gain), torch.empty_like(gain)
    dx = x if over == "x" else dz
    ops.execLayerNormGrad(dt, None, x, info(x), gain, mean, inv, dz, info(dz), dx, info(dx), dgain, dbias, [1], 1)
    check_backward(dt, keep[0], gain, mean, inv, keep[1], dx, dgain, dbias)


@pytest.mark.parametrize("cols", [200, 9000])
def test_backward_parts(ops, cols):
    x, dz = randn(1, 50, cols).float(), randn(2, 50, cols).float()
    gain = randn(3, cols).float()
    mean, inv = statistics(0, x)
    dx, dgain, dbias = torch.empty_like(x), torch.empty_like(gain), torch.empty_like(gain)
    for parts in [(dx, None, None), (None, dgain, None), (None, None, dbias), (None, dgain, dbias), (dx, dgain, None)]:
        for t in (dx, dgain, dbias):
            t.fill_(9)
        ops.execLayerNormGrad(0, None, x, info(x), gain, mean, inv, dz, info(dz), parts[0], None if parts[0] is None else info(dx),
                              parts[1], parts[2], [1], 1)
        check_backward(0, x, gain, mean, inv, dz, *parts)
        for t, p in zip((dx, dgain, dbias), parts):
            assert p is not None or (t == 9).all()


def test_gradient_agrees_with_differences(ops):
    rows, cols, eps = 3, 37, 1e-3
    x, gain, bias, w = randn(1, rows, cols), randn(2, cols), randn(3, cols), randn(4, rows, cols)

    def loss(x, gain, bias):
        z = torch.empty_like(x)
        ops.execLayerNorm(1, None, x, info(x), gain, bias, eps, z, info(z), None, None, [1], 1)
        return float((z * w).sum())
    z, mean, inv = torch.empty_like(x), torch.empty(rows, dtype=torch.float64, device="cuda"), torch.empty(rows, dtype=torch.float64, device="cuda")
    ops.execLayerNorm(1, None, x, info(x), gain, bias, eps, z, info(z), mean, inv, [1], 1)
    dx, dgain, dbias = torch.empty_like(x), torch.empty_like(gain), torch.empty_like(bias)
    ops.execLayerNormGrad(1, None, x, info(x), gain, mean, inv, w, info(w), dx, info(dx), dgain, dbias, [1], 1)
    step = 1e-5                                       # central differences: off by step^2 times the third derivative, and 1e-16 / step
    for i in range(0, cols, 5):
        for t, grad, at in [(x, dx, (1, i)), (gain, dgain, (i,)), (bias, dbias, (i,))]:
            keep = float(t[at])
            t[at] = keep + step
            up = loss(x, gain, bias)
            t[at] = keep - step
            down = loss(x, gain, bias)
            t[at] = keep
            assert abs((up - down) / (2 * step) - float(grad[at])) < 1e-7


def test_no_rows_give_zero_weights(ops):
    x = torch.empty(0, 48, device="cuda")
    dgain, dbias = torch.ones(48, device="cuda"), torch.ones(48, device="cuda")
    ops.execLayerNormGrad(0, None, x, info(x), None, None, None, x, info(x), None, None, dgain, dbias, [1], 1)
    assert (dgain == 0).all() and (dbias == 0).all()
    ops.execLayerNorm(0, None, x, info(x), None, None, 1e-5, x, info(x), None, None, [1], 1)
