"""Embedding lookup and the gradient of its table against 64-bit sums.

Bounds: a looked-up value has the rounding of the scale, of the product and of the stored type; a sum of c rows is off
by c u times the sum of the magnitudes at most, scaling, adding and storing it by one rounding each."""
import pytest
import torch

from tests.lm_cases import KIND, LAYOUTS, NAMES, STORE, TINY, TYPES, U, between, info, place, randn, within

pytestmark = pytest.mark.gpu


def draw_tokens(n, vocab, kind="text", seed=1):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if kind == "one":
        return torch.full((n,), vocab // 2, dtype=torch.int64, device="cuda")
    if kind == "all":
        return torch.arange(n, device="cuda").flip(0) % vocab
    t = torch.pow(float(vocab), torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)).long() - 1
    t = torch.randperm(vocab, device="cuda", generator=gen)[t.clamp(0, vocab - 1)]
    if kind == "outside":
        t[::3] = -1
        t[1::7] = vocab
        t[2::11] = 2 ** 40
        t[5::13] = -2 ** 40
    return t


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,vocab,cols", [(1, 1, 1), (1, 10, 4096), (5, 3, 7), (33, 1000, 64), (1000, 50, 17), (130, 70000, 96), (7, 20, 5000),
                                          (2001, 500, 1024)])
@pytest.mark.parametrize("kind", ["text", "outside"])
def test_lookup(ops, dt, n, vocab, cols, kind):
    table = randn(cols, vocab, cols, dtype=KIND[dt])
    tokens = draw_tokens(n, vocab, kind)
    z = torch.full((n, cols), 5, dtype=KIND[dt], device="cuda")
    ops.execEmbedding(dt, None, table, info(table), tokens, 1.7, z, info(z))
    want = table[tokens.clamp(0, vocab - 1)].double() * 1.7
    want[tokens < 0] = 0
    want[tokens >= vocab] = float("nan")
    within(z, want, (3 * U[dt] + STORE[dt]) * want.abs().nan_to_num(0) + TINY[dt])


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("tl", LAYOUTS)
@pytest.mark.parametrize("zl", LAYOUTS)
def test_lookup_layouts(ops, dt, tl, zl):
    table, tokens = place(randn(1, 40, 48, dtype=KIND[dt]), tl), draw_tokens(21, 40)
    z = place(torch.full((21, 48), 5, dtype=KIND[dt], device="cuda"), zl)
    ops.execEmbedding(dt, None, table, info(table), tokens, 1.0, z, info(z))
    assert torch.equal(z, table[tokens])                  # a scale of 1 copies
    assert between(z) or zl == "dense"


def check_gradient(ops, dt, tokens, vocab, dz, scale, accumulate, layout="dense"):
    cols = dz.shape[1]
    held = randn(77, vocab, cols, dtype=KIND[dt])
    grad = place(held, layout)
    ops.execEmbeddingGrad(dt, None, tokens, scale, dz, info(dz), grad, info(grad), accumulate)
    live = (tokens >= 0) & (tokens < vocab)
    total = torch.zeros(vocab, cols, dtype=torch.float64, device="cuda").index_add_(0, tokens[live], dz[live].double())
    size = torch.zeros(vocab, cols, dtype=torch.float64, device="cuda").index_add_(0, tokens[live], dz[live].double().abs())
    count = torch.bincount(tokens[live], minlength=vocab)[:, None].double()
    want = total * scale + (held.double() if accumulate else 0)
    bound = abs(scale) * (count + 3) * U[dt] * size + 2 * U[dt] * want.abs() + STORE[dt] * want.abs() + TINY[dt]
    within(grad, want, bound)
    if accumulate:
        absent = count[:, 0] == 0
        assert torch.equal(grad[absent], held[absent])
    assert between(grad) or layout == "dense"
    return grad


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,vocab,cols", [(1, 1, 1), (1, 300, 256), (5, 3, 7), (33, 1000, 64), (1000, 50, 17), (130, 70000, 96), (64, 20, 5000),
                                          (2001, 512, 130), (9000, 513, 40), (40000, 300000, 8), (70001, 1000, 12), (8192, 4000, 16)])
@pytest.mark.parametrize("kind", ["text", "outside", "one", "all"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient(ops, dt, n, vocab, cols, kind, accumulate):
    tokens = draw_tokens(n, vocab, kind)
    dz = randn(cols, n, cols, dtype=KIND[dt])
    a = check_gradient(ops, dt, tokens, vocab, dz, 0.3, accumulate)
    b = check_gradient(ops, dt, tokens, vocab, dz, 0.3, accumulate)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("gl", LAYOUTS)
@pytest.mark.parametrize("dl", LAYOUTS)
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_layouts(ops, dt, gl, dl, accumulate):
    dz = place(randn(1, 77, 48, dtype=KIND[dt]), dl)
    check_gradient(ops, dt, draw_tokens(77, 19), 19, dz, 1.0, accumulate, gl)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
def test_infinities_stay_in_their_rows(ops, dt):
    dz = randn(1, 300, 32, dtype=KIND[dt])
    dz[7], dz[9, 3] = float("inf"), float("nan")
    tokens = draw_tokens(300, 40, "all")
    grad = torch.empty(40, 32, dtype=KIND[dt], device="cuda")
    ops.execEmbeddingGrad(dt, None, tokens, 1.0, dz, info(dz), grad, info(grad))
    assert (grad[tokens[7]] == float("inf")).all() and bool(grad[tokens[9], 3].isnan())
    rest = torch.ones(40, dtype=torch.bool, device="cuda")
    rest[tokens[7]] = rest[tokens[9]] = False
    assert grad[rest].isfinite().all()


def test_no_tokens(ops):
    tokens, dz = torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, 24, device="cuda")
    for accumulate, want in ((True, 3.0), (False, 0.0)):
        grad = torch.full((50, 24), 3.0, device="cuda")
        ops.execEmbeddingGrad(0, None, tokens, 1.0, dz, info(dz), grad, info(grad), accumulate)
        assert (grad == want).all()
    table = torch.ones(50, 24, device="cuda")
    ops.execEmbedding(0, None, table, info(table), tokens, 1.0, dz, info(dz))


def test_lookup_and_gradient_are_transposed(ops):
    # <lookup(T), D> = <T, gradient(D)> in exact arithmetic
    table, dz, tokens = randn(1, 60, 40), randn(2, 333, 40), draw_tokens(333, 60)
    z, grad = torch.empty_like(dz), torch.empty_like(table)
    ops.execEmbedding(1, None, table, info(table), tokens, 2.5, z, info(z))
    ops.execEmbeddingGrad(1, None, tokens, 2.5, dz, info(dz), grad, info(grad))
    a, b = float((z * dz).sum()), float((table * grad).sum())
    assert abs(a - b) < 1e-9


def test_the_widest_rows(ops):
    # 2^31 - 2 columns, no whole words: a loop's last step would pass 2^31
    cols = 2 ** 31 - 2
    table = torch.randint(-30000, 30000, (1, cols), device="cuda", dtype=torch.int16).view(torch.float16)
    table[:, :] = table.nan_to_num(1.0, 1.0, 1.0)
    token = torch.zeros(1, dtype=torch.int64, device="cuda")
    z = torch.full((1, cols), 5.0, device="cuda", dtype=torch.float16)
    ops.execEmbedding(2, None, table, info(table), token, 1.0, z, info(z))
    assert torch.equal(z, table)
    z.fill_(5.0)
    ops.execEmbeddingGrad(2, None, token, 1.0, table, info(table), z, info(z))
    assert torch.equal(z, table)
