"""Log probabilities of tokens, entropies and best alternatives, and their gradient, against the formulas in 64 bits.

Bounds. With u the roundoff of the sums' type and E the relative error of an exponential (2^-22 for the float
instruction, 4 u for double), an exponential of d is off by E + 5 u |d| relative, a sum of n terms of one sign by another
D u with D the longest chain of additions. So log s is off by e_s = E + (D + 5 dbar) u, dbar = sum p |d|; log p by e_s
plus 6 u (|d| + |log p|); the entropy by (1 + dbar) e_s and its own roundings."""
import math

import pytest
import torch

from tests.lm_cases import KIND, LAYOUTS, NAMES, STORE, TINY, TYPES, U, WIDE, between, info, place, randn, within

pytestmark = pytest.mark.gpu
E = {0: 2.0 ** -22, 1: 4 * 2.0 ** -53, 2: 2.0 ** -22}


def truth(x, scale):
    """log p with -inf where p is 0, entropy, maximum, log sum; rows without a value: -inf, 0; odd rows: NaN."""
    x = x.double()
    top = x.max(1).values
    d = (x - top[:, None]) * scale
    s = torch.where(d > -math.inf, d.exp(), 0).sum(1)
    log_p = d - s.log()[:, None]
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, 0).sum(1)
    log_sum = s.log()
    empty = top == -math.inf
    log_p[empty], entropy[empty], log_sum[empty] = -math.inf, 0.0, -math.inf
    odd = x.isnan().any(1) | (x == math.inf).any(1)
    for t in (log_p, entropy, top, log_sum):
        t[odd] = math.nan
    return log_p, entropy, top, log_sum


def best(x, k):
    """Indices of the k best: NaN first, then by value, equal ones by index."""
    key = x.double().clone()
    key[key.isnan()] = math.inf
    first = x.isnan()
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    # among the largest, NaNs go before infinities
    rank = torch.gather(first, 1, order)
    again = torch.sort(rank.int(), dim=1, descending=True, stable=True).indices
    return torch.gather(order, 1, again)[:, :k]


def bounds(dt, x, log_p, entropy, log_sum, scale):
    u, vocab = U[dt], x.shape[1]
    d = (log_p + log_sum[:, None]).abs()
    p = log_p.exp()
    dbar = torch.where(p > 0, p * d, 0).sum(1)
    chain = vocab / 512 + 64 if dt != 1 else vocab / 256 + 64
    e_s = E[dt] + (chain + 5 * dbar) * u + 4 * u
    e_lp = e_s[:, None] + 6 * u * (d + log_p.abs())
    e_h = 2 * (1 + dbar) * e_s + 6 * u * (log_sum.abs() + dbar)
    return e_s, e_lp, e_h


def check(ops, dt, x, tokens, scale, k=0):
    rows, vocab = x.shape
    out = [torch.full((rows,), 9, dtype=WIDE[dt], device="cuda") for _ in range(4)]
    ids = torch.full((rows, k), 9, dtype=torch.int64, device="cuda") if k else None
    lps = torch.full((rows, k), 9, dtype=WIDE[dt], device="cuda") if k else None
    ops.execTokenLogProbs(dt, None, x, info(x), tokens, scale, *out, k, ids, lps)
    log_p, entropy, top, log_sum = truth(x, scale)
    e_s, e_lp, e_h = bounds(dt, x, log_p, entropy, log_sum, scale)
    pad = tokens < 0
    beyond = tokens >= vocab
    at = tokens.clamp(0, vocab - 1)[:, None]
    want = torch.where(beyond, math.nan, log_p.gather(1, at)[:, 0])
    zero = torch.zeros_like(want)
    within(out[0], torch.where(pad, zero, want), e_lp.gather(1, at)[:, 0].nan_to_num(0, 0, 0))
    within(out[1], torch.where(pad, zero, entropy), e_h.nan_to_num(0, 0, 0))
    assert torch.equal(out[2].double().nan_to_num(1e300), torch.where(pad, zero, top).nan_to_num(1e300))
    within(out[3], torch.where(pad, zero, log_sum), (e_s + 4 * U[dt] * log_sum.abs()).nan_to_num(0, 0, 0))
    if k:
        want_ids = best(x, k)
        assert torch.equal(ids, torch.where(pad[:, None], -1, want_ids))
        within(lps, torch.where(pad[:, None], 0.0, log_p.gather(1, want_ids)), e_lp.gather(1, want_ids).nan_to_num(0, 0, 0))
    return out


def some_tokens(rows, vocab, seed=1):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randint(0, vocab, (rows,), device="cuda", generator=gen)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (2, 7, 7), (5, 64, 5), (300, 100, 0), (4, 501, 64), (7, 1000, 20), (3, 4097, 1),
                                          (2, 20000, 20), (1, 50001, 33), (8, 131072, 20), (160, 9999, 3), (17, 32768, 0), (1, 600001, 10),
                                          (75, 40000, 16), (40, 66000, 17)])
def test_forward(ops, dt, rows, vocab, k):
    x = (randn(vocab, rows, vocab) * 3).to(KIND[dt])
    tokens = some_tokens(rows, vocab)
    if rows > 2:
        tokens[1] = -1
    if rows > 4:
        tokens[4] = vocab
    check(ops, dt, x, tokens, 0.7, k)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("rows,vocab", [(5, 100), (3, 4099), (2, 40003)])
def test_forward_layouts(ops, dt, layout, rows, vocab):
    x = place((randn(3, rows, vocab) * 2).to(KIND[dt]), layout)
    check(ops, dt, x, some_tokens(rows, vocab), 1.0, 9)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("vocab", [40, 3001, 70000])
def test_masks(ops, dt, vocab):
    low = torch.finfo(KIND[dt]).min
    x = (randn(9, 14, vocab) * 2).to(KIND[dt])
    x[0] = -math.inf                                      # nothing is left
    x[1, 3:] = -math.inf                                  # fewer values than alternatives
    x[2] = low                                            # the type's lowest everywhere: uniform
    x[3, : vocab - 2] = low                               # ... as a mask
    x[4, vocab // 2] = math.nan
    x[5, 5], x[5, 9] = math.inf, math.inf
    x[6] = 1.5                                            # all alike: ties
    x[7] = torch.linspace(-2, 2, vocab, device="cuda").to(KIND[dt])        # ascending
    x[8, ::2] = -math.inf
    x[9] = torch.where(x[9] > 0, torch.zeros_like(x[9]), -torch.zeros_like(x[9]))       # +0 and -0 are equal
    x[10] = -math.inf
    x[10, vocab - 1] = low                                # a single entry, the lowest one
    x[11] = torch.finfo(KIND[dt]).max                     # the largest everywhere
    x[12, : vocab // 2] = -math.inf
    x[13, 1], x[13, 2], x[13, 30] = math.nan, math.inf, math.nan
    tokens = torch.zeros(14, dtype=torch.int64, device="cuda")
    tokens[3] = vocab - 1
    check(ops, dt, x, tokens, 1.0, 16)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
def test_more_equal_values_than_the_list_holds(ops, dt):
    # the best values fill the slices of few threads: the collected candidates overflow
    x = torch.zeros(2, 131072, device="cuda", dtype=KIND[dt])
    V = 16 // x.element_size()
    for cluster in (1, 2, 4, 8):
        for word in range(20):
            x[:, word * V::512 * V * cluster] = 1.0
            x[1, word * V::512 * V * cluster] += torch.arange(0, x[1, word * V::512 * V * cluster].numel(), device="cuda").to(KIND[dt]) / 64
    check(ops, dt, x, torch.tensor([0, 5], device="cuda"), 1.0, 20)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("scale", [1e-3, 1.0, 40.0])
def test_scales_and_offsets(ops, dt, scale):
    x = (randn(2, 6, 5000) * 2 + 500 * randn(3, 6, 1)).to(KIND[dt])
    check(ops, dt, x, some_tokens(6, 5000), scale, 4)


def test_parts(ops):
    x = randn(1, 9, 777).float()
    tokens = some_tokens(9, 777)
    full = check(ops, 0, x, tokens, 1.0)
    for which in range(4):
        out = [torch.full((9,), 3.0, device="cuda") if i == which else None for i in range(4)]
        ops.execTokenLogProbs(0, None, x, info(x), tokens if which == 0 else None, 1.0, *out)
        assert torch.equal(out[which], full[which])
    ids, lps = torch.empty(9, 3, dtype=torch.int64, device="cuda"), torch.empty(9, 3, device="cuda")
    ops.execTokenLogProbs(0, None, x, info(x), None, 1.0, None, None, None, None, 3, ids, lps)
    assert torch.equal(ids, best(x, 3))


def grad_truth(x, tokens, scale, g, h):
    log_p, entropy, _, _ = truth(x, scale)
    vocab = x.shape[1]
    p = log_p.exp()
    p[(x == -math.inf).all(1)] = 0
    d = -g[:, None] * p
    rows = torch.arange(x.shape[0], device="cuda")
    d[rows, tokens.clamp(0, vocab - 1)] += g
    if h is not None:
        d = d - h[:, None] * torch.where(p > 0, p * (log_p + entropy[:, None]), torch.where(p.isnan(), p, 0))
    d *= scale
    d[(x == -math.inf).all(1)] = 0
    d[tokens >= vocab] = math.nan
    d[tokens < 0] = 0
    return d, log_p, entropy, p


def check_grad(ops, dt, x, tokens, scale, entropy_too, out_layout="dense", in_place=False):
    rows, vocab = x.shape
    _, H, top, log_sum = truth(x, scale)
    wide = [t.to(WIDE[dt]) for t in (top, log_sum, H)]
    g = randn(7, rows, dtype=WIDE[dt])
    h = randn(8, rows, dtype=WIDE[dt]) if entropy_too else None
    want, log_p, entropy, p = grad_truth(x, tokens, scale, g.double(), None if h is None else h.double())
    given = x.clone() if not in_place else x
    dx = x if in_place else place(torch.full_like(x, 5), out_layout)
    ops.execTokenLogProbsGrad(dt, None, x, info(x), tokens, scale, wide[0], wide[1], wide[2], g, h, dx, info(dx))
    u = U[dt]
    d = (log_p + log_sum[:, None]).abs()
    rel = E[dt] + u * (8 * d + 6 * log_p.abs() + 8 * log_sum.abs()[:, None] + 8)
    size = g.double().abs()[:, None] * p
    if h is not None:
        size = size + h.double().abs()[:, None] * p * (log_p.clamp(min=-1e4).abs() + entropy[:, None] + 1)
    shared = torch.where(p > 0, size * (rel + 6 * u), 0)          # p = 0 has no error, though its exponent is infinite
    bound = scale * shared + 6 * u * scale * g.double().abs()[:, None] + STORE[dt] * want.abs() + TINY[dt]
    within(dx, want, bound.nan_to_num(0, 0, 0))
    assert in_place or torch.equal(given.nan_to_num(3), x.nan_to_num(3))
    return dx


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 7), (5, 64), (300, 101), (4, 4097), (3, 8191), (2, 50001), (1, 131072)])
@pytest.mark.parametrize("entropy_too", [False, True])
def test_gradient(ops, dt, rows, vocab, entropy_too):
    x = (randn(vocab, rows, vocab) * 3).to(KIND[dt])
    tokens = some_tokens(rows, vocab)
    if rows > 2:
        tokens[1] = -1
    if rows > 4:
        tokens[4] = vocab
        x[3] = -math.inf
        x[2, ::2] = -math.inf
    check_grad(ops, dt, x, tokens, 0.7, entropy_too)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("out", LAYOUTS)
def test_gradient_layouts(ops, dt, layout, out):
    x = place((randn(3, 3, 1201) * 2).to(KIND[dt]), layout)
    dx = check_grad(ops, dt, x, some_tokens(3, 1201), 1.0, True, out)
    assert between(dx) or out == "dense"


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("layout", ["dense", "shifted", "every second"])
def test_gradient_in_place(ops, dt, layout):
    x = place((randn(3, 4, 1201) * 2).to(KIND[dt]), layout)
    check_grad(ops, dt, x, some_tokens(4, 1201), 1.0, True, in_place=True)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
def test_gradient_special_rows(ops, dt):
    x = (randn(9, 6, 900) * 2).to(KIND[dt])
    x[0] = -math.inf
    x[1, 4] = math.nan
    x[2] = torch.finfo(KIND[dt]).min
    x[3, 10:] = torch.finfo(KIND[dt]).min
    x[4, 3:] = -math.inf
    check_grad(ops, dt, x, torch.tensor([5, 5, 5, 5, 500, 5], device="cuda"), 1.0, True)


def test_gradient_agrees_with_differences(ops):
    rows, vocab, scale = 2, 23, 1.3
    x = randn(1, rows, vocab)
    tokens = torch.tensor([4, 20], device="cuda")
    g, h = randn(2, rows), randn(3, rows)
    out = [torch.empty(rows, dtype=torch.float64, device="cuda") for _ in range(4)]

    def loss():
        ops.execTokenLogProbs(1, None, x, info(x), tokens, scale, *out)
        return float((g * out[0] + h * out[1]).sum())
    loss()
    dx = torch.empty_like(x)
    ops.execTokenLogProbsGrad(1, None, x, info(x), tokens, scale, out[2].clone(), out[3].clone(), out[1].clone(), g, h, dx, info(dx))
    step = 1e-5
    for at in [(0, 4), (0, 0), (1, 20), (1, 7), (1, 22)]:
        keep = float(x[at])
        x[at] = keep + step
        up = loss()
        x[at] = keep - step
        down = loss()
        x[at] = keep
        assert abs((up - down) / (2 * step) - float(dx[at])) < 1e-7


def sharp_rows(dt, vocab):
    """Rows for scales at which a row's maximum takes nearly all of it: maxima all over a logit's usual range, maxima that
    two or three entries share, the largest half, masks."""
    x = (randn(17, 12, vocab) * 4).to(KIND[dt])
    x[1] = x[1] * 0.01 + 59.97
    x[2, vocab // 3], x[2, vocab - 1] = 37.3125, 37.3125
    x[3, 0], x[3, 1], x[3, vocab // 2] = 41.03125, 41.03125, 41.03125
    x[4, 7] = 65504.0
    x[5] = -65504.0
    x[6, 3:] = -math.inf
    x[7] = -math.inf
    x[8] = x[8].abs() * -30 - 1
    return x


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("scale", [170.0, 200.0, 1e6, 1e8, 1e29])
@pytest.mark.parametrize("vocab", [64, 3001, 70000])
def test_large_scales(ops, dt, scale, vocab):
    x = sharp_rows(dt, vocab)
    tokens = x.double().argmax(1)                         # log probabilities of nearly 0
    tokens[9], tokens[10], tokens[11] = 1, -1, vocab
    check(ops, dt, x, tokens, scale, 4)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("scale", [170.0, 200.0, 1e6, 1e8, 1e29])
@pytest.mark.parametrize("entropy_too", [False, True])
def test_gradient_at_large_scales(ops, dt, scale, entropy_too):
    # upstream gradients as small as the scale is large, so that the result stays in the range of a half
    vocab = 3001
    x = sharp_rows(dt, vocab)
    rows = x.shape[0]
    tokens = x.double().argmax(1)
    tokens[9], tokens[10], tokens[11] = 1, -1, vocab
    _, H, top, log_sum = truth(x, scale)
    wide = [t.to(WIDE[dt]) for t in (top, log_sum, H)]
    g = (randn(7, rows) / scale).to(WIDE[dt])
    h = (randn(8, rows) / scale).to(WIDE[dt]) if entropy_too else None
    want, log_p, entropy, p = grad_truth(x, tokens, scale, g.double(), None if h is None else h.double())
    dx = torch.full_like(x, 5)
    ops.execTokenLogProbsGrad(dt, None, x, info(x), tokens, scale, wide[0], wide[1], wide[2], g, h, dx, info(dx))
    u = U[dt]
    d = (log_p + log_sum[:, None]).abs()
    rel = E[dt] + u * (8 * d + 6 * log_p.abs() + 8 * log_sum.abs()[:, None] + 8)
    size = g.double().abs()[:, None] * p
    if h is not None:
        size = size + h.double().abs()[:, None] * p * (log_p.clamp(min=-1e4).abs() + entropy[:, None] + 1)
    shared = torch.where(p > 0, size * (rel + 6 * u), 0)
    # a probability below 2^-126 counts as 0 for float and half data: the shared part of it is below 2^-120
    bound = scale * shared + 6 * u * scale * g.double().abs()[:, None] + STORE[dt] * want.abs() + TINY[dt]
    within(dx, want, bound.nan_to_num(0, 0, 0))


def collected(x, cluster, k, vec):
    """How many candidates each CTA of a cluster collects for the k best of a row: the entries, at or above the k-th best of
    its threads' maxima, of the slices whose maximum reaches it (a slice: every 256 * cluster-th word of 16 bytes)."""
    words = x.double().view(-1, vec)
    counts = []
    for rank in range(cluster):
        slices = [words[rank * 256 + t::256 * cluster].flatten() for t in range(256)]
        tops = torch.stack([s.max() if s.numel() else torch.tensor(-math.inf, device=x.device, dtype=torch.float64) for s in slices])
        least = tops.sort(descending=True).values[k - 1]
        counts.append(sum(int((s >= least).sum()) for s, t in zip(slices, tops) if t >= least))
    return counts


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,vocab,cluster", [(160, 40000, 1), (3, 262144, 8)])
def test_candidates_beyond_the_list(ops, dt, rows, vocab, cluster):
    # the slices of nineteen threads lie above everything else, and those of a twentieth just below them: what reaches the
    # twentieth's maximum is more than the 1024 candidates that are collected, and the best are then taken one by one
    vec = 128 // torch.finfo(KIND[dt]).bits
    x = randn(5, rows, vocab).to(KIND[dt])
    span = 256 * cluster
    words = x.view(rows, vocab // vec, vec)

    def raise_slices(row, rank, first):
        for t in range(20):
            part = words[row, rank * 256 + first + t * 11::span]
            steps = torch.arange(part.numel(), device="cuda").view(part.shape)
            # distinct within a slice, in an order of their own, equal ones in other slices
            part.copy_((16.0 if t == 7 else 32 + (steps * 37 % part.numel()) / 64.0) * torch.ones_like(steps, dtype=torch.float64))
    raise_slices(0, 0, 3)
    raise_slices(1, cluster - 1, 20)
    for rank in range(cluster):
        raise_slices(2, rank, rank)
    x[2, 1] = 60000.0                                     # in the first of the raised slices
    for row, where in ((0, 0), (1, cluster - 1), (2, 0)):
        assert collected(x[row], cluster, 20, vec)[where] > 1024
    check(ops, dt, x, some_tokens(rows, vocab), 1.0, 20)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("scale", [1.0, 500.0])
@pytest.mark.parametrize("entropy_too", [False, True])
def test_gradient_of_rows_without_values_for_tokens_beyond_them(ops, dt, scale, entropy_too):
    x = (randn(9, 5, 333) * 2).to(KIND[dt])
    x[:3] = -math.inf
    check_grad(ops, dt, x, torch.tensor([333, 7, -1, 1000000, 5], device="cuda"), scale, entropy_too)
