"""Calls of the operators between a language model's matrix products that their documentation allows and that are easily
forgotten: arrays of more than 2^31 elements, reversed views, a process whose very first call is captured, a graph
replayed with new inputs, results left alone."""
import math
import os
import subprocess
import sys

import pytest
import torch

from libnd4j_b200 import shape as S
from tests.lm_cases import KIND, NAMES, STORE, TINY, TYPES, U, WIDE, info, randn, within

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_beyond_2_31_elements(ops):
    # the last rows of arrays of 2.2e9 halves, where a 32-bit offset would have wrapped
    rows, cols = 540000, 4096
    x = torch.randn(rows, cols, device="cuda", dtype=torch.float16)
    xi = info(x)
    mean, inv = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    z = torch.empty_like(x)
    ops.execLayerNorm(2, None, x, xi, None, None, 1e-5, z, xi, mean, inv, [1], 1)
    tail = x[-3:].double()
    m = tail.mean(1, keepdim=True)
    want = (tail - m) / torch.sqrt(((tail - m) ** 2).mean(1, keepdim=True) + 1e-5)
    within(z[-3:], want, 300 * U[2] * (want.abs() + 1) + STORE[2] * want.abs() + TINY[2])
    tokens = torch.full((rows,), 7, dtype=torch.int64, device="cuda")
    lp, top, lse = (torch.empty(rows, device="cuda") for _ in range(3))
    ops.execTokenLogProbs(2, None, x, xi, tokens, 1.0, lp, None, top, lse)
    log_p = torch.log_softmax(tail, 1)
    within(lp[-3:], log_p[:, 7], 1e-5 * torch.ones(3, device="cuda", dtype=torch.float64))
    g = torch.ones(rows, device="cuda")
    ops.execTokenLogProbsGrad(2, None, x, xi, tokens, 1.0, top, lse, None, g, None, z, xi)
    d = -log_p.exp()
    d[:, 7] += 1
    within(z[-3:], d, 1e-5 * d.abs() + STORE[2] * d.abs() + TINY[2])
    # the same memory as a table
    t = torch.tensor([rows - 1, 0, rows - 2, rows - 1], device="cuda")
    out = torch.empty(4, cols, device="cuda", dtype=torch.float16)
    ops.execEmbedding(2, None, x, xi, t, 1.0, out, info(out))
    assert torch.equal(out, x[t])
    ops.execEmbeddingGrad(2, None, t, 1.0, out, info(out), z, xi)
    within(z[rows - 1], 2 * x[rows - 1].double(), STORE[2] * 2 * x[rows - 1].double().abs())
    assert torch.equal(z[rows - 2], x[rows - 2]) and torch.equal(z[0], x[0]) and not z[1:rows - 2].any()
    norm = torch.empty(1, device="cuda")
    ops.execGlobalNorm(2, None, [x], [rows * cols], 1, norm)
    want = math.sqrt(float(sum((x[i:i + 20000].double() ** 2).sum() for i in range(0, rows, 20000))))
    assert abs(float(norm) - want) <= 8 * U[2] * want


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("cols", [64, 2047])
def test_reversed_rows_and_columns(ops, dt, cols):
    # negative strides: the pointer is that of the first element, the last in memory
    rows = 6
    base = randn(3, rows, cols, dtype=KIND[dt])
    for rs, cs in ((-1, 1), (1, -1), (-1, -1)):
        strides = [rs * cols, cs]
        first = (rows - 1) * cols * (rs < 0) + (cols - 1) * (cs < 0)
        view = S.shape_info([rows, cols], "c", strides, -1)
        at = base.data_ptr() + first * base.element_size()
        x = base.flip([d for d, s in ((0, rs), (1, cs)) if s < 0])
        z = torch.empty_like(base)
        ops.execLayerNorm(dt, None, at, view, None, None, 1e-5, z, info(z), None, None, [1], 1)
        w = x.double()
        m = w.mean(1, keepdim=True)
        want = (w - m) / torch.sqrt(((w - m) ** 2).mean(1, keepdim=True) + 1e-5)
        within(z, want, 200 * U[dt] * (want.abs() + 1) + STORE[dt] * want.abs() + TINY[dt])
        tokens = torch.arange(rows, device="cuda")
        lp = torch.empty(rows, dtype=WIDE[dt], device="cuda")
        ids, lps = torch.empty(rows, 3, dtype=torch.int64, device="cuda"), torch.empty(rows, 3, dtype=WIDE[dt], device="cuda")
        ops.execTokenLogProbs(dt, None, at, view, tokens, 1.0, lp, None, None, None, 3, ids, lps)
        log_p = torch.log_softmax(w, 1)
        within(lp, log_p.gather(1, tokens[:, None])[:, 0], torch.full((rows,), 64 * U[dt] * 16, device="cuda", dtype=torch.float64))
        assert torch.equal(ids, torch.sort(w, dim=1, descending=True, stable=True).indices[:, :3])
        out = torch.empty(rows, cols, dtype=KIND[dt], device="cuda")
        ops.execEmbedding(dt, None, at, view, tokens, 1.0, out, info(out))
        assert torch.equal(out, x)
        ops.execEmbeddingGrad(dt, None, tokens, 1.0, at, view, out, info(out))
        assert torch.equal(out, x)


@pytest.mark.parametrize("dt", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,cols", [(5, 8193), (40, 12345), (3, 16392), (2, 40001), (1, 70001)])
def test_long_rows_of_layer_norm_in_place(ops, dt, rows, cols):
    # rows that a cluster shares, and beyond; gradients and results in their operands' places
    x = randn(cols, rows, cols, dtype=KIND[dt])
    dz = randn(cols + 1, rows, cols, dtype=KIND[dt])
    gain = (1 + 0.2 * randn(2, cols)).to(KIND[dt])
    w = x.double()
    m = w.mean(1, keepdim=True)
    inv = 1 / torch.sqrt(((w - m) ** 2).mean(1, keepdim=True) + 1e-5)
    h = (w - m) * inv
    z = x.clone()
    mean, inv_std = torch.empty(rows, dtype=WIDE[dt], device="cuda"), torch.empty(rows, dtype=WIDE[dt], device="cuda")
    ops.execLayerNorm(dt, None, z, info(z), gain, None, 1e-5, z, info(z), mean, inv_std, [1], 1)
    want = h * gain.double()
    D = 320                                  # at most 70001 / 512 values per thread of the sweep, and the folds
    within(z, want, D * U[dt] * (want.abs() + gain.double().abs()) + STORE[dt] * want.abs() + TINY[dt])
    dx = dz.clone()
    dgain, dbias = torch.empty_like(gain), torch.empty_like(gain)
    ops.execLayerNormGrad(dt, None, x, info(x), gain, mean, inv_std, dx, info(dx), dx, info(dx), dgain, dbias, [1], 1)
    hh = (w - mean.double()[:, None]) * inv_std.double()[:, None]
    d = dz.double() * gain.double()
    sa, sb = d.abs().mean(1, keepdim=True), (d * hh).abs().mean(1, keepdim=True)
    want = inv_std.double()[:, None] * (d - d.mean(1, keepdim=True) - hh * (d * hh).mean(1, keepdim=True))
    bound = inv_std.double()[:, None] * U[dt] * (8 * d.abs() + D * sa + D * hh.abs() * sb)
    within(dx, want, bound + STORE[dt] * want.abs() + TINY[dt])
    g = (dz.double() * hh)
    within(dgain, g.sum(0), (rows + 60) * U[dt] * g.abs().sum(0) + STORE[dt] * g.sum(0).abs() + TINY[dt])
    within(dbias, dz.double().sum(0), (rows + 60) * U[dt] * dz.double().abs().sum(0) + STORE[dt] * dz.double().sum(0).abs() + TINY[dt])


FIRST = """
import torch
from libnd4j_b200 import shape as S
from libnd4j_b200.native_ops import NativeOps
ops = NativeOps()
torch.manual_seed(1)
x, dz = torch.randn(3000, 512, device="cuda"), torch.randn(3000, 512, device="cuda")
gain = torch.ones(512, device="cuda")
mean, inv = x.mean(1), 1 / torch.sqrt(x.var(1, correction=0) + 1e-5)
dx, dg, db, grad, norm = torch.empty_like(x), torch.empty_like(gain), torch.empty_like(gain), torch.empty(100, 512, device="cuda"), torch.zeros(1, device="cuda")
tokens = torch.randint(0, 100, (3000,), device="cuda")
torch.cuda.synchronize()
xi, gi = S.shape_info([3000, 512]), S.shape_info([100, 512])
def step():
    e = [None, torch.cuda.current_stream().cuda_stream]
    ops.execLayerNormGrad(0, e, x, xi, gain, mean, inv, dz, xi, dx, xi, dg, db, [1], 1)
    ops.execEmbeddingGrad(0, e, tokens, 1.0, dx, xi, grad, gi)
    ops.execClipByGlobalNorm(0, e, [grad, dg, db], None, [51200, 512, 512], 3, 1.0, norm)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    step()
g.replay()
torch.cuda.synchronize()
kept = [t.clone() for t in (dx, grad, dg, db, norm)]
for t in (dx, grad, dg, db, norm):
    t.fill_(float("nan"))
step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(kept, (dx, grad, dg, db, norm)))
assert kept[4] > 1
print("the captured first call equals the eager one")
"""


def test_a_process_whose_first_call_is_captured(ops):
    out = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "equals the eager one" in out.stdout, out.stderr[-2000:]


def test_rows_of_padding_cost_no_memory_access_and_leave_zeros(ops):
    # nothing of a padded row is read: it may hold anything
    x = randn(1, 6, 5000).float()
    x[2], x[4] = float("nan"), float("inf")
    tokens = torch.tensor([0, 1, -1, 3, -7, 5], device="cuda")
    out = [torch.full((6,), 9.0, device="cuda") for _ in range(4)]
    ids, lps = torch.full((6, 40), 9, dtype=torch.int64, device="cuda"), torch.full((6, 40), 9.0, device="cuda")
    ops.execTokenLogProbs(0, None, x, info(x), tokens, 1.0, *out, 40, ids, lps)
    for t in out:
        assert t[2] == 0 and t[4] == 0 and t[[0, 1, 3, 5]].isfinite().all()
    assert (ids[[2, 4]] == -1).all() and (lps[[2, 4]] == 0).all() and (ids[[0, 1, 3, 5]] >= 0).all()
    g = torch.full((6,), float("nan"), device="cuda")
    g[[0, 1, 3, 5]] = 1.0
    dx = torch.full_like(x, 9.0)
    ops.execTokenLogProbsGrad(0, None, x, info(x), tokens, 1.0, out[2], out[3], out[1], g, g, dx, info(dx))
    assert (dx[[2, 4]] == 0).all() and dx[[0, 1, 3, 5]].isfinite().all()


def test_ranks_repeated_dimensions_and_broadcast_rows(ops):
    # a vector as one TAD; an axis named twice; an operand whose rows are all the same memory
    x = randn(1, 5000).float()
    z = torch.empty_like(x)
    one = S.shape_info([5000])
    mean, inv = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    ops.execLayerNorm(0, None, x, one, None, None, 1e-5, z, one, mean, inv, [0], 1)
    w = x.double()
    want = (w - w.mean()) / torch.sqrt(w.var(correction=0) + 1e-5)
    within(z, want, 200 * U[0] * (want.abs() + 1))
    x = randn(2, 7, 640).float()
    a, b = torch.empty_like(x), torch.empty_like(x)
    ops.execLayerNorm(0, None, x, info(x), None, None, 1e-5, a, info(a), None, None, [1], 1)
    ops.execLayerNorm(0, None, x, info(x), None, None, 1e-5, b, info(b), None, None, [1, -1, 1], 3)
    assert torch.equal(a, b)
    same = S.shape_info([7, 640], "c", [0, 1], -1)
    ops.execLayerNorm(0, None, x[0], same, None, None, 1e-5, b, info(b), None, None, [1], 1)
    assert all(torch.equal(b[r], a[0]) for r in range(7))
    tokens = torch.arange(7, device="cuda")
    lp, full = torch.empty(7, device="cuda"), torch.empty(7, device="cuda")
    ops.execTokenLogProbs(0, None, x[0], same, tokens, 1.0, lp, None, None, None)
    ops.execTokenLogProbs(0, None, x[:1].expand(7, 640).contiguous(), info(x), tokens, 1.0, full, None, None, None)
    assert torch.equal(lp, full)
    grad = torch.empty(9, 640, device="cuda")
    ops.execEmbeddingGrad(0, None, torch.full((7,), 3, dtype=torch.int64, device="cuda"), 1.0, x[0], same, grad, info(grad))
    within(grad[3], 7 * x[0].double(), 10 * U[0] * 7 * x[0].double().abs())


def test_launches_without_overlap(ops):
    # programmatic launches switched off: the same bits
    x, dz = randn(1, 900, 1024).float(), randn(2, 900, 1024).float()
    gain, tokens = randn(3, 1024).float(), torch.randint(0, 50, (900,), device="cuda")
    mean, inv = x.mean(1), 1 / torch.sqrt(x.var(1, correction=0) + 1e-5)

    def run():
        dx, dg, db = torch.empty_like(x), torch.empty_like(gain), torch.empty_like(gain)
        grad, norm, lp = torch.empty(50, 1024, device="cuda"), torch.empty(1, device="cuda"), torch.empty(900, device="cuda")
        ops.execLayerNormGrad(0, None, x, info(x), gain, mean, inv, dz, info(dz), dx, info(dx), dg, db, [1], 1)
        ops.execEmbeddingGrad(0, None, tokens, 1.0, dx, info(dx), grad, info(grad))
        ops.execTokenLogProbs(0, None, dx, info(dx), tokens, 1.0, lp, None, None, None)
        ops.execClipByGlobalNorm(0, None, [grad, dg, db], None, [51200, 1024, 1024], 3, 0.5, norm)
        ops.execClipByGlobalNorm(0, None, [dg], None, [1024], 1, 0.1, norm)
        return dx, dg, db, grad, norm, lp
    a = run()
    ops._check(ops.lib.nd4jb200_set_tuning(3, 0))
    try:
        b = run()
    finally:
        ops._check(ops.lib.nd4jb200_set_tuning(3, 1))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_a_table_without_rows(ops):
    table, z = torch.empty(0, 16, device="cuda"), torch.empty(3, 16, device="cuda")
    ops.execEmbedding(0, None, table, info(table), torch.tensor([-1, 0, 5], device="cuda"), 1.0, z, info(z))
    assert (z[0] == 0).all() and z[1:].isnan().all()


def test_scratch_memory_goes_back_to_the_device(ops):
    # 2^22 tokens of 4096 halves: 65536 chunks of the sorted list with two partial rows of floats each, 2 GB, besides the
    # lists. After a synchronisation no more than 1 GB of scratch memory may still be held, and none once it is released.
    # (32 MB: what the driver may have taken for itself meanwhile.)
    n, cols = 1 << 22, 4096
    dz = torch.ones(cols, device="cuda", dtype=torch.float16)
    same = S.shape_info([n, cols], "c", [0, 1], -1)
    tokens = torch.arange(n, device="cuda") % 7
    grad = torch.empty(8, cols, device="cuda", dtype=torch.float16)
    few = S.shape_info([100, cols], "c", [0, 1], -1)
    ops.execEmbeddingGrad(2, None, tokens[:100], 2.0 ** -7, dz, few, grad, info(grad))          # loads what the calls need
    big = torch.empty(5, device="cuda")
    ops.execGlobalNorm(0, None, [big], [5], 1, torch.empty(1, device="cuda"))
    torch.cuda.synchronize()
    ops.releaseScratch()
    free = torch.cuda.mem_get_info()[0]
    ops.execEmbeddingGrad(2, None, tokens, 2.0 ** -7, dz, same, grad, info(grad))
    torch.cuda.synchronize()
    held = free - torch.cuda.mem_get_info()[0]
    counts = torch.bincount(tokens, minlength=8)
    within(grad, (counts.double() / 128)[:, None].expand(8, cols), STORE[2] * (counts.double() / 128)[:, None] + TINY[2])
    assert held <= (1024 + 32) << 20, "%d MB are held" % (held >> 20)
    ops.releaseScratch()
    held = free - torch.cuda.mem_get_info()[0]
    assert held <= 32 << 20, "%d MB are held after the release" % (held >> 20)


def test_scratch_memory_is_released_while_a_stream_is_captured(ops):
    x, dz = randn(1, 900, 512).float(), randn(2, 900, 512).float()
    mean, inv = x.mean(1), 1 / torch.sqrt(x.var(1, correction=0) + 1e-5)
    dx, dg = torch.empty_like(x), torch.empty(512, device="cuda")

    def step(extra):
        ops.execLayerNormGrad(0, extra, x, info(x), None, mean, inv, dz, info(dz), dx, info(dx), dg, None, [1], 1)
    step(None)
    torch.cuda.synchronize()
    want = dx.clone(), dg.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        extra = [None, torch.cuda.current_stream().cuda_stream]
        step(extra)
        ops.releaseScratch()
        step(extra)
    for t in (dx, dg):
        t.fill_(9)
    ops.releaseScratch()
    g.replay()
    step(None)
    torch.cuda.synchronize()
    assert torch.equal(dx, want[0]) and torch.equal(dg, want[1])
