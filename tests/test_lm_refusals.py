"""What the operators between a language model's matrix products refuse. Every call here ends in its argument checks,
before anything reaches a GPU; the pointers are never followed."""
import ctypes

import numpy as np
import pytest

from libnd4j_b200 import native_ops, shape as S

LP = ctypes.POINTER(ctypes.c_longlong)
IP = ctypes.POINTER(ctypes.c_int)
A, B, C, D, E, F, G = (0x10000000 * k for k in range(1, 8))          # seven arrays far from one another


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(native_ops.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return native_ops.load_library()


KEEP = []


def longs(a):
    a = np.ascontiguousarray(a, dtype=np.int64)
    KEEP.append(a)
    return a.ctypes.data_as(LP)


def ints(a):
    a = np.ascontiguousarray(a, dtype=np.int32)
    KEEP.append(a)
    return a.ctypes.data_as(IP)


def dense(*shape):
    return longs(S.shape_info(shape))


def strided(shape, strides):
    return longs(S.shape_info(shape, "c", strides))


def refused(lib, rc, word, code=1):
    assert rc == code, rc
    assert word in lib.nd4jb200_last_error().decode(), lib.nd4jb200_last_error().decode()


LN = dict(dtype=0, x=A, xi=(8, 64), gain=B, bias=C, eps=1e-5, z=D, zi=(8, 64), mean=E, inv=F, dims=(1,))


@pytest.mark.parametrize("change,word", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(x=None), "x is null"), (dict(z=None), "z is null"), (dict(eps=0.0), "epsilon"),
    (dict(eps=float("nan")), "epsilon"), (dict(eps=float("inf")), "epsilon"), (dict(eps=1e-300), "epsilon"), (dict(zi=(8, 32)), "shape"),
    (dict(zi=(8, 8, 8)), "not an axis|shape"), (dict(dims=()), "dimension"), (dict(dims=(2,)), "axis"), (dict(x=A + 2), "aligned"),
    (dict(mean=E + 1), "aligned"), (dict(z=A + 4), "overlaps"), (dict(mean=A), "overlaps"), (dict(inv=E), "overlaps"), (dict(gain=D), "overlaps"),
])
def test_layer_norm(lib, change, word):
    a = dict(LN, **change)
    rc = lib.nd4jb200_exec_layer_norm(None, a["dtype"], a["x"], dense(*a["xi"]), a["gain"], a["bias"], a["eps"], a["z"], dense(*a["zi"]),
                                      a["mean"], a["inv"], ints(a["dims"]), len(a["dims"]))
    assert rc == 1 and any(w in lib.nd4jb200_last_error().decode() for w in word.split("|")), lib.nd4jb200_last_error()


def test_layer_norm_descriptors(lib):
    refused(lib, lib.nd4jb200_exec_layer_norm(None, 0, A, None, None, None, 1e-5, B, dense(2, 3), None, None, ints([1]), 1), "shapeInfo")
    refused(lib, lib.nd4jb200_exec_layer_norm(None, 0, A, dense(2, 3), None, None, 1e-5, B, dense(2, 3), None, None, None, 1), "dimension")
    refused(lib, lib.nd4jb200_exec_layer_norm(None, 0, A, dense(4, 8), None, None, 1e-5, B, strided((4, 8), (0, 1)), None, None, ints([1]), 1),
            "stride of 0")


LNG = dict(dtype=2, x=A, xi=(8, 64), gain=B, mean=C, inv=D, dz=E, dzi=(8, 64), dx=F, dxi=(8, 64), dgain=G, dbias=G + 128, dims=(1,))


@pytest.mark.parametrize("change,word", [
    (dict(dtype=7), "dtype"), (dict(mean=None), "mean is null"), (dict(inv=None), "invStd is null"), (dict(dz=None), "dz is null"),
    (dict(dzi=(64, 8)), "shape"), (dict(dxi=(8, 63)), "shape"), (dict(dx=A + 2), "overlaps"), (dict(dx=E + 64), "overlaps"), (dict(dbias=G), "overlaps"),
    (dict(dgain=A), "overlaps"), (dict(dgain=C), "overlaps"), (dict(dx=B), "overlaps"), (dict(dims=(-3,)), "axis"), (dict(dgain=G + 1), "aligned"),
])
def test_layer_norm_gradient(lib, change, word):
    a = dict(LNG, **change)
    rc = lib.nd4jb200_exec_layer_norm_grad(None, a["dtype"], a["x"], dense(*a["xi"]), a["gain"], a["mean"], a["inv"], a["dz"], dense(*a["dzi"]),
                                           a["dx"], dense(*a["dxi"]), a["dgain"], a["dbias"], ints(a["dims"]), len(a["dims"]))
    refused(lib, rc, word)


LPF = dict(dtype=0, x=A, xi=(8, 64), tokens=B, scale=1.0, lp=C, h=C + 256, m=C + 512, s=C + 768, k=4, ids=D, lps=E)


@pytest.mark.parametrize("change,word", [
    (dict(dtype=9), "dtype"), (dict(x=None), "logits is null"), (dict(tokens=None), "tokens is null"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=1e31), "scale"), (dict(k=-1), "k must"), (dict(k=65), "k must"),
    (dict(xi=(8, 3)), "k exceeds"), (dict(ids=None), "topTokens"), (dict(lps=None), "topLogProbs"), (dict(xi=(8, 8, 8)), "rank 2"),
    (dict(lp=A), "overlaps"), (dict(h=C), "overlaps"), (dict(ids=B), "overlaps"), (dict(tokens=B + 4), "aligned"), (dict(xi=(8, 0)), "without entries"),
    (dict(lp=None, h=None, m=None, s=None, k=0), "no result"),
])
def test_token_log_probs(lib, change, word):
    a = dict(LPF, **change)
    rc = lib.nd4jb200_exec_token_log_probs(None, a["dtype"], a["x"], dense(*a["xi"]), a["tokens"], a["scale"], a["lp"], a["h"], a["m"], a["s"],
                                           a["k"], a["ids"], a["lps"])
    refused(lib, rc, word)


def test_rows_beyond_the_limit(lib):
    rc = lib.nd4jb200_exec_token_log_probs(None, 0, A, dense(1, (1 << 30) + 1), B, 1.0, C, None, None, None, 0, None, None)
    refused(lib, rc, "2^30", 5)
    rc = lib.nd4jb200_exec_embedding(None, 0, A, dense(1 << 31, 1), B, 1.0, C, dense(4, 1))
    refused(lib, rc, "2^31", 5)
    rc = lib.nd4jb200_exec_embedding_grad(None, 0, B, 1.0, C, dense((1 << 30) + 1, 1), A, dense(5, 1), 0)
    refused(lib, rc, "2^30", 5)


LPG = dict(dtype=1, x=A, xi=(8, 64), tokens=B, scale=1.0, m=C, s=C + 256, h=C + 512, g=C + 1024, gh=C + 2048, dx=D, dxi=(8, 64))


@pytest.mark.parametrize("change,word", [
    (dict(dtype=9), "dtype"), (dict(tokens=None), "tokens is null"), (dict(m=None), "rowMax"), (dict(s=None), "logSum"), (dict(h=None), "entropy"),
    (dict(g=None, gh=None), "no upstream"), (dict(dxi=(8, 65)), "shape"), (dict(dx=A + 8), "overlaps"), (dict(dx=B), "overlaps"),
    (dict(dx=C), "overlaps"), (dict(scale=float("inf")), "scale"), (dict(xi=(64,), dxi=(64,)), "rank 2"), (dict(g=C + 1028), "aligned"),
])
def test_token_log_probs_gradient(lib, change, word):
    a = dict(LPG, **change)
    rc = lib.nd4jb200_exec_token_log_probs_grad(None, a["dtype"], a["x"], dense(*a["xi"]), a["tokens"], a["scale"], a["m"], a["s"], a["h"],
                                                a["g"], a["gh"], a["dx"], dense(*a["dxi"]))
    refused(lib, rc, word)


def test_embedding(lib):
    def call(dtype=0, table=A, ti=(100, 16), tokens=B, scale=1.0, z=C, zi=(8, 16)):
        return lib.nd4jb200_exec_embedding(None, dtype, table, dense(*ti), tokens, scale, z, dense(*zi))
    refused(lib, call(dtype=4), "dtype")
    refused(lib, call(table=None), "table is null")
    refused(lib, call(tokens=None), "tokens is null")
    refused(lib, call(z=None), "z is null")
    refused(lib, call(scale=float("inf")), "scale")
    refused(lib, call(scale=1e300), "scale")
    refused(lib, call(zi=(8, 17)), "width")
    refused(lib, call(zi=(8, 1, 16)), "rank 2")
    refused(lib, call(z=A + 64), "overlaps")
    refused(lib, call(z=B), "overlaps")
    refused(lib, call(tokens=B + 1), "aligned")


def test_embedding_gradient(lib):
    def call(dtype=2, tokens=B, scale=1.0, dz=C, di=(8, 16), grad=A, gi=(100, 16), accumulate=0):
        return lib.nd4jb200_exec_embedding_grad(None, dtype, tokens, scale, dz, dense(*di), grad, dense(*gi), accumulate)
    refused(lib, call(dtype=4), "dtype")
    refused(lib, call(tokens=None), "tokens is null")
    refused(lib, call(dz=None), "dz is null")
    refused(lib, call(grad=None), "grad is null")
    refused(lib, call(di=(8, 15)), "width")
    refused(lib, call(dz=A + 32), "overlaps")
    refused(lib, call(grad=A + 1), "aligned")
    refused(lib, call(scale=float("nan")), "scale")
    rc = lib.nd4jb200_exec_embedding_grad(None, 0, B, 1.0, C, dense(8, 16), A, strided((100, 16), (0, 1)), 0)
    refused(lib, rc, "stride of 0")


def test_global_norm(lib):
    def pointers(*p):
        a = (ctypes.c_void_p * max(len(p), 1))(*p)
        KEEP.append(a)
        return a

    def clip(dtype=0, x=(A, B), z=(C, D), lengths=(100, 200), n=2, most=1.0, norm=E):
        return lib.nd4jb200_exec_clip_by_global_norm(None, dtype, None if x is None else pointers(*x), None if z is None else pointers(*z),
                                                     None if lengths is None else longs(lengths), n, most, norm)
    refused(lib, clip(dtype=3), "dtype")
    refused(lib, clip(n=-1), "negative")
    refused(lib, clip(x=None), "x is null")
    refused(lib, clip(lengths=None), "lengths is null")
    refused(lib, clip(norm=None), "norm is null")
    refused(lib, clip(norm=E + 2), "aligned")
    refused(lib, clip(most=-1.0), "maxNorm")
    refused(lib, clip(most=float("nan")), "maxNorm")
    refused(lib, clip(most=float("inf")), "maxNorm")
    refused(lib, clip(lengths=(100, -1)), "length")
    refused(lib, clip(x=(A, None)), "null")
    refused(lib, clip(z=(C, None)), "null")
    refused(lib, clip(x=(A, B + 1)), "aligned")
    refused(lib, clip(z=(C, C + 396)), "overlap")               # 100 floats take 400 bytes
    refused(lib, clip(z=(D + 4, D)), "overlap")
    refused(lib, clip(x=(A, A), z=None), "overlap")             # one tensor twice, in place
    refused(lib, clip(z=(A + 4, D)), "overlaps the operand")
    refused(lib, clip(z=(B, A)), "overlaps the operand")
    refused(lib, clip(norm=C + 8), "overlaps")
    rc = lib.nd4jb200_exec_global_norm(None, 0, pointers(A, B), longs((1, 1 << 60)), 2, E)
    refused(lib, rc, "length")


def test_the_mirror_checks_tensors(lib):
    import torch
    ops = native_ops.NativeOps()
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    info = S.shape_info([4, 8])
    for call in (lambda: ops.execLayerNorm(0, None, x, info, None, None, 1e-5, x, info, None, None, [1], 1),
                 lambda: ops.execTokenLogProbs(0, None, x, info, t, 1.0, t, None, None, None),
                 lambda: ops.execEmbedding(0, None, x, info, t, 1.0, x, info),
                 lambda: ops.execGlobalNorm(0, None, [x], [32], 1, x)):
        with pytest.raises(native_ops.Nd4jError, match="not in device memory"):
            call()
    with pytest.raises(native_ops.Nd4jError, match="not a list of axes"):
        ops.execLayerNorm(0, None, A, info, None, None, 1e-5, B, info, None, None, [5], 1)
    with pytest.raises(native_ops.Nd4jError, match="fewer"):
        ops.execGlobalNorm(0, None, [A, B], [3], 2, C)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_the_largest_scale_is_served(lib, dtype):
    # (float) 1e30 is a little above 1e30; the limit is that of the number given. Without rows nothing is launched.
    assert lib.nd4jb200_exec_token_log_probs(None, dtype, A, dense(0, 64), B, 1e30, C, None, None, None, 0, None, None) == 0
    assert lib.nd4jb200_exec_token_log_probs_grad(None, dtype, A, dense(0, 64), B, 1e30, C, D, None, E, None, F, dense(0, 64)) == 0
    refused(lib, lib.nd4jb200_exec_token_log_probs(None, dtype, A, dense(0, 64), B, np.nextafter(1e30, 2e30), C, None, None, None, 0, None,
                                                   None), "scale")


def test_the_mirror_does_not_read_beyond_a_dimension_list(lib):
    ops = native_ops.NativeOps()
    info = S.shape_info([4, 8])
    for dims, length in (([1], 2), ([], 1), ([1], 1 << 30), ([1], -1), (np.array([0, 1], dtype=np.int32), 3)):
        with pytest.raises(native_ops.Nd4jError, match="dimension list holds"):
            ops.execLayerNorm(0, None, A, info, None, None, 1e-5, B, info, None, None, dims, length)
        with pytest.raises(native_ops.Nd4jError, match="dimension list holds"):
            ops.execLayerNormGrad(0, None, A, info, None, B, C, D, info, E, info, None, None, dims, length)
    with pytest.raises(native_ops.Nd4jError, match="dimension list is empty"):
        ops.execLayerNorm(0, None, A, info, None, None, 1e-5, B, info, None, None, [1], 0)


def test_the_other_members_do_not_read_beyond_a_dimension_list_either(lib):
    ops = native_ops.NativeOps()
    info, row = S.shape_info([4, 8]), S.shape_info([1, 8])
    calls = (lambda d, n: ops.execReduceFloat(None, 1, A, info, None, B, row, d, n),
             lambda d, n: ops.execIndexReduceFloat(None, 0, A, info, None, B, row, d, n),
             lambda d, n: ops.execSummaryStatsFloat(None, 0, A, info, None, B, row, d, n, True),
             lambda d, n: ops.execReduce3Float(None, 1, A, info, None, B, info, C, row, d, n),
             lambda d, n: ops._execReduce3All(0, None, 1, A, info, None, B, info, C, info, d, n),
             lambda d, n: ops.execBroadcastFloat(None, 0, A, info, B, row, C, info, d, n),
             lambda d, n: ops.execChain(0, None, 0, A, info, B, row, d, n, 0, None, 0, None, None, None, C, info))
    for call in calls:
        with pytest.raises(native_ops.Nd4jError, match="dimension list holds 1 entries, not 4"):
            call([1], 4)


def test_the_mirror_does_not_read_beyond_a_descriptor(lib):
    ops = native_ops.NativeOps()
    good = S.shape_info([4, 8])
    for bad in (good[:7], list(good[:3]), [], [32] + [1] * 60):
        for call in (lambda: ops.execLayerNorm(0, None, A, bad, None, None, 1e-5, B, bad, None, None, [1], 1),
                     lambda: ops.execLayerNorm(0, None, A, good, None, None, 1e-5, B, bad, None, None, [1], 1),
                     lambda: ops.execLayerNormGrad(0, None, A, good, None, B, C, D, bad, E, good, None, None, [1], 1),
                     lambda: ops.execLayerNormGrad(0, None, A, good, None, B, C, D, good, E, bad, None, None, [1], 1),
                     lambda: ops.execTokenLogProbs(0, None, A, bad, B, 1.0, C, None, None, None),
                     lambda: ops.execTokenLogProbsGrad(0, None, A, good, B, 1.0, C, D, None, E, None, F, bad),
                     lambda: ops.execEmbedding(0, None, A, bad, B, 1.0, C, good),
                     lambda: ops.execEmbedding(0, None, A, good, B, 1.0, C, bad),
                     lambda: ops.execEmbeddingGrad(0, None, A, 1.0, B, bad, C, good),
                     lambda: ops.execEmbeddingGrad(0, None, A, 1.0, B, good, C, bad)):
            with pytest.raises(native_ops.Nd4jError, match="fewer than its rank"):
                call()


# layouts of results: whether two elements share a place is counted out
SHARED = [((4, 8), (7, 1)), ((4, 8), (1, 3)), ((4, 8), (-7, 1)), ((4, 8), (1, 1)), ((4, 8), (6, 4)), ((2, 3, 4), (6, 4, 1)), ((3, 3, 3), (1, 2, 4)),
          ((4, 1, 8), (5, 0, -1))]
APART = [((4, 8), (8, 1)), ((4, 8), (9, 1)), ((4, 8), (1, 4)), ((4, 8), (16, 2)), ((3, 2), (2, 3)), ((2, 2), (3, 2)), ((1, 8), (0, 1)), ((8, 1), (1, 0)),
         ((4, 8), (-8, -1)), ((2, 3, 4), (12, 4, 1)), ((2, 3, 4), (1, 2, 6)), ((7, 5), (5, 7))]


def test_the_layouts_do_and_do_not_share_places():
    for cases, want in ((SHARED, True), (APART, False)):
        for shape, strides in cases:
            places = [sum(i * s for i, s in zip(at, strides)) for at in np.ndindex(*shape)]
            assert (len(set(places)) < len(places)) is want, (shape, strides)


@pytest.mark.parametrize("shape,strides", SHARED)
def test_results_whose_elements_share_their_place(lib, shape, strides):
    last = ints([len(shape) - 1])
    word = "share their place"
    plain, odd = dense(*shape), strided(shape, strides)
    refused(lib, lib.nd4jb200_exec_layer_norm(None, 0, A, plain, None, None, 1e-5, B, odd, None, None, last, 1), word)
    refused(lib, lib.nd4jb200_exec_layer_norm(None, 0, A, odd, None, None, 1e-5, A, odd, None, None, last, 1), word)
    refused(lib, lib.nd4jb200_exec_layer_norm_grad(None, 0, A, plain, None, B, C, D, plain, E, odd, None, None, last, 1), word)
    if len(shape) == 2:
        refused(lib, lib.nd4jb200_exec_token_log_probs_grad(None, 0, A, plain, B, 1.0, C, D, None, E, None, F, odd), word)
        refused(lib, lib.nd4jb200_exec_embedding(None, 0, A, dense(100, shape[1]), B, 1.0, C, odd), word)
        refused(lib, lib.nd4jb200_exec_embedding_grad(None, 0, B, 1.0, C, dense(5, shape[1]), A, odd, 1), word)


@pytest.mark.parametrize("shape,strides", APART)
def test_results_whose_elements_lie_apart(lib, shape, strides):
    # the next check is reached: the statistics stand in the operand
    rc = lib.nd4jb200_exec_layer_norm(None, 0, A, dense(*shape), None, None, 1e-5, B, strided(shape, strides), A, None, ints([len(shape) - 1]), 1)
    refused(lib, rc, "mean overlaps")


def test_overlaps_of_arrays_with_gaps(lib):
    # rows 80 floats apart, of which 64 are the array's: the first and the last element are known to be there
    one, other = strided((8, 64), (80, 1)), strided((8, 64), (72, 1))

    def norm(x=A, xi=one, gain=B, z=C, zi=one, mean=D, eps=1e-5):
        return lib.nd4jb200_exec_layer_norm(None, 0, x, xi, gain, None, eps, z, zi, mean, None, ints([1]), 1)
    refused(lib, norm(z=A, zi=other), "overlaps")                       # the same first element, other rows
    refused(lib, norm(z=A, zi=strided((8, 64), (-80, 1))), "overlaps")  # ... in other directions
    refused(lib, norm(z=A + 4 * 56, zi=other), "overlaps")              # the same last element
    refused(lib, norm(z=A - 4 * 100, zi=dense(8, 64)), "overlaps")      # the first one inside a dense array
    refused(lib, norm(z=A + 4 * 500, zi=dense(8, 64)), "overlaps")      # the last one
    refused(lib, norm(mean=A), "overlaps")
    refused(lib, norm(gain=C + 4 * (7 * 80 + 63)), "overlaps")          # its first value is z's last
    # what may lie in the gaps is let through, up to a check behind these
    beyond = dict(mean=D + 1)
    refused(lib, norm(z=A + 4 * 64, zi=strided((8, 16), (80, 1)), xi=strided((8, 16), (80, 1)), **beyond), "aligned")
    refused(lib, norm(x=A, xi=strided((8, 40), (80, 2)), z=A + 4, zi=strided((8, 40), (80, 2)), **beyond), "aligned")
    rc = lib.nd4jb200_exec_token_log_probs_grad(None, 0, A, one, B, 1.0, C, D, None, E, None, A, other)
    refused(lib, rc, "overlaps")
    rc = lib.nd4jb200_exec_embedding_grad(None, 0, B, 1.0, A + 4 * (7 * 80 + 63), dense(5, 64), A, one, 0)
    refused(lib, rc, "overlaps")
