"""What the tests of the operators between a language model's matrix products share: element types with their unit
roundoffs, shapeInfos of torch views, and views of the layouts that the operators meet."""
import torch

from libnd4j_b200 import shape as S

TYPES = [0, 1, 2]                     # float, double, half, as the calls number them
NAMES = {0: "float", 1: "double", 2: "half"}
KIND = {0: torch.float32, 1: torch.float64, 2: torch.float16}
WIDE = {0: torch.float32, 1: torch.float64, 2: torch.float32}
# half a unit in the last place, relative: of the type that sums are held in, and of the stored type
U = {0: 2.0 ** -24, 1: 2.0 ** -53, 2: 2.0 ** -24}
STORE = {dt: torch.finfo(KIND[dt]).eps / 2 for dt in TYPES}
# the same below the normal range: half the smallest step of the stored type
TINY = {dt: torch.finfo(KIND[dt]).smallest_normal * torch.finfo(KIND[dt]).eps / 2 for dt in TYPES}


def info(t):
    return S.shape_info(t.shape, "c", t.stride())


def place(values, layout):
    """`values` (rank 2) in a view of the layout: dense, rows further apart than long (by an odd number of elements), shifted
    off the 16-byte grid, every second column of a wider array, or columns contiguous."""
    rows, cols = values.shape
    if layout == "dense":
        return values.clone()
    if layout == "apart":
        v = torch.full((rows, cols + 5), 7.0, dtype=values.dtype, device=values.device)[:, :cols]
    elif layout == "shifted":
        v = torch.full((rows * cols + 1,), 7.0, dtype=values.dtype, device=values.device)[1:].view(rows, cols)
    elif layout == "every second":
        v = torch.full((rows, 2 * cols), 7.0, dtype=values.dtype, device=values.device)[:, ::2]
    else:
        assert layout == "columns"
        v = torch.full((cols, rows), 7.0, dtype=values.dtype, device=values.device).t()
    v.copy_(values)
    return v


LAYOUTS = ["dense", "apart", "shifted", "every second", "columns"]


def randn(seed, *shape, dtype=torch.float64):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float64).to(dtype)


def within(got, want, bound):
    """Every element of `got` lies within `bound` of `want` (both compared in 64 bits); equal infinities and NaNs agree."""
    got, want = got.double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = (got - want).abs()
    bad = ~(same | (off <= bound))
    assert not bad.any(), "%d of %d values are off, the worst by %.3g where %.3g is allowed" % (
        int(bad.sum()), bad.numel(), float(off[bad].max()), float(torch.as_tensor(bound, device=off.device).expand_as(off)[bad].min()))


def between(x, outside=7.0):
    """The memory around a view made by `place` still holds what it held."""
    base = x._base if x._base is not None else x
    flat = base.as_strided((base.untyped_storage().nbytes() // base.element_size(),), (1,), 0).clone()
    view = flat.as_strided(x.shape, x.stride(), x.storage_offset())
    view.fill_(outside)
    return bool((flat == outside).all())
