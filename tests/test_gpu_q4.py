"""4-bit matrices on the GPU against the definitions in 64 bits."""
import math

import pytest
import torch

import matxtract_b200 as mx

from conftest import has_gpu
from q4_cases import TINY, U, dense64, entries, make, matrix, rounded, steps64

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not has_gpu(), reason="needs a CUDA device")]

TYPES = [torch.float16, torch.bfloat16]
# rows, columns, group, zero points, density of the residual (None: none)
SHAPES = [(1, 1, 32, True, None), (1, 32, 32, False, 0.2), (3, 33, 32, True, 0.3), (16, 128, 128, False, None),
          (17, 129, 64, True, 0.05), (64, 256, 32, False, 0.02), (130, 320, 96, True, 0.02),
          (128, 1024, 128, False, 0.01), (257, 516, 256, True, 0.01), (40, 2051, 64, True, 0.005),
          (300, 96, 1024, True, 0.05), (33, 4128, 128, False, 0.01)]
VECTORS = [1, 2, 5, 8, 9, 16, 31, 64, 130, 300]


def normal(seed, *shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def close(got, want, allowed):
    off = (got.double() - want).abs()
    bad = ~(off <= allowed)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()} (allowed {allowed[bad][0].item():.3g})")


def weight_roundings(m):
    return 1 if m["residual"] is None else 2


def check_product(m, t, seed, x=None, y=None):
    n, k, dtype = m["n"], m["k"], m["dtype"]
    x = normal(seed, t, k, dtype=dtype) if x is None else x
    y = torch.full((t, n), math.nan, dtype=dtype, device="cuda") if y is None else y
    matrix(m).product(x, y)
    w, xd = dense64(m), x.double()
    close(y, xd @ w.T, rounded(xd @ w.T, xd.abs() @ w.abs().T, k, dtype, weight_roundings(m)))
    return x, y


def check_product_t(m, t, seed, dy=None, dx=None):
    n, k, dtype = m["n"], m["k"], m["dtype"]
    dy = normal(seed, t, n, dtype=dtype) if dy is None else dy
    dx = torch.full((t, k), math.nan, dtype=dtype, device="cuda") if dx is None else dx
    matrix(m).product_t(dy, dx)
    w, dd = dense64(m), dy.double()
    close(dx, dd @ w, rounded(dd @ w, dd.abs() @ w.abs(), n, dtype, weight_roundings(m)))
    return dy, dx


def check_grad(m, t, seed, x=None, dy=None):
    n, k, dtype = m["n"], m["k"], m["dtype"]
    x = normal(seed, t, k, dtype=dtype) if x is None else x
    dy = normal(seed + 1, t, n, dtype=dtype, scale=0.1) if dy is None else dy
    d_scales = torch.full_like(m["scales"], math.nan)
    d_val = torch.full_like(m["residual"][2], 7.0) if m["residual"] is not None else None
    matrix(m).grad(x, dy, d_scales, d_val)
    steps, of = steps64(m)
    g, size = dy.double().T @ x.double(), dy.double().abs().T @ x.double().abs()
    total = lambda a: torch.zeros(m["scales"].shape, dtype=torch.float64, device="cuda").index_add_(1, of, a)  # noqa: E731
    close(d_scales, total(g * steps), rounded(total(g * steps), total(size * steps.abs()), t + m["group"], dtype, 0))
    if d_val is not None:
        row, col, val = entries(m)
        close(d_val[: val.numel()], g[row, col], rounded(g[row, col], size[row, col], t, dtype, 0))
        assert (d_val[val.numel():] == 7.0).all()  # room behind the last entry is left alone
    return x, dy, d_scales, d_val


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_expand(shape, dtype):
    n, k, group, zeros, density = shape
    m = make(n, k, group, dtype, zeros, density, 1)
    big = torch.full((n, k + 3), 9.0, dtype=dtype, device="cuda")
    matrix(m).expand(big[:, :k])
    w = dense64(m)
    # one rounding of the exact sum, which is taken in 32 bits
    close(big[:, :k], w, w.abs() * U[dtype] * 1.01 + w.abs().max() * 2.0 ** -22 + TINY[dtype])
    assert (big[:, k:] == 9.0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_product(shape, dtype):
    for t in VECTORS:
        check_product(make(*shape[:3], dtype, *shape[3:], 2), t, t)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_product_t(shape, dtype):
    for t in VECTORS:
        check_product_t(make(*shape[:3], dtype, *shape[3:], 3), t, t)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_grad(shape, dtype):
    for t in VECTORS:
        check_grad(make(*shape[:3], dtype, *shape[3:], 4), t, t)


@pytest.mark.parametrize("t", [1, 8, 20, 200])
@pytest.mark.parametrize("n,k", [(1500, 640), (512, 4096)])
def test_larger_matrices(n, k, t):
    m = make(n, k, 64, torch.bfloat16, True, 0.005, 8)
    check_product(m, t, 1)
    check_product_t(m, t, 2)
    check_grad(m, t, 3)


@pytest.mark.parametrize("t", [1, 8, 16, 40])
@pytest.mark.parametrize("group", [96, 128, 160, 256, 384, 1024, 1056, 4096])
def test_wide_groups(group, t):
    """Groups that take several tiles of the kernels, whole or not."""
    m = make(140, 8256, group, torch.bfloat16, True, 0.002, group)
    for _ in range(3):
        check_product(m, t, 1)
        check_product_t(m, t, 2)
        check_grad(m, t, 3)


@pytest.mark.parametrize("t", [17, 100, 200, 600])
@pytest.mark.parametrize("n,k", [(200, 8200), (6000, 300), (1300, 5000)])
def test_many_tiles(n, k, t):
    """Contractions many times as long as what is under way at a time, in each width of tile."""
    m = make(n, k, 128, torch.float16, True, 0.004, t)
    for _ in range(3):
        check_product(m, t, 1)
        check_product_t(m, t, 2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,k,group,density", [(4100, 1032, 128, 0.005), (1032, 4100, 32, 0.02), (8200, 520, 96, None),
                                               (4224, 1024, 1024, 0.2), (520, 8200, 64, 0.005)])
def test_large_products(n, k, group, density, dtype):
    """Many tiles of many vectors, with last ones that are cut short in each direction."""
    m = make(n, k, group, dtype, True, density, 5)
    for t in (1030, 1500):
        check_product(m, t, 1)
        check_product_t(m, t, 2)
        check_grad(m, t, 3)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("t", [1, 7, 40, 150])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_strided_vectors(t, dtype, shift):
    """Rows that lie apart, on any border; what lies between them stays."""
    m = make(70, 200, 64, dtype, True, 0.03, 5)
    for pad in (1, 8):
        wide_x = normal(6, t + 1, 200 + pad + shift, dtype=dtype)
        wide_y = torch.full((t + 1, 70 + pad + shift), 9.0, dtype=dtype, device="cuda")
        x, y = wide_x[:t, shift:shift + 200], wide_y[:t, shift:shift + 70]
        check_product(m, t, 0, x, y)
        assert (wide_y[t] == 9).all() and (wide_y[:, :shift] == 9).all() and (wide_y[:, shift + 70:] == 9).all()
        wide_dx = torch.full((t + 1, 200 + pad + shift), 9.0, dtype=dtype, device="cuda")
        dy, dx = normal(7, t + 1, 70 + pad + shift, dtype=dtype)[:t, shift:shift + 70], wide_dx[:t, shift:shift + 200]
        check_product_t(m, t, 0, dy, dx)
        assert (wide_dx[t] == 9).all() and (wide_dx[:, :shift] == 9).all() and (wide_dx[:, shift + 200:] == 9).all()
        check_grad(m, t, 0, x, dy)


@pytest.mark.parametrize("t", [0, 1, 64])
@pytest.mark.parametrize("n,k", [(0, 64), (5, 0), (0, 0), (5, 64)])
def test_empty_sizes(n, k, t):
    m = make(n, k, 32, torch.float16, True, 0.1 if n and k else None, 1)
    q = matrix(m)
    x, y = normal(1, t, k, dtype=torch.float16), torch.full((t, n), 9.0, dtype=torch.float16, device="cuda")
    q.product(x, y)
    dy, dx = normal(2, t, n, dtype=torch.float16), torch.full((t, k), 9.0, dtype=torch.float16, device="cuda")
    q.product_t(dy, dx)
    ds = torch.full_like(m["scales"], 9.0)
    q.grad(x, dy, ds)
    torch.cuda.synchronize()
    if k == 0:
        assert (y == 0).all()
    if n == 0:
        assert (dx == 0).all()
    if t == 0:
        assert (ds == 0).all()  # a sum over no vectors
    w = torch.empty(n, k, dtype=torch.float16, device="cuda")
    q.expand(w)
    q.quantize(w, threshold=1.0)
    q.check()


def test_repeated_columns_add_up():
    m = make(40, 256, 128, torch.float16, False, 0.0, 9)
    col = torch.tensor([0, 0, 5, 5, 5, 255], dtype=torch.int32, device="cuda")
    ptr = torch.zeros(41, dtype=torch.int32, device="cuda")
    ptr[20:] = 6  # row 19 alone
    m["residual"] = (ptr, col, torch.tensor([1, 2, 0.5, 0.25, 4, -3], dtype=torch.float16, device="cuda"))
    w = torch.empty(40, 256, dtype=torch.float16, device="cuda")
    matrix(m).expand(w)
    assert w[19, 5] == dense64(m)[19, 5].half() and w[19, 0] == dense64(m)[19, 0].half()
    for t in (1, 30, 200):
        # up to three roundings of one weight on top of the codes' own
        x = normal(t, t, 256, dtype=torch.float16)
        y = torch.empty(t, 40, dtype=torch.float16, device="cuda")
        matrix(m).product(x, y)
        wd, xd = dense64(m), x.double()
        close(y, xd @ wd.T, rounded(xd @ wd.T, xd.abs() @ (wd.abs().T + 8), 256, torch.float16, 4))
        dy = normal(t, t, 40, dtype=torch.float16)
        dx = torch.empty(t, 256, dtype=torch.float16, device="cuda")
        matrix(m).product_t(dy, dx)
        dd = dy.double()
        close(dx, dd @ wd, rounded(dd @ wd, dd.abs() @ (wd.abs() + 8), 40, torch.float16, 4))
        check_grad(m, t, t)


def test_bad_residuals_are_told_and_stay_in_bounds():
    """Row pointers and columns that point nowhere: refused by check, never followed by the other calls."""
    good = make(50, 300, 64, torch.bfloat16, True, 0.05, 11)
    matrix(good).check()
    ptr, col, val = good["residual"]
    nnz = int(ptr[-1])
    for what in ("column", "negative", "order", "pointer", "decreasing", "past", "start"):
        p, c = ptr.clone(), col.clone()
        if what == "column":
            c[nnz // 2] = 300
        elif what == "negative":
            c[0] = -5
        elif what == "order":
            c[int(p[0])], c[int(p[0]) + 1] = 200, 100
        elif what == "pointer":
            p[20] = 2 ** 30
        elif what == "decreasing":
            p[21] = int(p[20]) - 1
        elif what == "past":
            p[50] = col.numel() + 1
        else:
            p[0] = -7
        m = dict(good, residual=(p, c, val))
        with pytest.raises(mx.MxError) as e:
            matrix(m).check()
        assert e.value.status == 1
        q = matrix(m)
        for t in (1, 20, 140):
            x, dy = normal(1, t, 300, dtype=torch.bfloat16), normal(2, t, 50, dtype=torch.bfloat16)
            y, dx = torch.empty(t, 50, dtype=torch.bfloat16, device="cuda"), torch.empty_like(x)
            q.product(x, y), q.product_t(dy, dx)
            q.grad(x, dy, torch.empty_like(m["scales"]), torch.empty_like(val))
        q.expand(torch.empty(50, 300, dtype=torch.bfloat16, device="cuda"))
        torch.cuda.synchronize()
    # nothing that happened above left a mark on a good matrix
    check_product(good, 20, 1)


# ---- quantise -------------------------------------------------------------------------------------------------------


def fresh(n, k, group, dtype, zeros, cap):
    groups, width = -(-k // group), -(-k // 32) * 16
    m = {"n": n, "k": k, "group": group, "dtype": dtype, "residual": None,
         "codes": torch.full((n, width), 0xAB, dtype=torch.uint8, device="cuda"),
         "scales": torch.zeros(n, groups, dtype=dtype, device="cuda"),
         "zeros": torch.full((n, groups), 99, dtype=torch.uint8, device="cuda") if zeros else None}
    if cap is not None:
        m["residual"] = (torch.full((n + 1,), -1, dtype=torch.int32, device="cuda"),
                         torch.full((cap,), -1, dtype=torch.int32, device="cuda"),
                         torch.full((cap,), 5.0, dtype=dtype, device="cuda"))
    return m


def quantized64(w, group, dtype, zeros, threshold):
    """codes, scales, zero points and the residual by the definition."""
    n, k = w.shape
    w64 = w.double()
    far = w64.abs() > threshold if threshold is not None else torch.zeros_like(w64, dtype=torch.bool)
    near = torch.where(far, 0.0, w64)
    groups = -(-k // group)
    of = torch.arange(k, device="cuda") // group
    padded = torch.zeros(n, groups * group, dtype=torch.float64, device="cuda")
    padded[:, :k] = near
    g = padded.view(n, groups, group)
    lo, hi = g.amin(2).clamp(max=0), g.amax(2).clamp(min=0)
    # the quotient in 32 bits; tensors on both sides, since torch multiplies by the reciprocal of a plain number
    if zeros:
        s = ((hi.float() - lo.float()) / torch.full_like(hi, 15).float()).to(dtype)
        z = torch.where(s > 0, torch.round(-lo / s.double()), 0.0).clamp(0, 15)
    else:
        s = (torch.maximum(hi, -lo).float() / torch.full_like(hi, 7).float()).to(dtype)
        z = torch.full_like(lo, 8.0)
    sk, zk = s.double()[:, of], z[:, of]
    c = (torch.where(sk > 0, torch.round(near / sk), 0.0) + zk).clamp(0 if zeros else 1, 15)
    return c, s, z, far


@pytest.mark.parametrize("source", ["own", "fp32"])
@pytest.mark.parametrize("threshold", [None, 0.0, 1.2, 100.0])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 32, True), (3, 31, 32, False), (9, 65, 32, True), (20, 200, 96, False),
                                   (65, 1024, 128, True), (33, 771, 256, False), (130, 96, 1024, True),
                                   (70, 4100, 64, True)], ids=str)
def test_quantize(shape, dtype, threshold, source):
    n, k, group, zeros = shape
    w = normal(3, n, k + 5, dtype=torch.float32 if source == "fp32" else dtype)[:, 2:k + 2]
    w[:, ::7] = 0
    if n > 2:
        w[2] = 0  # a row without anything
        w[1] = w[1].abs() * (1 if zeros else -1)  # all of one sign
    cap = n * k + 3 if threshold is not None else None
    m = fresh(n, k, group, dtype, zeros, cap)
    q = matrix(m)
    q.quantize(w, threshold=threshold)
    q.check()
    c, s, z, far = quantized64(w, group, dtype, zeros, threshold)
    assert torch.equal(m["scales"], s)
    if zeros:
        assert torch.equal(m["zeros"].double(), z)
    raw = m["codes"].long()
    got = torch.stack([raw % 16, raw // 16], 2).reshape(n, -1)
    assert torch.equal(got[:, :k].double(), c)
    assert (raw[:, (k + 1) // 2:] == 0xAB).all()  # bytes behind the last code are left alone
    if threshold is not None:
        ptr, col, val = m["residual"]
        row, column = far.nonzero(as_tuple=True)
        nnz = row.numel()
        assert torch.equal(ptr[1:].long(), far.sum(1).cumsum(0)) and ptr[0] == 0
        assert torch.equal(col[:nnz].long(), column) and torch.equal(val[:nnz], w[row, column].to(dtype))
        assert (col[nnz:] == -1).all() and (val[nnz:] == 5.0).all()
    # every entry that stayed is at most half a step away, and at most what the scale's own rounding adds at the ends
    err = (dense64(m) - w.double()).abs()
    of = torch.arange(k, device="cuda") // group
    step = s.double()[:, of]
    assert (err <= 0.5 * step + 16 * step * U[dtype] + w.double().abs() * U[dtype] + TINY[dtype]).all()


def test_quantize_borders():
    """Quotients that are exactly half-way go to the even number, and 32-bit values next to the border to their side."""
    s = 0.5
    vals = torch.tensor([7 * s] + [(i + 0.5) * s for i in range(-7, 7)] + [0.0], dtype=torch.float32, device="cuda")
    up, down = torch.nextafter(vals, torch.tensor(9.0, device="cuda")), torch.nextafter(vals, torch.tensor(-9.0, device="cuda"))
    up[0] = down[0] = 7 * s
    for v in (vals, up, down):
        w = torch.zeros(1, 32, dtype=torch.float32, device="cuda")
        w[0, :16] = v
        m = fresh(1, 32, 32, torch.bfloat16, False, None)
        matrix(m).quantize(w)
        c, sc, _, _ = quantized64(w, 32, torch.bfloat16, False, None)
        assert sc[0, 0] == s and torch.equal(m["scales"], sc)
        raw = m["codes"].long()
        assert torch.equal(torch.stack([raw % 16, raw // 16], 2).reshape(1, -1).double(), c)


def test_quantize_without_room_keeps_what_fits():
    w = normal(5, 30, 200, dtype=torch.float16)
    full, short = fresh(30, 200, 64, torch.float16, True, 6000), fresh(30, 200, 64, torch.float16, True, 700)
    for m in (full, short):
        matrix(m).quantize(w, threshold=0.5)
    nnz = int(full["residual"][0][-1])
    assert nnz > 700 and torch.equal(full["residual"][0], short["residual"][0])  # the true count is told
    assert torch.equal(full["residual"][1][:700], short["residual"][1])
    assert torch.equal(full["residual"][2][:700], short["residual"][2])
    with pytest.raises(mx.MxError):
        matrix(short).check()


def test_quantize_values_that_are_not_finite():
    """A group that holds a NaN or an infinity says so in its scale and nowhere else; infinities may be outliers."""
    w = normal(6, 4, 128, dtype=torch.bfloat16)
    w[1, 40], w[2, 70] = math.nan, math.inf
    for zeros in (False, True):
        m = fresh(4, 128, 32, torch.bfloat16, zeros, None)
        matrix(m).quantize(w)
        bad = torch.zeros(4, 4, dtype=torch.bool, device="cuda")
        bad[1, 1] = bad[2, 2] = True
        assert torch.equal(~m["scales"].isfinite(), bad) and m["scales"][1, 1].isnan() and m["scales"][2, 2].isinf()
    m = fresh(4, 128, 32, torch.bfloat16, True, 50)
    matrix(m).quantize(w, threshold=100.0)
    assert m["residual"][0].tolist() == [0, 0, 0, 1, 1] and m["residual"][2][0].isinf()
    assert m["scales"][2].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_quantize_tiny_and_huge_values(dtype):
    for scale in (1e-7, 1e-30, 6e4, 1e30):
        w = normal(7, 6, 64, dtype=torch.float32, scale=scale)
        m = fresh(6, 64, 32, dtype, True, None)
        matrix(m).quantize(w)
        c, s, z, _ = quantized64(w, 32, dtype, True, None)
        assert torch.equal(m["scales"], s)
        ok = s.isfinite()
        assert torch.equal(m["zeros"].double()[ok], z[ok])


# ---- as they are used together --------------------------------------------------------------------------------------


def test_they_work_together():
    """Quantise a layer, run it, take every gradient, and step the scales and outliers against a target."""
    n, k, t = 192, 512, 48
    w = normal(1, n, k, dtype=torch.bfloat16, scale=0.05)
    m = fresh(n, k, 64, torch.bfloat16, True, n * k // 20)
    q = matrix(m)
    q.quantize(w, threshold=0.14)
    q.check()
    nnz = int(m["residual"][0][-1])
    assert 0 < nnz < n * k // 20
    dense = torch.empty_like(w)
    q.expand(dense)
    x = normal(2, t, k, dtype=torch.bfloat16)
    y = torch.empty(t, n, dtype=torch.bfloat16, device="cuda")
    q.product(x, y)
    size = x.double().abs() @ dense.double().abs().T
    # y and x times the expanded matrix: the expanded weights are rounded once, so may be the product's
    close(y, x.double() @ dense.double().T, rounded(x.double() @ dense.double().T, size, k, torch.bfloat16, 3))
    dy = ((y.float() - (x.float() @ w.float().T)) / t).to(torch.bfloat16)
    check_product_t(m, t, 0, dy)
    check_grad(m, t, 0, x, dy)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("group", [32, 64, 96])
@pytest.mark.parametrize("k", [128, 416, 448, 480, 512])
def test_numbers_on_any_border(k, group, shift):
    """Rows of scales and zero points of any length, from an address of any alignment."""
    n, groups = 150, -(-k // group)
    m = make(n, k, group, torch.float16, True, 0.01, k)
    for name in ("scales", "zeros"):
        room = torch.empty(n * groups + shift, dtype=m[name].dtype, device="cuda")
        moved = room[shift:].view(n, groups)
        moved.copy_(m[name])
        m[name] = moved
    for t in (1, 8, 12, 40, 130):
        check_product(m, t, 1)
        check_product_t(m, t, 2)
        check_grad(m, t, 3)


def test_calls_behind_one_another():
    """Calls that start while the one in front still runs see what it writes: vectors and workspaces of each are made anew."""
    n, k = 517, 1037  # rows on no 16-byte border: every call copies its vectors first
    m = make(n, k, 64, torch.bfloat16, True, 0.01, 23)
    q = matrix(m)
    for t in (3, 30, 300):
        x0 = normal(1, t, k, dtype=torch.bfloat16, scale=0.1)

        def chain(pause):
            x, seen = x0.clone(), []
            for _ in range(6):
                y, ds = torch.empty(t, n, dtype=torch.bfloat16, device="cuda"), torch.empty_like(m["scales"])
                dv = torch.zeros_like(m["residual"][2])
                for call in (lambda: q.product(x, y), lambda: q.grad(x, y, ds, dv), lambda: q.product_t(y, x)):
                    call()
                    if pause:
                        torch.cuda.synchronize()
                x = x / x.float().abs().max().to(torch.bfloat16)
                seen += [y, ds, dv, x]
            torch.cuda.synchronize()
            return seen

        for a, b in zip(chain(True), chain(False)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_changed_numbers_count():
    """Nothing of a matrix is kept from one call for the next."""
    m = make(300, 640, 32, torch.float16, True, 0.02, 24)
    q = matrix(m)
    for t in (2, 40, 1100):
        x, y = normal(t, t, 640, dtype=torch.float16), torch.empty(t, 300, dtype=torch.float16, device="cuda")
        q.product(x, y)
        m["scales"].mul_(2)
        m["codes"].copy_(m["codes"].flip(0))
        m["residual"][2].mul_(-1)
        check_product(m, t, t, x, y)
        check_product_t(m, t, t)
        check_grad(m, t, t)


def test_codes_of_more_than_two_gigabytes():
    """The last rows of a matrix whose codes and values lie further off than 32 bits count."""
    n, k, last, dtype = 70000, 65536, 96, torch.bfloat16
    m = make(1, 64, 128, dtype, True, None, 25)
    codes = torch.randint(0, 2 ** 31 - 1, (n, k // 8), dtype=torch.int32, device="cuda").view(torch.uint8)
    scales = torch.rand(n, k // 128, device="cuda").add_(0.01).to(dtype)
    zeros = torch.randint(0, 16, (n, k // 128), dtype=torch.uint8, device="cuda")
    ptr = torch.arange(0, 2 * n + 2, 2, dtype=torch.int32, device="cuda")
    col = torch.randint(0, k // 2, (n, 2), dtype=torch.int32, device="cuda")
    col[:, 1] += k // 2
    val = normal(26, 2 * n, dtype=dtype)
    m.update(n=n, k=k, codes=codes, scales=scales, zeros=zeros, residual=(ptr, col.view(-1), val))
    end = dict(m, n=last, codes=codes[-last:], scales=scales[-last:], zeros=zeros[-last:],
               residual=(ptr[: last + 1], col.view(-1)[-2 * last:], val[-2 * last:]))
    q, w = matrix(m), dense64(end)
    for t in (2, 40, 300):
        x, y = normal(t, t, k, dtype=dtype), torch.empty(t, n, dtype=dtype, device="cuda")
        q.product(x, y)
        xd = x.double()
        close(y[:, -last:], xd @ w.T, rounded(xd @ w.T, xd.abs() @ w.abs().T, k, dtype, 2))
        dy, dx = torch.zeros_like(y), torch.empty_like(x)
        dy[:, -last:] = normal(t + 1, t, last, dtype=dtype)
        q.product_t(dy, dx)
        dd = dy[:, -last:].double()
        close(dx, dd @ w, rounded(dd @ w, dd.abs() @ w.abs(), n, dtype, 2))
        ds, dv = torch.empty_like(scales), torch.empty_like(val)
        q.grad(x, dy, ds, dv)
        steps, _ = steps64(end)
        g, size = dd.T @ xd, dd.abs().T @ xd.abs()
        sums = lambda a: a.view(last, -1, 128).sum(2)  # noqa: E731
        close(ds[-last:], sums(g * steps), rounded(sums(g * steps), sums(size * steps.abs()), t + 128, dtype, 0))
        row, at, _ = entries(end)
        close(dv[-2 * last:], g[row, at], rounded(g[row, at], size[row, at], t, dtype, 0))
    del x, y, dy, dx, ds, dv
    dense = torch.empty(n, k, dtype=dtype, device="cuda")
    q.expand(dense)
    close(dense[-last:], w, w.abs() * U[dtype] * 1.01 + TINY[dtype])
    codes.zero_()
    val.zero_()
    q.quantize(dense, threshold=1e30)
    assert int(ptr[-1]) == 0
    # a group reaches over 15 of its old steps at most, so the new step is no larger; half a step is the code's rounding,
    # half the zero point's, and the step's own rounding makes 15 x 2^-8 of one
    close(dense[-last:], dense64(dict(end, residual=None)), 1.07 * scales[-last:].double().repeat_interleave(128, 1))


def test_captured_and_replayed():
    m = make(200, 384, 128, torch.float16, True, 0.02, 21)
    q = matrix(m)
    for t in (1, 24, 160):
        x, dy = normal(1, t, 384, dtype=torch.float16), normal(2, t, 200, dtype=torch.float16)
        out = [torch.zeros(t, 200, dtype=torch.float16, device="cuda"), torch.zeros_like(x),
               torch.zeros_like(m["scales"]), torch.zeros_like(m["residual"][2])]

        def run(stream):
            q.product(x, out[0], stream=stream)
            q.product_t(dy, out[1], stream=stream)
            q.grad(x, dy, out[2], out[3], stream=stream)

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(torch.cuda.current_stream().cuda_stream)
        x.copy_(normal(3, t, 384, dtype=torch.float16))
        dy.copy_(normal(4, t, 200, dtype=torch.float16))
        graph.replay()
        torch.cuda.synchronize()
        seen = [o.clone() for o in out]
        run(0)
        torch.cuda.synchronize()
        for a, b in zip(seen, out):
            assert torch.equal(a, b)
        check_product(m, t, 0, x)


@pytest.mark.parametrize("t", [0, 1, 12, 40, 300])
def test_either_gradient_alone(t):
    m = make(300, 640, 96, torch.float16, True, 0.02, 28)
    x, dy, ds, dv = check_grad(m, t, 1) if t else (torch.empty(0, 640, dtype=torch.float16, device="cuda"),
                                                   torch.empty(0, 300, dtype=torch.float16, device="cuda"),
                                                   torch.zeros_like(m["scales"]), None)
    if t == 0:
        dv = torch.full_like(m["residual"][2], 7.0)
        dv[: int(m["residual"][0][-1])] = 0
    alone, other = torch.full_like(ds, math.nan), torch.full_like(dv, 7.0)
    matrix(m).grad(x, dy, alone)
    matrix(m).grad(x, dy, None, other)
    assert torch.equal(alone, ds) and torch.equal(other, dv)


FIRST_CALL = """
import sys
sys.path[:0] = [{tests!r}, {root!r}]
import torch
from q4_cases import make, matrix
m = make(200, 384, 128, torch.float16, True, 0.02, 21)
q, op, t = matrix(m), {op!r}, {t}
x, dy = (torch.randn(t, c, device="cuda").half() for c in (384, 200))
w, ds, dv = torch.randn(200, 384, device="cuda"), torch.empty_like(m["scales"]), torch.empty_like(m["residual"][2])
calls = dict(product=lambda s: q.product(x, dy, stream=s), product_t=lambda s: q.product_t(dy, x, stream=s),
             grad=lambda s: q.grad(x, dy, ds, dv, stream=s), quantize=lambda s: q.quantize(w, 2.5, stream=s))
outputs = dict(product=dy, product_t=x, grad=ds, quantize=m["scales"])
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls[op](torch.cuda.current_stream().cuda_stream)
outputs[op].zero_()
graph.replay()
torch.cuda.synchronize()
seen = outputs[op].clone()
calls[op](0)
torch.cuda.synchronize()
assert torch.equal(seen, outputs[op]) and seen.abs().max() > 0
"""


@pytest.mark.parametrize("op,t", [("product", 1), ("product", 40), ("product_t", 3), ("grad", 4), ("grad", 40), ("quantize", 1)])
def test_a_process_first_call_may_be_captured(op, t):
    import os
    import subprocess
    import sys

    tests = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL.format(tests=tests, root=os.path.dirname(tests), op=op, t=t)],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_two_graphs_at_once():
    """Graphs of calls that need workspaces (vectors on no 16-byte border, a residual), replayed on two streams together."""
    n, k = 517, 1037
    m = make(n, k, 64, torch.bfloat16, True, 0.01, 27)
    q, graphs = matrix(m), []
    for t in (3, 21, 300):
        x, dy = normal(t, t, k, dtype=torch.bfloat16), normal(t + 1, t, n, dtype=torch.bfloat16)
        out = [torch.empty(t, n, dtype=torch.bfloat16, device="cuda"), torch.empty_like(x), torch.empty_like(m["scales"]),
               torch.zeros_like(m["residual"][2])]

        def run(stream, x=x, dy=dy, out=out):
            q.product(x, out[0], stream=stream)
            q.product_t(dy, out[1], stream=stream)
            q.grad(x, dy, out[2], out[3], stream=stream)

        run(0)
        torch.cuda.synchronize()
        want = [o.clone() for o in out]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(torch.cuda.current_stream().cuda_stream)
        graphs.append((graph, torch.cuda.Stream(), out, want, x, dy))  # which the graph reads
    for _ in range(10):
        for _, _, out, *_ in graphs:
            for o in out:
                o.zero_()
        torch.cuda.synchronize()
        for graph, stream, *_ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out, want, *_ in graphs:
            for o, w in zip(out, want):
                assert torch.equal(o.view(torch.int16), w.view(torch.int16))


def test_streams_do_not_disturb_each_other():
    m = make(500, 1024, 64, torch.bfloat16, True, 0.01, 22)
    q = matrix(m)
    jobs = []
    for i, t in enumerate((1, 3, 33, 200)):
        x, dy = normal(i, t, 1024, dtype=torch.bfloat16), normal(i + 9, t, 500, dtype=torch.bfloat16)
        jobs.append((x, dy, torch.empty(t, 500, dtype=torch.bfloat16, device="cuda"), torch.empty_like(x),
                     torch.empty_like(m["scales"])))
    want = []
    for x, dy, y, dx, ds in jobs:
        q.product(x, y), q.product_t(dy, dx), q.grad(x, dy, ds)
        want.append([y.clone(), dx.clone(), ds.clone()])
        y.zero_(), dx.zero_(), ds.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(5):
        for s, (x, dy, y, dx, ds) in zip(streams, jobs):
            q.product(x, y, stream=s.cuda_stream)
            q.product_t(dy, dx, stream=s.cuda_stream)
            q.grad(x, dy, ds, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for (x, dy, y, dx, ds), w in zip(jobs, want):
        assert torch.equal(y, w[0]) and torch.equal(dx, w[1]) and torch.equal(ds, w[2])


def test_refusals_on_the_gpu():
    m = make(20, 96, 32, torch.float16, True, 0.1, 30)
    q = matrix(m)
    h = torch.float16
    x, y = normal(1, 3, 96, dtype=h), torch.empty(3, 20, dtype=h, device="cuda")
    for bad in (lambda: q.product(x[:, :95], y), lambda: q.product(x, y[:2]), lambda: q.product(x.float(), y),
                lambda: q.product(x.cpu(), y), lambda: q.product(x.T.contiguous().T, y),
                lambda: q.product(x[:1].expand(3, 96), y), lambda: q.product_t(y, x[:2]),
                lambda: q.grad(x, y, m["scales"][:, :1]), lambda: q.grad(x, y, None, m["residual"][2][:-1]),
                lambda: q.expand(y), lambda: q.quantize(x), lambda: q.quantize(torch.zeros(20, 96, device="cuda")),
                lambda: mx.Q4Matrix(20, 96, 32, m["codes"][:, :40], m["scales"]),
                lambda: mx.Q4Matrix(20, 96, 32, m["codes"], m["scales"], zeros=m["zeros"].int()),
                lambda: mx.Q4Matrix(20, 96, 32, m["codes"], m["scales"], res_row_ptr=m["residual"][0])):
        with pytest.raises(mx.MxError) as e:
            bad()
        assert e.value.status == 1
    q.product(x, y)
    torch.cuda.synchronize()
