"""4-bit matrices on the GPU: numbers at the ends of their types, and what lies behind a matrix's last column."""
import math
import threading

import pytest
import torch

import matxtract_b200 as mx

from conftest import has_gpu
from q4_cases import dense64, entries, make, matrix, rounded
from test_gpu_q4 import TYPES, check_grad, check_product, check_product_t, close, fresh, normal

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not has_gpu(), reason="needs a CUDA device")]

# vectors, rows: few vectors, two widths of tile, pairs of blocks
FORMS = [(1, 40), (8, 300), (9, 40), (40, 300), (1100, 40), (1100, 4100)]


# ---- columns behind the last ----------------------------------------------------------------------------------------


def finite_product(m, t, scale):
    """The product with vectors of about `scale`, whose results and weights are all far from the type's ends."""
    n, k, dtype = m["n"], m["k"], m["dtype"]
    x = normal(t, t, k, dtype=torch.float32).mul_(scale).to(dtype)
    y = torch.full((t, n), math.nan, dtype=dtype, device="cuda")
    matrix(m).product(x, y)
    w, xd = dense64(m), x.double()
    want = xd @ w.T
    assert w.abs().max() < torch.finfo(dtype).max and want.abs().max() < torch.finfo(dtype).max / 2
    assert y.isfinite().all()
    close(y, want, rounded(want, xd.abs() @ w.abs().T, k, dtype, 1 if m["residual"] is None else 2))


@pytest.mark.parametrize("t,n", FORMS)
@pytest.mark.parametrize("k", [33, 96, 127, 1037])
def test_the_largest_weights_of_a_last_group(k, t, n):
    """A weight near the type's end makes a scale whose eightfold is no number of the type: no code is 8 below its zero
    point, but the bytes behind the last column may be."""
    w = normal(k, n, k, dtype=torch.float32).mul_(1e4).clamp_(-6e4, 6e4).half()
    w[:, k - 1] = 65472
    for fill in (0x00, 0xFF):
        m = fresh(n, k, 32, torch.float16, False, None)
        m["codes"].fill_(fill)
        matrix(m).quantize(w)
        finite_product(m, t, 1e-4)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("t,n", FORMS)
@pytest.mark.parametrize("k,group", [(33, 64), (96, 96), (1037, 32), (1037, 128), (1037, 2048)])
def test_any_codes_behind_the_last_column(k, group, t, n, dtype):
    """Codes up to 7 stand for numbers of the type, those behind the last column do not."""
    m = make(n, k, group, dtype, True, 0.01, k)
    s = 4900.0 if dtype is torch.float16 else 2.5e37
    m["scales"].fill_(s)
    m["zeros"].zero_()
    m["codes"].bitwise_and_(0x77)
    m["codes"][:, (k + 1) // 2:] = 0xFF
    if k % 2:
        m["codes"][:, k // 2] |= 0xF0
    if m["residual"] is not None:
        m["residual"][2].mul_(s / 4)
    finite_product(m, t, (0.5 if dtype is torch.float16 else 25) / s)


# ---- a weight that a code and a residual's entries share is rounded once ---------------------------------------------


def products_with_unit_vectors(m, t):
    """W by mx_q4_expand, and by products and transposed products with unit vectors, t of them a call: W's own values."""
    n, k, dtype = m["n"], m["k"], m["dtype"]
    w = torch.empty(n, k, dtype=dtype, device="cuda")
    q = matrix(m)
    q.expand(w)
    assert w.isfinite().all()
    rows, cols = torch.empty_like(w), torch.empty_like(w)
    for size, call, out in ((k, q.product, cols.T), (n, q.product_t, rows)):
        unit = torch.eye(size, dtype=dtype, device="cuda")
        for i in range(0, size, t):
            got = torch.empty(min(t, size - i), n + k - size, dtype=dtype, device="cuda")
            call(unit[i:i + t], got)
            out[i:i + t] = got
    return w, cols, rows


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("t,n,k,group,density", [
    (3, 60, 330, 32, 0.02), (40, 60, 330, 32, 0.02), (70, 130, 330, 96, 0.3), (300, 300, 1037, 128, 0.01),
    (1100, 4100, 1100, 64, 0.02), (2300, 1037, 2300, 128, 0.1)])
def test_products_take_the_expanded_weights(t, n, k, group, density, dtype):
    """More than 8 vectors, and transposed products with a residual, multiply by what mx_q4_expand gives, bit for bit."""
    m = make(n, k, group, dtype, True, density, t)
    w, cols, rows = products_with_unit_vectors(m, t)
    if t > 8:
        assert torch.equal(cols, w)
    assert torch.equal(rows, w)


@pytest.mark.parametrize("repeats", [1, 2, 7])
@pytest.mark.parametrize("t", [5, 40, 1100])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_residual_entry_that_cancels_a_code(dtype, t, repeats):
    """Little is left of a code's value and an entry (or several of one column), and a code's value alone may be no number
    of the type: 7 x 143 = 1001 and about -994; 7 x 10000 and about -10000 in fp16."""
    n, k = (4100 if t > 1000 else 300), 1100
    s, parts = (10000.0, -10000.0) if dtype is torch.float16 else (143.0, -994.0)
    m = make(n, k, 64, dtype, False, 0.0, 7)
    m["codes"].fill_(0x88)  # nothing
    m["scales"].fill_(s)
    at = torch.arange(n, device="cuda") * 37 % (k - 1)
    m["codes"].view(n, -1)[torch.arange(n, device="cuda"), at // 2] = 0xFF  # 7 steps at `at` and beside it
    pair = (at // 2 * 2)[:, None] + torch.tensor([0, 1], device="cuda")
    col = pair.repeat_interleave(repeats, 1).int().reshape(-1)
    val = torch.full((col.numel(),), parts / repeats, dtype=dtype, device="cuda")
    ptr = torch.arange(n + 1, dtype=torch.int32, device="cuda") * 2 * repeats
    m["residual"] = (ptr, col, val)
    exact = dense64(m)
    w, cols, rows = products_with_unit_vectors(m, t)
    assert torch.equal(w, exact.to(dtype)) and w.abs().max() > 0
    assert torch.equal(rows, w)
    assert torch.equal(cols, w)  # up to 8 vectors: codes and entries each exact in 32 bits


# ---- groups that are wider than the matrix --------------------------------------------------------------------------


@pytest.mark.parametrize("t", [1, 8, 9, 16, 40])
@pytest.mark.parametrize("k,group", [(300, 320), (300, 4096), (300, 1 << 20), (1100, 1024), (2500, 1 << 30), (40, 1 << 30),
                                     (1290, 640), (1400, 288)])
def test_groups_that_reach_behind_the_last_column(k, group, t):
    m = make(140, k, group, torch.bfloat16, True, 0.02, k)
    check_product(m, t, 1)
    check_product_t(m, t, 2)
    check_grad(m, t, 3)
    w = normal(4, 140, k, dtype=torch.bfloat16)
    q = [matrix(fresh(140, k, g, torch.bfloat16, True, None)) for g in (group, -(-k // 32) * 32)]
    for one in q:
        one.quantize(w)
    if k <= group:
        assert torch.equal(q[0].codes, q[1].codes) and torch.equal(q[0].scales, q[1].scales)


@pytest.mark.parametrize("t", [1, 16])
def test_gradients_cost_what_the_columns_do(t):
    """A group that says "the whole row" by a large number is worked on as far as the row goes."""
    took, seen = [], []
    for group in (320, 1 << 20):
        m = make(140, 300, group, torch.bfloat16, True, None, 1)
        q, ds = matrix(m), torch.empty_like(m["scales"])
        x, dy = normal(1, t, 300, dtype=torch.bfloat16), normal(2, t, 140, dtype=torch.bfloat16)
        for _ in range(3):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            q.grad(x, dy, ds)
            b.record()
            b.synchronize()
        took.append(a.elapsed_time(b))
        seen.append(ds)
    assert torch.equal(*seen)
    assert took[1] < 0.5 + 5 * took[0]  # 3 tiles of 128 columns, not 8192: some 4 ms


# ---- sizes whose products pass 32 bits ------------------------------------------------------------------------------


def test_no_vectors_and_very_many_rows():
    """Sums over no vectors are 0 in the last of 2^27 rows and more, too."""
    n = (1 << 27) + 300
    codes = torch.empty(n, 16, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n, 1, dtype=torch.float16, device="cuda")
    ptr = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    col, val = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.float16, device="cuda")
    q = mx.Q4Matrix(n, 1, 32, codes, scales, res_row_ptr=ptr, res_col_ind=col, res_val=val)
    ds, dv = torch.full_like(scales, 7.0), torch.full_like(val, 7.0)
    none = torch.empty(0, 1, dtype=torch.float16, device="cuda")
    q.grad(none, torch.empty(0, n, dtype=torch.float16, device="cuda"), ds, dv)
    assert not ds.any() and not dv.any()


def test_quantize_counts_that_pass_32_bits():
    """Eight rows of 2^29 outliers each: the counts behind them stand at their limit, and none begins anew."""
    k = 1 << 29
    w = torch.ones(9, k, dtype=torch.float16, device="cuda")
    w[8] = 2
    m = fresh(9, k, k, torch.float16, False, 64)
    matrix(m).quantize(w, threshold=0.5)
    ptr, col, val = m["residual"]
    assert ptr.tolist() == [0] + [min(i * k, 2 ** 31 - 1) for i in range(1, 10)]
    assert torch.equal(col, torch.arange(64, dtype=torch.int32, device="cuda")) and (val == 1).all()
    assert not m["scales"].any() and (m["codes"] == 0x88).all()


def test_a_residual_at_the_far_end_of_its_buffers():
    """Entries' places up to 2^31 - 2, the last that there are: the same results as at the buffers' front."""
    n, k, room, dtype = 140, 8400, 2 ** 31 - 1, torch.bfloat16
    near = make(n, k, 64, dtype, True, 0.02, 41, spare=0)
    ptr, col, val = near["residual"]
    nnz = col.numel()
    far = dict(near, residual=(ptr + (room - nnz), torch.empty(room, dtype=torch.int32, device="cuda"),
                               torch.empty(room, dtype=dtype, device="cuda")))
    far["residual"][1][room - nnz:] = col
    far["residual"][2][room - nnz:] = val
    a, b = matrix(near), matrix(far)
    d_near, d_far = torch.empty_like(val), torch.empty(room, dtype=dtype, device="cuda")
    for t in (0, 1, 8, 12, 40, 1100):
        x, dy = normal(t, t, k, dtype=dtype), normal(t + 1, t, n, dtype=dtype)
        seen = []
        for q, dv in ((a, d_near), (b, d_far)):
            y, dx, ds = torch.empty_like(dy), torch.empty_like(x), torch.empty_like(near["scales"])
            dv[-nnz:] = 7.0
            q.product(x, y), q.product_t(dy, dx), q.grad(x, dy, ds, dv)
            w = torch.empty(n, k, dtype=dtype, device="cuda")
            q.expand(w)
            seen.append((y, dx, ds, dv[-nnz:], w))
        for one, other in zip(*seen):
            assert torch.equal(one, other)


# ---- waits that ran out -----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_a_wait_that_ran_out_is_told_once(which):
    """By the next check on the GPU, which goes on to tell of a bad residual afterwards; results that follow are right."""
    good = make(50, 300, 64, torch.bfloat16, True, 0.05, 11)
    matrix(good).check()
    ptr, col, val = good["residual"]
    bad = matrix(dict(good, residual=(ptr, col.clone().index_fill_(0, torch.tensor([3], device="cuda"), 300), val)))

    def status(q):
        try:
            q.check()
        except mx.MxError as e:
            return e.status
        return 0

    assert mx.lib().mx_q4_wait_in_vain(0, which, 100, None) == 0
    assert [status(matrix(good)) for _ in range(2)] == [6, 0]
    assert mx.lib().mx_q4_wait_in_vain(0, which, 1, torch.cuda.current_stream().cuda_stream) == 0
    assert [status(bad) for _ in range(2)] == [6, 1]
    assert status(matrix(good)) == 0
    check_product(good, 12, 1)


def test_a_wait_ends_within_seconds():
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    assert mx.lib().mx_q4_wait_in_vain(0, 1, 0, torch.cuda.current_stream().cuda_stream) == 0
    b.record()
    b.synchronize()
    m = make(50, 300, 64, torch.bfloat16, True, 0.05, 11)
    with pytest.raises(mx.MxError) as e:
        matrix(m).check()
    assert e.value.status == 6 and 100 < a.elapsed_time(b) < 8000


# ---- values that are not finite -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("group", [32, 64, 96, 128, 4096])
@pytest.mark.parametrize("t,n", [(2, 150), (7, 150), (9, 150), (16, 150), (40, 300), (1100, 4100)])
def test_values_that_are_not_finite_stay_where_they_belong(t, n, group):
    """A NaN or an infinity in one vector, one row's numbers or one entry shows in what it enters and changes nothing else."""
    k, i, j, v = 710, 77, 333, t - 1  # a row, a column, a vector
    m = make(n, k, group, torch.bfloat16, True, 0.02, 3)
    q = matrix(m)
    x, dy = normal(1, t, k, dtype=torch.bfloat16), normal(2, t, n, dtype=torch.bfloat16)
    row, col, val = entries(m)

    def run(x=x, dy=dy):
        y, dx = torch.empty_like(dy), torch.empty_like(x)
        ds, dv = torch.empty_like(m["scales"]), torch.empty_like(m["residual"][2])
        q.product(x, y), q.product_t(dy, dx), q.grad(x, dy, ds, dv)
        return y, dx, ds, dv[: val.numel()]

    def only(got, want, hit):
        hit = hit.expand_as(want)
        assert not got[hit].isfinite().any() and torch.equal(got[~hit], want[~hit])

    def mask(size, at):
        return torch.arange(size, device="cuda") == at

    clean = run()
    groups = torch.arange(m["scales"].shape[1], device="cuda")
    for bad in (math.nan, math.inf, -math.inf):
        x2, dy2 = x.clone(), dy.clone()
        x2[v, j] = bad
        y, _, ds, dv = run(x=x2)
        only(y, clean[0], mask(t, v)[:, None])
        # G's column j: all rows' sums of that group but where every code in it is its zero point, which NaN turns up in too
        only(ds, clean[2], (groups == j // group)[None])
        only(dv, clean[3], col == j)
        dy2[v, i] = bad
        _, dx, ds, dv = run(dy=dy2)
        only(dx, clean[1], mask(t, v)[:, None])
        only(ds, clean[2], mask(n, i)[:, None])
        only(dv, clean[3], row == i)
        # the row's scale of that group
        was = m["scales"][i, j // group].clone()
        m["scales"][i, j // group] = bad
        y, dx, ds, dv = run()
        m["scales"][i, j // group] = was
        only(y, clean[0], mask(n, i)[None])
        only(dx, clean[1], (torch.arange(k, device="cuda") // group == j // group)[None])
        assert torch.equal(ds, clean[2]) and torch.equal(dv, clean[3])
        # an entry
        e = val.numel() // 2
        was = m["residual"][2][e].clone()
        m["residual"][2][e] = bad
        y, dx, ds, dv = run()
        m["residual"][2][e] = was
        only(y, clean[0], mask(n, row[e])[None])
        only(dx, clean[1], mask(k, col[e])[None])
        assert torch.equal(ds, clean[2]) and torch.equal(dv, clean[3])


# ---- calls from several threads ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("t", [1, 5, 12, 40, 1100])
@pytest.mark.parametrize("name", ["product", "product_t", "grad", "expand", "quantize", "check"])
def test_a_thread_s_first_call(name, t):
    n, k = 512, 1024  # rows on 16-byte borders: no workspace is taken before the call's own work
    m = make(n, k, 64, torch.bfloat16, True, 0.01 if t == 5 else None, 27)
    q, f = matrix(m), matrix(fresh(n, k, 64, torch.bfloat16, True, None))
    x, dy = normal(t, t, k, dtype=torch.bfloat16), normal(t, t, n, dtype=torch.bfloat16)
    w, ds = normal(1, n, k, dtype=torch.bfloat16), torch.empty_like(m["scales"])
    call = {"product": lambda: q.product(x, dy), "product_t": lambda: q.product_t(dy, x), "grad": lambda: q.grad(x, dy, ds),
            "expand": lambda: q.expand(w), "quantize": lambda: f.quantize(w), "check": lambda: q.check()}[name]
    told = []

    def work():
        try:
            call()
        except Exception as e:  # noqa: BLE001
            told.append(e)

    torch.cuda.synchronize()
    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not told


def test_threads_that_call_at_once():
    """Each with a stream and vectors of its own, on one matrix: what each gets alone."""
    n, k, jobs = 517, 1037, []  # rows on no 16-byte border: every call takes workspaces
    m = make(n, k, 64, torch.bfloat16, True, 0.01, 27)
    q = matrix(m)

    def run(job, stream):
        x, dy, (y, dx, ds, dv, w) = job
        q.product(x, y, stream=stream)
        q.product_t(dy, dx, stream=stream)
        q.grad(x, dy, ds, dv, stream=stream)
        q.expand(w, stream=stream)

    for t in (1, 5, 12, 40, 300, 1100):
        x, dy = normal(t, t, k, dtype=torch.bfloat16), normal(t + 1, t, n, dtype=torch.bfloat16)
        out = (torch.empty_like(dy), torch.empty_like(x), torch.empty_like(m["scales"]), torch.zeros_like(m["residual"][2]),
               torch.empty(n, k, dtype=torch.bfloat16, device="cuda"))
        run((x, dy, out), 0)
        torch.cuda.synchronize()
        jobs.append((x, dy, out, [o.clone() for o in out], torch.cuda.Stream()))
        for o in out:
            o.zero_()
    torch.cuda.synchronize()
    told = []

    def work(job):
        try:
            for _ in range(30):
                run(job[:3], job[4].cuda_stream)
        except Exception as e:  # noqa: BLE001
            told.append(e)

    threads = [threading.Thread(target=work, args=(job,)) for job in jobs]
    for one in threads:
        one.start()
    for one in threads:
        one.join()
    torch.cuda.synchronize()
    assert not told
    for _, _, out, want, _ in jobs:
        for o, w in zip(out, want):
            assert torch.equal(o.view(torch.int16), w.view(torch.int16))
