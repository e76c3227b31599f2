"""4-bit matrices on the GPU: numbers at the ends of their types, and what lies behind a matrix's last column."""
import math

import pytest
import torch

from conftest import has_gpu
from q4_cases import dense64, make, matrix, rounded
from test_gpu_q4 import TYPES, close, fresh, normal

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
