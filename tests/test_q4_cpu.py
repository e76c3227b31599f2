"""4-bit matrices: what the C ABI refuses before it looks for a GPU, and the definitions' own consistency."""
import ctypes as C

import pytest
import torch

import matxtract_b200 as mx
from matxtract_b200 import capi

from conftest import has_gpu
from q4_cases import dense64, make

P = 1 << 20  # an address that is never followed


def _m(**kw):
    a = dict(n_rows=4, n_cols=70, group=32, dtype=mx.FP16, device=0, res_cap=8, code_ld=48, codes=P, scales=P, zeros=P,
             res_row_ptr=P, res_col_ind=P, res_val=P)
    a.update(kw)
    return C.byref(capi._Q4Matrix(**a))


def _calls(m, n_vec=3, x=P, ld_x=70, y=P, ld_y=4):
    L = capi.lib()
    return {"expand": L.mx_q4_expand(m, x, ld_x, None),
            "quantize": L.mx_q4_quantize(m, mx.FP32, x, ld_x, 1.0, None),
            "product": L.mx_q4_product(m, n_vec, x, ld_x, y, ld_y, None),
            "product_t": L.mx_q4_product_t(m, n_vec, y, ld_y, x, ld_x, None),
            "grad": L.mx_q4_grad(m, n_vec, x, ld_x, y, ld_y, P, P, None)}


BAD = [dict(n_rows=-1), dict(n_cols=-1), dict(group=0), dict(group=-32), dict(group=48), dict(dtype=mx.FP64),
       dict(dtype=mx.FP32), dict(dtype=9), dict(device=-1), dict(res_cap=-1), dict(code_ld=32), dict(code_ld=36),
       dict(code_ld=-48), dict(codes=None), dict(codes=P + 8), dict(scales=None), dict(scales=P + 1),
       dict(res_col_ind=None), dict(res_val=None), dict(res_row_ptr=P + 2), dict(res_val=P + 1),
       dict(n_cols=(1 << 30) + 1, code_ld=1 << 30), dict(n_rows=(1 << 30) + 1), dict(group=(1 << 30) + 32)]


@pytest.mark.parametrize("bad", BAD, ids=lambda b: ",".join(f"{k}={v}" for k, v in b.items()))
def test_bad_matrices_are_refused(bad):
    assert set(_calls(_m(**bad)).values()) == {1}
    assert capi.lib().mx_q4_check(_m(**bad), None) == 1


@pytest.mark.parametrize("bad", [dict(n_vec=-1), dict(n_vec=(1 << 30) + 1), dict(x=None), dict(y=None), dict(ld_x=69),
                                 dict(ld_y=3), dict(x=P + 1), dict(y=P + 1)])
def test_bad_vectors_are_refused(bad):
    got = _calls(_m(), **bad)
    for name in ("product", "product_t", "grad"):
        assert got[name] == 1, name


def test_other_refusals():
    L = capi.lib()
    assert set(_calls(None).values()) == {1} and L.mx_q4_check(None, None) == 1
    assert L.mx_q4_quantize(_m(), mx.FP64, P, 70, 1.0, None) == 1
    assert L.mx_q4_quantize(_m(), mx.FP32, P + 2, 70, 1.0, None) == 1  # 32-bit values on a 2-byte border
    assert L.mx_q4_quantize(_m(), mx.FP32, P, 69, 1.0, None) == 1
    assert L.mx_q4_grad(_m(res_row_ptr=None), 1, P, 70, P, 4, None, P, None) == 1  # no residual to have a gradient
    assert L.mx_q4_grad(_m(), 1, P, 70, P, 4, P + 1, None, None) == 1
    assert capi.lib().mx_create(C.byref(C.c_void_p()), 0, mx.BF16) == 1  # the types of these entry points only


@pytest.mark.skipif(has_gpu(), reason="only meaningful on a machine without a GPU")
def test_good_calls_fail_loudly_without_a_gpu():
    assert set(_calls(_m()).values()) == {8}
    assert set(_calls(_m(zeros=None, res_row_ptr=None, res_col_ind=None, res_val=None)).values()) == {1, 8}  # grad: 1
    assert capi.lib().mx_q4_check(_m(), None) == 8


def test_the_binding_refuses_what_does_not_fit():
    n, k, g = 4, 64, 32
    codes, scales = torch.zeros(n, 32, dtype=torch.uint8), torch.zeros(n, 2, dtype=torch.float16)
    for kw in (dict(codes=codes), dict(scales=scales.double()), dict(scales=scales[:, :1]), dict(group=33),
               dict(codes=codes[:, :31]), dict(codes=codes.int()), dict(n_rows=5)):
        a = dict(n_rows=n, n_cols=k, group=g, codes=codes, scales=scales) | kw
        with pytest.raises(mx.MxError) as e:  # the first one too: the tensors are on the CPU
            mx.Q4Matrix(**a)
        assert e.value.status == 1


def test_struct_layout_matches_the_header(tmp_path):
    import subprocess
    from pathlib import Path

    root = Path(__file__).resolve().parent.parent
    src = tmp_path / "t.c"
    src.write_text('#include "mx_capi.h"\n#include <stddef.h>\n#include <stdio.h>\nint main(void){printf("%zu", '
                   "sizeof(mx_q4_matrix));\n" + "".join(f'printf(" %zu", offsetof(mx_q4_matrix, {name}));\n'
                                                        for name, _ in capi._Q4Matrix._fields_) + "return 0;}\n")
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{root / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(capi._Q4Matrix)] + [getattr(capi._Q4Matrix, name).offset for name, _ in capi._Q4Matrix._fields_]


def test_gradients_of_the_definition():
    """The formulas of mx_q4_product_t and mx_q4_grad against differences of the product's definition."""
    m = make(5, 70, 32, torch.float16, True, 0.1, 3, device="cpu")
    x = torch.randn(3, 70, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    dy = torch.randn(3, 5, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    from q4_cases import entries, steps64

    steps, of = steps64(m)
    g = dy.T @ x
    d_scales = torch.zeros(5, 3, dtype=torch.float64).index_add_(1, of, g * steps)
    row, col, val = entries(m)
    scales = m["scales"].double()

    def loss(s, v, xx):
        w = steps * s[:, of]
        w = w.index_put((row, col), v, accumulate=True)
        return ((xx @ w.T) * dy).sum()

    v64 = val.double()
    h = 1e-6
    for i, j in ((0, 0), (2, 1), (4, 2)):
        e = torch.zeros_like(scales)
        e[i, j] = h
        assert abs((loss(scales + e, v64, x) - loss(scales - e, v64, x)) / (2 * h) - d_scales[i, j]) < 1e-6
    e = torch.zeros_like(v64)
    e[3] = h
    assert abs((loss(scales, v64 + e, x) - loss(scales, v64 - e, x)) / (2 * h) - g[row[3], col[3]]) < 1e-6
    e = torch.zeros_like(x)
    e[1, 69] = h
    assert abs((loss(scales, v64, x + e) - loss(scales, v64, x - e)) / (2 * h) - (dy @ dense64(m))[1, 69]) < 1e-6


def test_waiting_in_vain_is_bounded():
    L = capi.lib()
    for bad in ((-1, 0, 1), (0, -1, 1), (0, 4, 1), (0, 0, (1 << 16) + 1)):
        assert L.mx_q4_wait_in_vain(*bad, None) == 1


def test_the_binding_hands_no_size_on_that_an_int_does_not_hold():
    """2^32 + 1 vectors are not one vector."""
    q = object.__new__(mx.Q4Matrix)
    q.vdt, q.device = torch.float16, torch.device("meta")
    assert q._rows(torch.empty(1 << 30, 1, dtype=torch.float16, device="meta"), "x", 1) == (1 << 30, 1)
    for rows in ((1 << 30) + 1, (1 << 32) + 1):
        with pytest.raises(mx.MxError) as e:
            q._rows(torch.empty(rows, 1, dtype=torch.float16, device="meta"), "x", 1)
        assert e.value.status == 1 and "2^30" in str(e.value)
    for n, k, g in (((1 << 32) + 4, 64, 32), (4, (1 << 32) + 64, 32), (4, 64, (1 << 32) + 32)):
        with pytest.raises(mx.MxError) as e:
            mx.Q4Matrix(n, k, g, torch.empty(n, max(16, k // 2), dtype=torch.uint8, device="meta"),
                        torch.empty(n, -(-k // g), dtype=torch.float16, device="meta"))
        assert e.value.status == 1 and "2^30" in str(e.value)
