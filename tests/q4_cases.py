"""4-bit matrices with group scales and a CSR residual: inputs and the definitions in 64 bits (plain torch)."""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step: the relative error of one rounding
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a step of the smallest values


def make(n, k, group, dtype, zeros, density, seed, device="cuda", empty_rows=True, spare=5):
    """A matrix whose numbers are drawn freely: codes 0..15, zero points, scales over three orders of magnitude."""
    g = torch.Generator(device=device).manual_seed(seed)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=device)

    groups = -(-k // group)
    width = -(-k // 32) * 16
    # the bytes behind a row's last code hold codes too: they must not count
    codes = torch.randint(0, 256, (n, width), generator=g, device=device, dtype=torch.int32).to(torch.uint8)
    scales = torch.exp(uniform(n, groups) * 4 - 6).to(dtype)
    z = torch.randint(0, 16, (n, groups), generator=g, device=device, dtype=torch.int32).to(torch.uint8) if zeros else None
    m = {"n": n, "k": k, "group": group, "dtype": dtype, "codes": codes, "scales": scales, "zeros": z,
         "residual": None}
    if density is not None:
        hit = uniform(n, k) < density
        if empty_rows and n > 2:
            hit[1::3] = False
        if n and k:
            hit[0, k - 1] = True  # the last column, and row ends that meet row starts
        ptr = torch.zeros(n + 1, dtype=torch.int32, device=device)
        ptr[1:] = hit.sum(1).cumsum(0)
        row, col = hit.nonzero(as_tuple=True)
        val = (torch.randn(col.numel(), generator=g, device=device) * 2).to(dtype)
        pad = torch.full((spare,), 2 ** 30, dtype=torch.int32, device=device)  # room behind the last entry
        m["residual"] = (ptr, torch.cat([col.int(), pad]), torch.cat([val, torch.full((spare,), math.nan, dtype=dtype,
                                                                                     device=device)]))
    return m


def steps64(m):
    k = m["k"]
    c = m["codes"].long()
    c = torch.stack([c % 16, c // 16], 2).reshape(m["n"], -1)[:, :k].double()
    of = torch.arange(k, device=c.device) // m["group"]
    return c - (m["zeros"].double()[:, of] if m["zeros"] is not None else 8.0), of


def entries(m):
    ptr, col, val = m["residual"]
    nnz = int(ptr[-1])
    row = torch.repeat_interleave(torch.arange(m["n"], device=ptr.device), ptr.diff().long())
    return row, col[:nnz].long(), val[:nnz]


def dense64(m):
    steps, of = steps64(m)
    w = steps * m["scales"].double()[:, of]
    if m["residual"] is not None:
        row, col, val = entries(m)
        w.index_put_((row, col), val.double(), accumulate=True)
    return w


def rounded(value, magnitude, terms, dtype, weights=1):
    """How far a result may be from `value`, the exact sum of `terms` products whose magnitudes sum to `magnitude`:
    every weight may be rounded once to the type (`weights` = 1; 2 where a residual value is added to a rounded one),
    the sum is taken in 32 bits (each addition off by at most one step, 2^-23, of a partial sum) and rounded once."""
    return value.abs() * U[dtype] * 1.01 + magnitude * (weights * U[dtype] + (terms + 8) * 2.0 ** -23) * 1.01 + TINY[dtype]


def matrix(m):
    import matxtract_b200 as mx

    r = m["residual"] or (None, None, None)
    return mx.Q4Matrix(m["n"], m["k"], m["group"], m["codes"], m["scales"], zeros=m["zeros"], res_row_ptr=r[0],
                       res_col_ind=r[1], res_val=r[2])
