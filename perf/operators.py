"""Measured cases of the 4-bit matrix operators (``mx_q4_*``): quantise and expand, product, transposed product and the
gradients of scales and residual values.

A matrix W of n_rows x n_cols is held as 4-bit codes with one scale (and, optionally, one zero point) per group of
consecutive columns of a row, plus a CSR residual of the entries that were too large for the codes:

    W[i, k] = scale[i, k // group] * (code[i, k] - zero[i, k // group]) + R[i, k]

``run`` computes either the plain form (elementary torch operations in 32 bits) or, where ``own`` is true, calls the
framework.  ``exact`` computes the definitions in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    def case(name, op, t, n, k, dtype, group, zeros, threshold, source=""):
        return {"name": name, "op": op, "t": t, "n": n, "k": k, "dtype": dtype, "group": group, "zeros": zeros,
                "threshold": threshold, "source": source or dtype}

    return [
        # one projection of a small model: quantised in place of a fake-quantisation step, no outliers
        case("quantize small", "quantize", 0, 1024, 1024, "bf16", 64, False, 0.0),
        # a large layer, zero points, half a percent of the entries kept apart as outliers
        case("quantize large", "quantize", 0, 8192, 8192, "bf16", 128, True, 2.8),
        # decoding one token through a small layer: latency is everything
        case("product 1 token small", "product", 1, 1024, 1024, "fp16", 32, False, 0.0),
        # decoding one token through a large layer with outliers: the weights' bytes are everything
        case("product 1 token large", "product", 1, 16384, 8192, "bf16", 128, True, 2.8),
        # a ragged batch of decoded tokens; odd rows, a short last group
        case("product 13 tokens ragged", "product", 13, 4099, 4104, "fp16", 64, True, 2.8),
        # a prompt
        case("product 2048 tokens", "product", 2048, 8192, 8192, "bf16", 128, False, 2.8),
        # gradient of the inputs of a handful of tokens through a frozen layer
        case("transposed 8 tokens", "transposed", 8, 4096, 4096, "fp16", 128, False, 0.0),
        # the same for a training batch
        case("transposed 2048 tokens", "transposed", 2048, 8192, 8192, "bf16", 128, True, 2.8),
        # odd everything
        case("transposed 333 tokens ragged", "transposed", 333, 2050, 2088, "bf16", 32, True, 2.8),
        # training scales on few tokens
        case("gradient 16 tokens", "gradient", 16, 4096, 4096, "bf16", 128, False, 0.0),
        # training scales and outliers on a batch
        case("gradient 2048 tokens", "gradient", 2048, 8192, 8192, "bf16", 64, True, 2.8),
        # odd everything
        case("gradient 517 tokens ragged", "gradient", 517, 1000, 4100, "fp16", 32, False, 2.8),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["quantize", "product", "product", "transposed", "gradient"])
    dtype = rng.choice(["fp16", "bf16"])
    n = size(256, 16384)
    k = size(256, 16384)
    if rng.random() < 0.75:  # most layers are whole numbers of groups wide
        k = max(256, k // 128 * 128)
    k, n = min(k, (1 << 26) // n), min(n, (1 << 26) // k)
    t = 0 if op == "quantize" else size(1, 2048)
    source = rng.choice([dtype, dtype, "fp32"]) if op == "quantize" and n * k <= 1 << 25 else dtype
    return {"op": op, "t": t, "n": n, "k": k, "dtype": dtype, "group": rng.choice([32, 64, 128, 256]),
            "zeros": rng.random() < 0.5, "threshold": rng.choice([0.0, 2.5, 2.8, 3.2]), "source": source}


def _outliers(case):
    """Expected number of residual entries: threshold is in standard deviations of normal weights; 0 = no residual."""
    p = math.erfc(case["threshold"] / math.sqrt(2)) if case["threshold"] else 0.0
    return int(p * case["n"] * case["k"])


def work(case):
    n, k, t = case["n"], case["k"], case["t"]
    groups = n * -(-k // case["group"])
    nnz = _outliers(case)
    scales = 2 * groups + (groups if case["zeros"] else 0)
    residual = 6 * nnz + 4 * (n + 1) if case["threshold"] else 0
    codes = n * -(-k // 2)
    if case["op"] == "quantize":
        source = 4 if case["source"] == "fp32" else 2
        return {"bytes": n * k * source + 2 * (codes + scales + residual) + 2 * n * k, "flops": 6 * n * k}
    # the gradients do not read the scales and the residual's values, but write as many
    moved = codes + scales + residual + 2 * t * (n + k)
    return {"bytes": moved, "flops": 2 * t * (n * k + nnz)}


# ---- plain form ----------------------------------------------------------------------------------------------------


def _grouped(a, group):
    """[n, k] -> [n, groups, group], the last group filled with zeros."""
    n, k = a.shape
    groups = -(-k // group)
    if groups * group != k:
        a = torch.cat([a, a.new_zeros(n, groups * group - k)], 1)
    return a.view(n, groups, group)


def _spread(a, group, k):
    """One value per group -> one per column."""
    n, groups = a.shape
    return a[:, :, None].expand(n, groups, group).reshape(n, groups * group)[:, :k]


def _quantize_plain(w, group, dtype, zeros, threshold):
    """codes, scales, zero points and the residual's (row pointers, columns, values) of w."""
    n, k = w.shape
    w32 = w.float()
    out = w32.abs() > threshold if threshold is not None else None
    kept = w32.masked_fill(out, 0.0) if out is not None else w32
    g = _grouped(kept, group)
    if zeros:
        lo, hi = g.amin(2).clamp(max=0), g.amax(2).clamp(min=0)
        s = ((hi - lo) / torch.full_like(hi, 15)).to(dtype)
        # quotients of values with few bits lie on the border between two whole numbers, hence 64 bits
        z = torch.round(-lo.double() / s.double()).clamp(0, 15)
        z = torch.where(s == 0, torch.zeros_like(z), z).float()
    else:
        amax = g.abs().amax(2)
        s = (amax / torch.full_like(amax, 7)).to(dtype)
        z = torch.full_like(s, 8, dtype=torch.float32)
    c = torch.round(g.double() / s.double()[:, :, None]).float()
    c = torch.where((s == 0)[:, :, None], torch.zeros_like(c), c) + z[:, :, None]
    c = c.clamp(0 if zeros else 1, 15).to(torch.uint8).view(n, -1)[:, :k]
    if out is None:
        return c, s, z, None
    row_ptr = torch.zeros(n + 1, dtype=torch.int32, device=w.device)
    row_ptr[1:] = out.sum(1).cumsum(0)
    row, col = out.nonzero(as_tuple=True)
    return c, s, z, (row_ptr, col.int(), w[row, col].to(dtype))


def _unpack(codes, k):
    return torch.stack([codes & 15, codes >> 4], 2).view(codes.shape[0], -1)[:, :k]


def _pack(c):
    """Two codes a byte, even column in the low half; rows padded to a multiple of 16 bytes."""
    n, k = c.shape
    full = c.new_zeros(n, -(-k // 32) * 32)
    full[:, :k] = c
    return (full[:, 0::2] | (full[:, 1::2] << 4)).contiguous()


def _steps(codes, zeros, group, k):
    """code - zero in 32 bits."""
    c = _unpack(codes, k).float()
    return c - (8 if zeros is None else _spread(zeros, group, k).float())


def _rows_of(row_ptr, count):
    """The row of each residual entry."""
    rows = torch.arange(row_ptr.numel() - 1, device=row_ptr.device)
    return torch.repeat_interleave(rows, row_ptr.diff(), output_size=count)


def _entries(st):
    """Rows, columns and values of the residual's entries; the buffers have room for more."""
    row_ptr, col, val = st["residual"]
    count = int(row_ptr[-1])
    return _rows_of(row_ptr, count), col[:count], val[:count]


def _dense_plain(st):
    k, group = st["k"], st["group"]
    w = _steps(st["codes"], st["zeros"], group, k) * _spread(st["scales"], group, k).float()
    if st["residual"] is not None:
        row, col, val = _entries(st)
        w[row, col] += val.float()
    return w


def _run_plain(st):
    dtype, group = st["dtype"], st["group"]
    if st["op"] == "quantize":
        c, s, z, residual = _quantize_plain(st["w"], group, dtype, st["use_zeros"], st["threshold"])
        n, k = c.shape
        w = (c.float() - _spread(z, group, k)) * _spread(s, group, k).float()
        answer = {"scales": s}
        if st["use_zeros"]:
            answer["zeros"] = z.to(torch.uint8)
        if residual is not None:
            row_ptr, col, val = residual
            m = min(col.numel(), st["cap"])
            answer["row_ptr"] = row_ptr
            answer["col"] = torch.zeros(st["cap"], dtype=torch.int32, device=w.device)
            answer["val"] = torch.zeros(st["cap"], dtype=dtype, device=w.device)
            answer["col"][:m], answer["val"][:m] = col[:m], val[:m]
            w[_rows_of(row_ptr, col.numel()), col] += val.float()
        return answer | {"w": w.to(dtype)}
    if st["op"] == "product":
        return (st["x"].float() @ _dense_plain(st).T).to(dtype)
    if st["op"] == "transposed":
        return (st["dy"].float() @ _dense_plain(st)).to(dtype)
    g = st["dy"].float().T @ st["x"].float()
    steps = _steps(st["codes"], st["zeros"], group, st["k"])
    answer = {"scales": _grouped(g * steps, group).sum(2).to(dtype)}
    if st["residual"] is not None:
        row, col, _ = _entries(st)
        answer["val"] = torch.zeros_like(st["residual"][2])
        answer["val"][: row.numel()] = g[row, col].to(dtype)
    return answer


# ---- the framework's operators -------------------------------------------------------------------------------------


def _run_own(st):
    stream = torch.cuda.current_stream().cuda_stream
    dtype, n, k, q = st["dtype"], st["n"], st["k"], st["matrix"]
    if st["op"] == "quantize":
        q.quantize(st["w"], threshold=st["threshold"], stream=stream)
        w = torch.empty(n, k, dtype=dtype, device="cuda")
        q.expand(w, stream=stream)
        answer = {"scales": q.scales}
        if st["use_zeros"]:
            answer["zeros"] = q.zeros
        if st["threshold"] is not None:
            answer |= {"row_ptr": q.res_row_ptr, "col": q.res_col_ind, "val": q.res_val}
        return answer | {"w": w}
    if st["op"] == "product":
        y = torch.empty(st["x"].shape[0], n, dtype=dtype, device="cuda")
        q.product(st["x"], y, stream=stream)
        return y
    if st["op"] == "transposed":
        dx = torch.empty(st["dy"].shape[0], k, dtype=dtype, device="cuda")
        q.product_t(st["dy"], dx, stream=stream)
        return dx
    d_scales = torch.empty_like(st["scales"])
    # only as many values as there are entries are written
    d_val = torch.zeros_like(st["residual"][2]) if st["residual"] is not None else None
    q.grad(st["x"], st["dy"], d_scales, d_val, stream=stream)
    return {"scales": d_scales} if d_val is None else {"scales": d_scales, "val": d_val}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, k, t, group = case["n"], case["k"], case["t"], case["group"]
    dtype = _TYPES[case["dtype"]]
    sigma = 1 / math.sqrt(k)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    st = {"op": case["op"], "n": n, "k": k, "group": group, "dtype": dtype, "use_zeros": case["zeros"]}
    threshold = case["threshold"] * sigma if case["threshold"] else None
    # room for the outliers: their expected number and as much again
    cap = 2 * _outliers(case) + 1024
    w = (normal(n, k) * sigma).to(_TYPES[case["source"]])
    if case["op"] == "quantize":
        st |= {"w": w, "threshold": threshold, "cap": cap}
        fresh = {"codes": torch.zeros(n, -(-k // 32) * 16, dtype=torch.uint8, device="cuda"),
                 "scales": torch.zeros(n, -(-k // group), dtype=dtype, device="cuda"),
                 "zeros": torch.zeros(n, -(-k // group), dtype=torch.uint8, device="cuda") if case["zeros"] else None,
                 "residual": None}
        if threshold is not None:
            fresh["residual"] = (torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
                                 torch.zeros(cap, dtype=torch.int32, device="cuda"),
                                 torch.zeros(cap, dtype=dtype, device="cuda"))
        st |= fresh
    else:
        c, s, z, residual = _quantize_plain(w, group, dtype, case["zeros"], threshold)
        if residual is not None:
            row_ptr, col, val = residual
            spare = max(0, cap - col.numel())
            residual = (row_ptr, torch.cat([col, col.new_zeros(spare)])[:cap],
                        torch.cat([val, val.new_zeros(spare)])[:cap])
        st |= {"codes": _pack(c), "scales": s, "zeros": z.to(torch.uint8) if case["zeros"] else None,
               "residual": residual}
        del w, c
        # activations: normal, with a few channels an order of magnitude louder than the others
        loud = 1 + 9 * (torch.rand(k, generator=gen, device="cuda") < 0.002).float()
        st["x"] = (normal(t, k) * loud).to(dtype)
        st["dy"] = (normal(t, n) * 0.01).to(dtype)
    if own:  # the view of these buffers that a program keeps; no data is touched
        import matxtract_b200 as mx

        res = st["residual"] or (None, None, None)
        st["matrix"] = mx.Q4Matrix(n, k, group, st["codes"], st["scales"], zeros=st["zeros"], res_row_ptr=res[0],
                                   res_col_ind=res[1], res_val=res[2])
    return st


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    n, k, group, dtype = case["n"], case["k"], case["group"], st["dtype"]
    of = torch.arange(k, device="cuda") // group  # a column's group
    groups = -(-k // group)
    if case["op"] == "quantize":
        w = st["w"].double()
        far = w.abs() > (math.inf if st["threshold"] is None else
                         torch.tensor(st["threshold"], dtype=torch.float32, device="cuda").double())
        near = torch.where(far, 0.0, w)
        index = of[None].expand(n, k)
        hi = torch.zeros(n, groups, dtype=torch.float64, device="cuda").scatter_reduce(1, index, near, "amax")
        lo = torch.zeros(n, groups, dtype=torch.float64, device="cuda").scatter_reduce(1, index, near, "amin")
        if case["zeros"]:
            s = ((hi - lo) / 15).to(dtype).double()
            z = torch.where(s > 0, (-lo / s).round(), 0.0).clamp(0, 15)
            lowest = 0
        else:
            s = (torch.maximum(hi, -lo) / 7).to(dtype).double()
            z = torch.full_like(s, 8)
            lowest = 1
        sk, zk = s[:, of], z[:, of]
        c = (torch.where(sk > 0, near / sk, 0.0).round() + zk).clamp(lowest, 15)
        value = (c - zk) * sk + torch.where(far, w.to(dtype).double(), 0.0)
        answer = {"scales": s}
        if case["zeros"]:
            answer["zeros"] = None
        if st["threshold"] is not None:
            at = far.reshape(-1).nonzero()[:, 0][: st["cap"]]
            val = torch.zeros(st["cap"], dtype=torch.float64, device="cuda")
            val[: at.numel()] = w.reshape(-1)[at].to(dtype).double()
            answer |= {"row_ptr": None, "col": None, "val": val}
        return answer | {"w": value}
    low, high = st["codes"].bitwise_and(15), st["codes"].div(16, rounding_mode="floor")
    code = torch.empty(n, 2 * st["codes"].shape[1], dtype=torch.float64, device="cuda")
    code[:, 0::2], code[:, 1::2] = low.double(), high.double()
    code = code[:, :k]
    code -= st["zeros"].double()[:, of] if case["zeros"] else 8.0
    flat = None
    if st["residual"] is not None:
        row_ptr, col, val = st["residual"]
        entry = torch.arange(int(row_ptr[n]), device="cuda")
        row = torch.searchsorted(row_ptr[1:].long(), entry, right=True)
        flat = row * k + col[: entry.numel()].long()
    x, dy = st["x"].double(), st["dy"].double()
    if case["op"] == "gradient":
        g = torch.einsum("tn,tk->nk", dy, x)
        total = torch.zeros(n, groups, dtype=torch.float64, device="cuda").index_add_(1, of, g * code)
        if flat is None:
            return {"scales": total}
        value = torch.zeros(st["residual"][2].numel(), dtype=torch.float64, device="cuda")
        value[: flat.numel()] = g.reshape(-1)[flat]
        return {"scales": total, "val": value}
    w = code * st["scales"].double()[:, of]
    if flat is not None:
        w.view(-1).index_add_(0, flat, val[: flat.numel()].double())
    if case["op"] == "product":
        return torch.einsum("tk,nk->tn", x, w)
    return torch.einsum("tn,nk->tk", dy, w)
