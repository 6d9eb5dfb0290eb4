"""The K/V cache operators' definition in plain 64-bit torch on the CPU, for tests/test_gpu_kv_cache.py: what an append
stores, what a read returns, and where a token lies."""
import torch

QMIN = {"int8": -128, "int4": -8}
QMAX = {"int8": 127, "int4": 7}
FORMATS = ["16", "fp8", "int8", "int4", "int8_tok", "int4_tok", "int8_g64", "int4_g64"]
INT_OF = {torch.float16: torch.int16, torch.bfloat16: torch.int16, torch.float8_e4m3fn: torch.uint8}


def kind_of(fmt):
    return fmt.split("_")[0]


def pool_dtype(fmt, dtype):
    return {"16": dtype, "fp8": torch.float8_e4m3fn, "int8": torch.int8, "int4": torch.uint8}[kind_of(fmt)]


def pool_width(fmt, dim):
    return dim // 2 if kind_of(fmt) == "int4" else dim


def pair_shape(fmt, pages, page, heads, dim):
    return [pages, page, heads] + ([dim // 64] if fmt.endswith("g64") else []) + [2]


def to_e4m3(y):
    """The nearest e4m3 value of float64 y (ties to even), saturating at +-448; NaN stays NaN."""
    y = y.clamp(-448.0, 448.0)
    _, e = torch.frexp(y)
    step = torch.exp2((e.double() - 1).clamp_min(-6.0) - 3.0)
    return torch.round(y / step) * step


def quantise(x, fmt, scale):
    """(values of the format: float64 numbers or integers [tokens, heads, dim]; pairs float32 or None) of 16-bit rows x."""
    xd, kind = x.double(), kind_of(fmt)
    if kind == "16":
        return xd, None
    if "_" not in fmt:
        y = xd / (torch.ones(x.shape[1]) if scale is None else scale).double()[None, :, None]
        if kind == "fp8":
            return to_e4m3(y), None
        n = torch.round(y).clamp(QMIN[kind], QMAX[kind])
        return torch.where(torch.isnan(n), torch.zeros_like(n), n), None
    xr = xd.unflatten(-1, (-1, 64)) if fmt.endswith("g64") else xd[..., None, :]
    lo, hi = xr.amin(-1, keepdim=True), xr.amax(-1, keepdim=True)
    sc = ((hi - lo) / float(QMAX[kind] - QMIN[kind])).float().clamp_min(1e-8)
    zero = (QMIN[kind] - lo / sc.double()).float()
    n = torch.round(xr / sc.double() + zero.double()).clamp(QMIN[kind], QMAX[kind]).flatten(-2)
    pair = torch.cat([sc, zero], dim=-1)
    return torch.where(torch.isnan(n), torch.zeros_like(n), n), pair if fmt.endswith("g64") else pair[..., 0, :]


def stored_values(rows, fmt):
    """The numbers that pool rows stand for before their factors, float64."""
    if kind_of(fmt) == "int4":
        r = rows.to(torch.int16)
        return torch.stack([((r & 15) ^ 8) - 8, ((r >> 4) ^ 8) - 8], dim=-1).flatten(-2).double()
    return rows.double()


def read_values(n, fmt, scale, pair, dtype):
    """What a read returns for stored numbers n (float64), one float32 rounding per operation and then one to dtype."""
    nf = n.float()
    if kind_of(fmt) == "16":
        return n.to(dtype)
    if "_" not in fmt:
        return (nf if scale is None else nf * scale[None, :, None]).to(dtype)
    if fmt.endswith("g64"):
        return (pair[..., :1] * (nf.unflatten(-1, (-1, 64)) - pair[..., 1:])).flatten(-2).to(dtype)
    return (pair[..., :1] * (nf - pair[..., 1:])).to(dtype)


def places(table, lens, cu, tokens, page, pages):
    """(page, row within it) of every token of a call, or None where it has no place; lists on the CPU."""
    out = []
    batch = len(lens)
    for t in range(tokens):
        if cu is None:
            b, pos = t, lens[t] - 1
        else:
            if t < cu[0] or t >= cu[batch]:
                out.append("behind")
                continue
            b = max(i for i in range(batch) if cu[i] <= t)
            pos = lens[b] - (cu[b + 1] - t)
        if pos < 0 or pos // page >= table.shape[1]:
            out.append(None)
            continue
        pg = int(table[b, pos // page])
        out.append((pg, pos % page) if 0 <= pg < pages else None)
    return out
