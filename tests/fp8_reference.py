"""Plain 64-bit forms of the block-scaled 8-bit floating point operators, on the CPU, for tests."""
import math

import torch

BLOCK, TOP = 128, 448.0
LEAST = TOP * 2.0 ** -126


def nearest_e4m3(v):
    """The e4m3 value next to each v (float64), half to even; |v| < 464."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.pow(2.0, exponent - 3)
    r = torch.round(v / step) * step
    assert bool((r[torch.isfinite(v)].abs() <= TOP).all())
    return r


def blocks_of(k):
    return torch.arange(k) // BLOCK


def row_maxima(y):
    """[M, blocks] largest finite magnitude of y [M, K] in each block, at least LEAST."""
    m, k = y.shape
    a = torch.where(torch.isfinite(y), y.abs(), torch.zeros_like(y))
    top = torch.full((m, -(-k // BLOCK)), LEAST, dtype=torch.float64)
    return top.scatter_reduce_(1, blocks_of(k).expand(m, k), a, "amax")


def f32(v):
    return v.to(torch.float32).double()


def quantize_with(x, top):
    """(codes as float64, scales as float32) of x (float64 holding storage values) for block maxima `top`, spread to x's
    shape by the caller: the fp32 arithmetic that the operator documents, step by step."""
    t32 = top.to(torch.float32)
    inv = (torch.tensor(TOP, dtype=torch.float32) / t32).double()
    v = f32(x * inv)                       # one fp32 product: the float64 product of two fp32 values is exact
    return nearest_e4m3(v)


def quantize_rows(x):
    x = x.double().cpu()
    top = row_maxima(x)
    q = quantize_with(torch.where(torch.isfinite(x), x, torch.full_like(x, math.nan)), top[:, blocks_of(x.shape[1])])
    scale = top.to(torch.float32) / torch.tensor(TOP, dtype=torch.float32)
    return q, scale.t().contiguous()


def quantize_weight(w):
    w = w.double().cpu()
    n, k = w.shape
    rows = torch.arange(n) // BLOCK
    by_row = row_maxima(w)
    top = torch.full((-(-n // BLOCK), by_row.shape[1]), LEAST, dtype=torch.float64)
    top.scatter_reduce_(0, rows[:, None].expand_as(by_row), by_row, "amax")
    q = quantize_with(torch.where(torch.isfinite(w), w, torch.full_like(w, math.nan)), top[rows][:, blocks_of(k)])
    return q, top.to(torch.float32) / torch.tensor(TOP, dtype=torch.float32)


def row_values(q, s):
    """float64 values of activation codes."""
    return q.cpu().to(torch.float32).double() * s.cpu().double().t()[:, blocks_of(q.shape[1])]


def weight_values(q, s):
    n, k = q.shape
    rows = torch.arange(n) // BLOCK
    return q.cpu().to(torch.float32).double() * s.cpu().double()[rows][:, blocks_of(k)]


def product(xq, xs, wq, ws):
    """(exact product, sum of magnitudes) in float64."""
    x, w = row_values(xq, xs), weight_values(wq, ws)
    return x @ w.t(), x.abs() @ w.abs().t()


def product_error(mag, k):
    """Bound on |fp32 result - exact| for a sum of magnitudes `mag` over k columns.  Products of two e4m3 values are exact in
    fp32 (8 significant bits).  A block's 128 products meet in at most 128 additions, its sum is scaled (two roundings: the
    scales' product and the scaled sum) and added (one) for each of ceil(k / 128) blocks.  Each step is off by at most one
    unit (2^-23; a matrix instruction may truncate where the vector unit rounds by half a unit) of a partial sum that the
    sum of magnitudes bounds."""
    return (128 + 2 + -(-k // BLOCK) + 2) * 2.0 ** -23 * mag


def act(g, name):
    return g * torch.sigmoid(g) if name == "silu" else g * torch.special.ndtr(g)


def check_codes_of(q, s, y, dy):
    """Codes q with scales s [blocks, M] stand for y (float64, known to dy): each scale is the block maximum / 448 up to dy
    and two fp32 roundings, and each code's value is within half an e4m3 step (2^-4 relative; 2^-10 of the scale below the
    normal range), dy, and the three fp32 roundings of the quotients and the product."""
    m, k = y.shape
    b = blocks_of(k)
    s = s.cpu().double()
    assert tuple(s.shape) == (-(-k // BLOCK), m)
    top = row_maxima(y)
    slack = torch.zeros_like(top).scatter_reduce_(1, b.expand(m, k), dy, "amax")
    bad = (s.t() * TOP - top).abs() > slack + 2.0 ** -22 * top
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} scales are off"
    value = q.cpu().to(torch.float32).double() * s.t()[:, b]
    tol = (2.0 ** -4 + 2.0 ** -20) * (y.abs() + dy) + 2.0 ** -10 * s.t()[:, b] + dy
    # the largest of a block maps to 448 by its own maximum; dy may move it past by a relative slack / top
    tol = tol + slack[:, b]
    off = (value - y).abs()
    assert bool((off <= tol).all()), f"{int((off > tol).sum())} of {off.numel()} values are off, worst {float((off / tol).max()):.3g} of the bound"
