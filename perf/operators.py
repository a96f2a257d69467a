"""Cases of the block-scaled 8-bit floating point operators: quantizer, root-mean-square norm, Linear and gated Linear.

Codes are OCP e4m3 (largest value 448).  An activation x [M, K] has a scale for each row and block of 128 columns, held
block-major as [ceil(K / 128), M]; a weight w [N, K] has one for each block of 128 x 128, [ceil(N / 128), ceil(K / 128)].
The value of a code is code * scale.
"""
import math

import torch

own = False

BLOCK = 128
TOP = 448.0                        # the largest e4m3 value
LEAST = TOP * 2.0 ** -126          # a block's maximum is taken as at least this, so that its scale is a normal number
EPS = 1e-6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZEOF = {"f32": 4, "f16": 2, "bf16": 2}

# The most that a drawn case costs: the largest listed product, and the largest listed pass over memory.
MOST_FLOPS = 2 * 8192 ** 3
MOST_BYTES = 8192 * 8192 * 7


def listed():
    return [
        # the activations of a prompt between two layers: the input of a down projection
        {"name": "quantize hidden 2048x14336", "op": "quantize", "M": 2048, "K": 14336, "dtype": "bf16"},
        # a layer's weight when the layer is built
        {"name": "quantize weight 14336x4096", "op": "quantize_weight", "N": 14336, "K": 4096, "dtype": "f32"},
        # one token through a layer's norm: a launch's latency
        {"name": "norm 1x4096", "op": "norm", "M": 1, "K": 4096, "dtype": "bf16", "residual": True},
        # a width that is no multiple of the block, a row count that is no multiple of anything, no residual
        {"name": "norm 777x5000", "op": "norm", "M": 777, "K": 5000, "dtype": "f16", "residual": False},
        # a long prompt, or a full batch of them
        {"name": "norm 8192x8192", "op": "norm", "M": 8192, "K": 8192, "dtype": "bf16", "residual": True},
        # one token through a down projection
        {"name": "linear 1x4096x14336", "op": "linear", "M": 1, "N": 4096, "K": 14336, "dtype": "bf16", "bias": False},
        # a decode batch of a serving engine through a wide projection
        {"name": "linear 77x14336x4096", "op": "linear", "M": 77, "N": 14336, "K": 4096, "dtype": "bf16", "bias": False},
        # an output layer of odd width with a bias, fp32 out; K ends inside a block
        {"name": "linear 1000x10001x4000", "op": "linear", "M": 1000, "N": 10001, "K": 4000, "dtype": "f32", "bias": True},
        # the benchmark's square product
        {"name": "linear 8192x8192x8192", "op": "linear", "M": 8192, "N": 8192, "K": 8192, "dtype": "bf16", "bias": False},
        # the gate and up projections of one token, of a decode batch, of a prompt
        {"name": "gated 1x14336x4096", "op": "gated", "M": 1, "N": 14336, "K": 4096, "act": "silu"},
        {"name": "gated 48x14336x4096", "op": "gated", "M": 48, "N": 14336, "K": 4096, "act": "silu"},
        {"name": "gated 4096x14336x4096", "op": "gated", "M": 4096, "N": 14336, "K": 4096, "act": "silu"},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["quantize", "quantize_weight", "norm", "linear", "linear", "gated", "gated"])
        width = _log_uniform(rng, 128, 28672)
        step = rng.choice([1, 16, 16, 128, 128])   # what the width is a multiple of: odd ones, whole vectors, whole blocks
        K = max(step, width // step * step)
        M = _log_uniform(rng, 1, 8192)
        N = _log_uniform(rng, 64, 28672)
        if op == "quantize":
            case = {"op": op, "M": M, "K": K, "dtype": rng.choice(["f32", "f16", "bf16"])}
        elif op == "quantize_weight":
            case = {"op": op, "N": N, "K": K, "dtype": rng.choice(["f32", "f16", "bf16"])}
        elif op == "norm":
            case = {"op": op, "M": M, "K": min(K, 16384), "dtype": rng.choice(["f32", "f16", "bf16"]), "residual": rng.random() < 0.6}
        elif op == "linear":
            case = {"op": op, "M": M, "N": N, "K": K, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "bias": rng.random() < 0.3}
        else:
            case = {"op": op, "M": M, "N": min(N, 14336), "K": K, "act": rng.choice(["silu", "silu", "gelu"])}
        w = work(case)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES:
            return case


def work(case):
    op, K = case["op"], case["K"]
    kb = -(-K // BLOCK)
    if op == "quantize_weight":
        n = case["N"]
        return {"bytes": n * K * (SIZEOF[case["dtype"]] + 1) + 4 * -(-n // BLOCK) * kb, "flops": 3 * n * K}
    m = case["M"]
    if op == "quantize":
        return {"bytes": m * K * (SIZEOF[case["dtype"]] + 1) + 4 * m * kb, "flops": 3 * m * K}
    if op == "norm":
        size = SIZEOF[case["dtype"]]
        return {"bytes": m * K * (size * (3 if case["residual"] else 1) + 1) + K * size + 4 * m * kb, "flops": 8 * m * K}
    n = case["N"]
    nb = -(-n // BLOCK)
    if op == "linear":
        moved = m * K + n * K + 4 * (m * kb + nb * kb) + m * n * SIZEOF[case["dtype"]] + (4 * n if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * m * n * K}
    return {"bytes": m * K + 2 * n * K + 4 * (m * kb + 2 * nb * kb) + m * n + 4 * m * nb, "flops": 4 * m * n * K}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _activations(m, k, gen, dev):
    """Rows of different sizes, with the few large columns that activations of language models have."""
    x = torch.randn(m, k, generator=gen, device=dev)
    x *= torch.exp(0.5 * torch.randn(m, 1, generator=gen, device=dev))
    return x * torch.where(torch.rand(k, generator=gen, device=dev) < 0.005, 20.0, 1.0)


def _weights(n, k, gen, dev):
    w = torch.randn(n, k, generator=gen, device=dev)
    return w.mul_(1.0 / math.sqrt(k)).mul_(torch.exp(0.3 * torch.randn(n, 1, generator=gen, device=dev)))


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, K = case["op"], case["K"]
    state = {"case": case}
    if op == "quantize_weight":
        state["w"] = _weights(case["N"], K, gen, dev).to(DTYPES[case["dtype"]])
        return state
    x = _activations(case["M"], K, gen, dev)
    if op in ("quantize", "norm"):
        state["x"] = x.to(DTYPES[case["dtype"]])
        if op == "norm":
            state["g"] = (1.0 + 0.1 * torch.randn(K, generator=gen, device=dev)).to(DTYPES[case["dtype"]])
            state["r"] = _activations(case["M"], K, gen, dev).to(DTYPES[case["dtype"]]) if case["residual"] else None
        return state
    state["xq"], state["xs"] = _plain_quantize(x)
    for name in ("w",) if op == "linear" else ("wg", "wu"):
        state[name + "q"], state[name + "s"] = _plain_quantize_weight(_weights(case["N"], K, gen, dev))
    if op == "linear":
        state["bias"] = torch.randn(case["N"], generator=gen, device=dev) if case["bias"] else None
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _padded(t, rows):
    """t [R, C] with zeros up to whole blocks of `rows` x 128."""
    r, c = t.shape
    more_r, more_c = -r % rows, -c % BLOCK
    if not (more_r or more_c):
        return t
    out = t.new_zeros(r + more_r, c + more_c)
    out[:r, :c] = t
    return out


def _plain_quantize(x):
    m, k = x.shape
    x = _padded(x.float(), 1).view(m, -1, BLOCK)
    top = x.abs().amax(dim=2).clamp(min=LEAST)
    q = (x * (TOP / top)[:, :, None]).to(torch.float8_e4m3fn).view(m, -1)
    return q[:, :k].contiguous(), (top / TOP).t().contiguous()


def _plain_quantize_weight(w):
    n, k = w.shape
    w = _padded(w.float(), BLOCK)
    w = w.view(w.shape[0] // BLOCK, BLOCK, w.shape[1] // BLOCK, BLOCK)
    top = w.abs().amax(dim=(1, 3)).clamp(min=LEAST)
    q = (w * (TOP / top)[:, None, :, None]).to(torch.float8_e4m3fn).view(w.shape[0] * BLOCK, -1)
    return q[:n, :k].contiguous(), top / TOP


def _plain_norm(x, r, g):
    if r is not None:
        x = (x.float() + r.float()).to(x.dtype)
    h = x.float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * g.float()
    return (*_plain_quantize(y), x) if r is not None else _plain_quantize(y)


def _plain_values(q, s):
    """The values that an activation's codes stand for, fp32."""
    m, k = q.shape
    return (_padded(q.float(), 1).view(m, -1, BLOCK) * s.t()[:, :, None]).view(m, -1)[:, :k]


def _plain_weight_values(q, s):
    n, k = q.shape
    w = _padded(q.float(), BLOCK)
    w = w.view(s.shape[0], BLOCK, s.shape[1], BLOCK) * s[:, None, :, None]
    return w.view(s.shape[0] * BLOCK, -1)[:n, :k]


def _plain_product(xq, xs, wq, ws):
    return _plain_values(xq, xs) @ _plain_weight_values(wq, ws).t()


def _plain_gated(state, act):
    g = _plain_product(state["xq"], state["xs"], state["wgq"], state["wgs"])
    u = _plain_product(state["xq"], state["xs"], state["wuq"], state["wus"])
    a = g / (1.0 + torch.exp(-g)) if act == "silu" else 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return _plain_quantize(a * u)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from quantization_amd import block_fp8
        if op == "quantize":
            return block_fp8.quantize_blocks_fp8(state["x"])
        if op == "quantize_weight":
            return block_fp8.quantize_weight_fp8(state["w"])
        if op == "norm":
            return block_fp8.rms_norm_fp8(state["x"], state["g"], EPS, residual=state["r"])
        if op == "linear":
            return block_fp8.linear_fp8(state["xq"], state["xs"], state["wq"], state["ws"], state["bias"], DTYPES[case["dtype"]])
        return block_fp8.gated_linear_fp8(state["xq"], state["xs"], state["wgq"], state["wgs"], state["wuq"], state["wus"],
                                          case["act"])
    if op == "quantize":
        return _plain_quantize(state["x"])
    if op == "quantize_weight":
        return _plain_quantize_weight(state["w"])
    if op == "norm":
        return _plain_norm(state["x"], state["r"], state["g"])
    if op == "linear":
        out = _plain_product(state["xq"], state["xs"], state["wq"], state["ws"])
        if state["bias"] is not None:
            out = out + state["bias"]
        return out.to(DTYPES[case["dtype"]])
    return _plain_gated(state, case["act"])


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _nearest_e4m3(v):
    """The e4m3 value next to each v (half to even), in 64 bits: three mantissa bits down to 2^-6, steps of 2^-9 below."""
    exponent = torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 1
    step = torch.ldexp(torch.ones_like(v), exponent - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _exact_rows(y):
    """Codes and scales [ceil(K / 128), M] of y [M, K], a column index for each block's members."""
    m, k = y.shape
    block = torch.arange(k, device=y.device) // BLOCK
    top = torch.full((m, -(-k // BLOCK)), LEAST, dtype=torch.float64, device=y.device)
    top.scatter_reduce_(1, block.expand(m, k), y.abs(), "amax")
    return _nearest_e4m3(y * TOP / top[:, block]), (top / TOP).t().contiguous()


def _exact_product(xq, xs, wq, ws):
    n, k = wq.shape
    block = torch.arange(k, device=xq.device) // BLOCK
    rows = torch.arange(n, device=xq.device) // BLOCK
    x = xq.double() * xs.double().t()[:, block]
    w = wq.double() * ws.double()[rows][:, block]
    return torch.matmul(x, w.t())


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_rows(state["x"].double())
    if op == "quantize_weight":
        w = state["w"].double()
        n, k = w.shape
        nb, kb = -(-n // BLOCK), -(-k // BLOCK)
        col = torch.arange(k, device=w.device) // BLOCK
        row = torch.arange(n, device=w.device) // BLOCK
        by_col = torch.zeros(n, kb, dtype=torch.float64, device=w.device).scatter_reduce_(1, col.expand(n, k), w.abs(), "amax")
        top = torch.full((nb, kb), LEAST, dtype=torch.float64, device=w.device)
        top.scatter_reduce_(0, row[:, None].expand(n, kb), by_col, "amax")
        return _nearest_e4m3(w * TOP / top[row][:, col]), top / TOP
    if op == "norm":
        h = state["x"].double()
        if state["r"] is not None:
            stored = (h + state["r"].double()).to(state["x"].dtype)   # the sum is kept in the stream's own type
            h = stored.double()
        y = h / torch.sqrt(h.square().sum(dim=1, keepdim=True) / case["K"] + EPS) * state["g"].double()
        return (*_exact_rows(y), h) if state["r"] is not None else _exact_rows(y)
    if op == "linear":
        out = _exact_product(state["xq"], state["xs"], state["wq"], state["ws"])
        return out if state["bias"] is None else out + state["bias"].double()
    g = _exact_product(state["xq"], state["xs"], state["wgq"], state["wgs"])
    u = _exact_product(state["xq"], state["xs"], state["wuq"], state["wus"])
    a = g * torch.sigmoid(g) if case["act"] == "silu" else g * torch.special.ndtr(g)
    return _exact_rows(a * u)
