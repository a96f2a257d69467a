"""Block-scaled 8-bit floating point: activations and weights as e4m3 codes with a scale for each block of 128, and the
operators of a feed-forward block that hand such activations to each other.

    q, s       = quantize_blocks_fp8(x)                        x [..., K] -> codes [..., K], scales [ceil(K/128), M]
    q, s[, h]  = rms_norm_fp8(x, g, eps, residual=r)           the norm of x (or of h = x + r, returned), as codes
    q, s       = gated_linear_fp8(q, s, wg, sg, wu, su)        act(x . Wg^T) * (x . Wu^T), as codes
    y          = linear_fp8(q, s, w, sw)                       x . W^T, floating point
    w, sw      = quantize_weight_fp8(weight)                   [N, K] -> codes [N, K], scales [ceil(N/128), ceil(K/128)]

The int8 path has one scale for a whole activation tensor (activation.py) and one for each output channel of a weight
(the reference's scheme, quant/Weight_Only/Qop.py:74-102); a few large columns, which the activations of language models
have, then take the codes of all others.  A scale for each 128 columns of a row keeps them to their own block.

M is the number of rows, the product of all dimensions but the last.  An activation's scales are block-major ([blocks, M],
dense).  Codes are torch.float8_e4m3fn; the value of a code is code * scale.  include/miq.h states the formulas.
"""
import torch

from . import _native


def _rows(x):
    """x [..., K] as a dense matrix."""
    if x.dim() == 2 and x.is_contiguous():
        return x
    if x.dim() < 1:
        raise RuntimeError("input must have at least one dimension")
    return x.reshape(x.shape[:-1].numel(), x.shape[-1]).contiguous()


def quantize_blocks_fp8(x):
    """x [..., K] float32, float16 or bfloat16 -> (codes [..., K], scales [ceil(K / 128), M])."""
    q, scale = _native.quantize_blocks_fp8(_rows(x))
    return q if x.dim() == 2 else q.view(x.shape), scale


def quantize_weight_fp8(w):
    """w [N, K] -> (codes [N, K], scales [ceil(N / 128), ceil(K / 128)]); once, when a layer is built."""
    return _native.quantize_weight_fp8(w)


def rms_norm_fp8(x, weight, eps=1e-6, residual=None):
    """The codes of h / rms(h) * weight, with h = x (returns codes, scales) or, with a residual, h = x + residual rounded to
    x's type (returns codes, scales, h).  weight: [K] of x's type or float32."""
    q, scale, total = _native.rms_norm_fp8(_rows(x), weight, eps, None if residual is None else _rows(residual))
    if x.dim() != 2:
        q, total = q.view(x.shape), None if total is None else total.view(x.shape)
    return (q, scale) if residual is None else (q, scale, total)


def linear_fp8(x, x_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16):
    """x [..., K] codes with their scales, times w [N, K] codes with theirs, plus bias [N] -> [..., N] of out_dtype."""
    y = _native.gemm_fp8(_rows(x), x_scale, w, w_scale, bias, out_dtype)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[-1])


def gated_linear_fp8(x, x_scale, w_gate, gate_scale, w_up, up_scale, act="silu"):
    """The codes of act(x . w_gate^T) * (x . w_up^T): (codes [..., N], scales [ceil(N / 128), M]).  act: "silu" or "gelu"."""
    q, scale = _native.gated_fp8(_rows(x), x_scale, w_gate, gate_scale, w_up, up_scale, act)
    return (q if x.dim() == 2 else q.view(*x.shape[:-1], q.shape[-1])), scale
