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

BlockFP8Linear and BlockFP8GatedMLP hold such weights as layers, built from float ones (from_float, as the int8 Quantizer
layers are, quant/Weight_Only/Quantizer.py:93-112).

Forward only, like the rest of the package: results carry no gradient.  M is the number of rows, the product of all dimensions but the last.  An activation's scales are block-major ([blocks, M],
dense).  Codes are torch.float8_e4m3fn; the value of a code is code * scale.  include/miq.h states the formulas.
"""
import torch
import torch.nn as nn

from . import _native
from .qop import _to_gpu


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
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError(f"residual must be {tuple(x.shape)}, got {tuple(residual.shape)}")
    q, scale, total = _native.rms_norm_fp8(_rows(x), weight, eps, None if residual is None else _rows(residual))
    if x.dim() != 2:
        q, total = q.view(x.shape), None if total is None else total.view(x.shape)
    return (q, scale) if residual is None else (q, scale, total)


def linear_fp8(x, x_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16):
    """x [..., K] codes with their scales, times w [N, K] codes with theirs, plus bias [N] -> [..., N] of out_dtype.  Sums of more
    than 16 rows for a 16-bit out_dtype are off by some 3e-5 of the outputs' root mean square beside the output's own rounding
    (bfloat16 1.7e-3, float16 2.1e-4); float32 keeps 24 bits throughout, at half the matrix rate."""
    y = _native.gemm_fp8(_rows(x), x_scale, w, w_scale, bias, out_dtype)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[-1])


def gated_linear_fp8(x, x_scale, w_gate, gate_scale, w_up, up_scale, act="silu"):
    """The codes of act(x . w_gate^T) * (x . w_up^T): (codes [..., N], scales [ceil(N / 128), M]).  act: "silu" or "gelu"."""
    q, scale = _native.gated_fp8(_rows(x), x_scale, w_gate, gate_scale, w_up, up_scale, act)
    return (q if x.dim() == 2 else q.view(*x.shape[:-1], q.shape[-1])), scale


class _BlockFP8Module(nn.Module):
    """Codes and scales as buffers that keep their types: .half() or .to(torch.bfloat16) of a model moves them and no more
    (a scale rounded to 16 bits, or codes cast to another type, would be other weights)."""

    def _apply(self, fn, recurse=True):
        def moved(t):
            new = fn(t)
            return new if new.dtype == t.dtype else t.to(new.device)
        if recurse:
            for child in self.children():   # by their own rule
                child._apply(fn)
        return super()._apply(moved, recurse=False)

    @staticmethod
    def _codes(x):
        """The codes and scales of an activation: as they are (a pair, what a norm or a gated product returned) or of a float
        tensor.  Returns (codes, scales, the float type to answer in)."""
        if isinstance(x, (tuple, list)):
            return x[0], x[1], torch.bfloat16
        return (*quantize_blocks_fp8(x), x.dtype)


class BlockFP8Linear(_BlockFP8Module):
    """nn.Linear on block-scaled e4m3 codes.  forward() takes a float tensor (which it quantizes) or a pair (codes, scales); its
    output is of the layer's out_dtype, of forward()'s where the layer has none, else of the tensor's type, bfloat16 for a pair."""

    def __init__(self, weight, weight_scale, bias=None, out_dtype=None):
        super().__init__()
        self.out_features, self.in_features = weight.shape
        self.out_dtype = out_dtype
        self.register_buffer("weight", weight)
        self.register_buffer("weight_scale", weight_scale)
        self.register_buffer("bias", None if bias is None else bias.detach().to(torch.float32, copy=True).contiguous())

    @classmethod
    def from_float(cls, module, out_dtype=None):
        w, scale = quantize_weight_fp8(_to_gpu(module.weight.detach()).contiguous())
        home = module.weight.device
        return cls(w.to(home), scale.to(home), module.bias, out_dtype)

    def forward(self, x, out_dtype=None):
        q, scale, dtype = self._codes(x)
        return linear_fp8(q, scale, self.weight, self.weight_scale, self.bias, self.out_dtype or out_dtype or dtype)

    def extra_repr(self):
        return f"{self.in_features}, {self.out_features}, bias={self.bias is not None}"


class BlockFP8GatedMLP(_BlockFP8Module):
    """down(act(gate(x)) * up(x)) on block-scaled e4m3 codes, 8 bits between the products: two launches for a prompt (the
    gated product ends in codes), one more to quantize a float input.  forward() takes what BlockFP8Linear takes; rms_norm_fp8
    makes such a pair of a layer's input.  `down` is called as a module, down((codes, scales), out_dtype=the type to answer in),
    so that its hooks run and another module may stand in its place."""

    def __init__(self, gate, gate_scale, up, up_scale, down, act="silu"):
        super().__init__()
        if act not in _native._ACT_CODES:
            raise RuntimeError(f"unknown activation {act!r}: silu or gelu")
        self.act = act
        for name, t in (("gate", gate), ("gate_scale", gate_scale), ("up", up), ("up_scale", up_scale)):
            self.register_buffer(name, t)
        self.down = down

    @classmethod
    def from_float(cls, gate, up, down, act="silu", out_dtype=None):
        """gate, up, down: nn.Linear layers; the first two without a bias (it would have to be added before the activation)."""
        if gate.bias is not None or up.bias is not None:
            raise NotImplementedError("gate and up projections with a bias are not implemented")
        parts = []
        for m in (gate, up):
            parts += [t.to(m.weight.device) for t in quantize_weight_fp8(_to_gpu(m.weight.detach()).contiguous())]
        return cls(*parts, BlockFP8Linear.from_float(down, out_dtype), act)

    def forward(self, x):
        q, scale, dtype = self._codes(x)
        hidden = gated_linear_fp8(q, scale, self.gate, self.gate_scale, self.up, self.up_scale, self.act)
        return self.down(hidden, out_dtype=dtype)
