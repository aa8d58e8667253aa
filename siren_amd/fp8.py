"""Layers whose products run on 8-bit operands with one power-of-two scale for each block of 128.

    w8 = fp8.quantize(weight, 'tile')                    # once: a weight (out, in) held in 8 bits
    y = fp8.linear(x, w8, bias)                          # x quantised on the way, from one row to a whole image
    y = fp8.linear(x, weight, bias, activation='sine')   # training: forward and both backward products in 8 bits

A block is 128 values along the axis that a product sums over (activations, gradients: 'row') or 128 x 128 (weights:
'tile', which serve both directions). Its scale is the smallest power of two with which the largest finite magnitude is
at most 448; values are then rounded once, to the nearest e4m3 number. Sums, bias and sine are in 32 bits. NaN stays NaN
and infinities become NaN. The products are exact for blocks whose largest magnitude lies between 2^-116 and 2^128 (1 - 2^-5);
smaller blocks are held to multiples of 2^-133 there, a value that rounds to 2^128 is an infinity. BatchLinear, FCBlock, SingleBVPNet and HyperNetwork take it as precision='fp8'.

The kernels are gfx950 only (include/siren_amd.h, "8-bit training"): there is no CPU path. Calls are asynchronous on the
current stream of x's device and allocate from torch's caching allocator, so they can be captured into a graph. A captured
backward needs torch's own rule for captures: no eager graph of the same leaves alive while it is recorded.
"""
from typing import NamedTuple

import torch

from . import _lib

BLOCK = 128
_FORMATS = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_ACTIVATIONS = {None: 0, 'sine': 1}


class Blocks(NamedTuple):
    """A (rows, cols) tensor in 8 bits: data (rows, cols rounded up to 128; the padding zero) in e4m3 or e5m2, scale
    (rows, or ceil(rows / 128) of a tiled tensor; ceil(cols / 512) * 4) exponent bytes: value * 2^(byte - 127)."""
    data: torch.Tensor
    scale: torch.Tensor
    cols: int

    @property
    def tiled(self):
        # one row is both: its tile is its row block
        return self.scale.shape[0] != self.data.shape[0]


def _format(dtype, what='dtype'):
    if dtype not in _FORMATS:
        raise TypeError('%s must be torch.float8_e4m3fn or torch.float8_e5m2; got %s' % (what, dtype))
    return _FORMATS[dtype]


def _activation(activation):
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be None or 'sine'; got %r" % (activation,))
    return _ACTIVATIONS[activation]


def quantize(x, block='row', dtype=torch.float8_e4m3fn, transposed=False):
    """x (rows, cols), fp32, bf16 or fp16 -> Blocks quantised along the columns, with a scale per 1 x 128 ('row') or per
    128 x 128 ('tile'). dtype: torch.float8_e4m3fn or torch.float8_e5m2. transposed=True: (Blocks, Blocks of the (cols, rows)
    transpose, quantised along the rows), from one pass over x."""
    if block not in ('row', 'tile'):
        raise ValueError("block must be 'row' or 'tile'; got %r" % (block,))
    fmt, tiles = _format(dtype), block == 'tile'
    if not transposed:
        return Blocks(*_lib.native().quantize(x, tiles, fmt), x.shape[1])
    q, s, qt, st = _lib.native().quantize_both(x, tiles, fmt)
    return Blocks(q, s, x.shape[1]), Blocks(qt, st, x.shape[0])


def dequantize(b):
    """The fp32 values (rows, cols) that Blocks stand for (elementary torch operations: not a hot path)."""
    rows, kb = b.data.shape[0], b.data.shape[1] // BLOCK
    byte = b.scale[:, :kb].to(torch.int32)
    s = torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)  # byte 0 is 2^-127, a subnormal number
    if b.tiled:
        s = s.repeat_interleave(BLOCK, 0)[:rows]
    return (b.data.float().view(rows, kb, BLOCK) * s[:, :, None]).view(rows, kb * BLOCK)[:, :b.cols]


def matmul(a, b, bias=None, activation=None, omega=30., dtype=torch.float32, derivative=False):
    """act(a b^T + bias) of two Blocks (m, k) and (n, k), quantised along the axis they are summed over -> (m, n) in dtype
    (fp32, bf16 or fp16). a may be e5m2. derivative=True with the sine: also omega cos(omega z), in bf16. No gradients."""
    if not isinstance(a, Blocks) or not isinstance(b, Blocks):
        raise TypeError('matmul takes two Blocks (quantize)')
    if a.cols != b.cols:
        raise ValueError('a sums over %d columns, b over %d' % (a.cols, b.cols))
    act = _activation(activation)
    if derivative and not act:
        raise ValueError("derivative belongs to activation='sine'")
    y, d = _lib.native().matmul(a.data, a.scale, b.data, b.scale, a.cols, bias, act, omega, dtype, derivative)
    return (y, d) if derivative else y


def linear(x, weight, bias=None, activation=None, omega=30., grad_dtype=torch.float8_e4m3fn):
    """act(x weight^T + bias): x (..., in) fp32, bf16 or fp16 -> (..., out) in x's type.

    weight: a tensor (out, in) of any of the three types, quantised on the way and differentiable, or Blocks from
    quantize(weight, 'tile') (a weight that stays in 8 bits: forward only). activation: None or 'sine', sin(omega z).
    A layer has fewer than 2^22 outputs and, where x or the weight need gradients, fewer than 2^22 inputs (2^24 - 128 at
    most otherwise); a weight's gradient sums over at most 2^24 - 128 rows.
    The backward gives dx, dW and db; its gradients are rounded to grad_dtype (e4m3 or e5m2) and are not differentiable
    again. dW is quantised products of gradients and activations, so its relative error is that of e4m3's 3 bits. The sine's
    derivative omega cos(omega z) is kept in bf16 from the forward to the backward: each term of db is dy times that, off by
    2^-8 of itself at most, and summed in 32 bits."""
    act = _activation(activation)
    if isinstance(weight, Blocks):
        return _lib.native().linear_packed(x, weight.data, weight.scale, weight.cols, bias, act, omega)
    if isinstance(weight, torch.Tensor) and weight.dim() != 2:
        raise _lib.SirenUnsupported('fp8.linear takes one weight (out, in); got %s' % (tuple(weight.shape),))
    return _lib.native().linear(x, weight, bias, act, omega, _format(grad_dtype, 'grad_dtype'))
