"""Layers whose products run on 8-bit operands with one power-of-two scale for each block of 128.

    w8 = fp8.quantize(weight, 'tile')                    # once: a weight (out, in) held in 8 bits
    y = fp8.linear(x, w8, bias)                          # x quantised on the way, from one row to a whole image
    y = fp8.linear(x, weight, bias, activation='sine')   # training: forward and both backward products in 8 bits

A block is 128 values along the axis that a product sums over (activations, gradients: 'row') or 128 x 128 (weights:
'tile', which serve both directions). Its scale is the smallest power of two with which the largest finite magnitude is
at most 448; values are then rounded once, to the nearest e4m3 number. Sums, bias and sine are in 32 bits. NaN stays NaN
and infinities become NaN. BatchLinear, FCBlock, SingleBVPNet and HyperNetwork take it as precision='fp8'.

The kernels are gfx950 only (include/siren_amd.h, "8-bit training"): there is no CPU path. Calls are asynchronous on the
current stream of x's device and allocate from torch's caching allocator, so they can be captured into a graph. A captured
backward needs torch's own rule for captures: no eager graph of the same leaves alive while it is recorded.
"""
import ctypes
from typing import NamedTuple

import torch

from . import _lib

BLOCK = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FORMATS = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_ACTIVATIONS = {None: 0, 'sine': 1}


class Blocks(NamedTuple):
    """A (rows, cols) tensor in 8 bits: data (rows, cols rounded up to 128; the padding zero) in e4m3 or e5m2, scale
    (rows, or ceil(rows / 128) of a tiled tensor; ceil(cols / 512) * 4) exponent bytes: value * 2^(byte - 127)."""
    data: torch.Tensor
    scale: torch.Tensor
    cols: int

    @property
    def rows(self):
        return self.data.shape[-2]

    @property
    def tiled(self):
        # one row is both: its tile is its row block
        return self.scale.shape[0] != self.rows

    @property
    def layout(self):
        # what _quantize(panels=True) makes for a product is (cols / 64, rows, 64)
        return int(self.tiled) | (2 if self.data.dim() == 3 else 0)


def _p(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


class _On:
    """Makes a tensor's device current for a launch when it is not."""

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.device.index:
            torch.cuda.set_device(self.device)

    def __exit__(self, *exc):
        if self.before != self.device.index:
            torch.cuda.set_device(self.before)


def _check_input(x, what='x'):
    if not isinstance(x, torch.Tensor):
        raise TypeError('%s must be a torch.Tensor' % what)
    if x.device.type != 'cuda':
        raise RuntimeError('siren_amd.fp8 runs on ROCm devices (MI355X) only; got a %s tensor' % x.device.type)
    if x.dtype not in _DTYPES:
        raise TypeError('%s must be fp32, bf16 or fp16; got %s' % (what, x.dtype))


def _rows_of(x):
    """x as the kernels read it: columns one element apart, rows any non-overlapping distance."""
    if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]):
        return x, (x.stride(0) if x.shape[0] > 1 else x.shape[1])
    x = x.contiguous()
    return x, x.shape[1]


def _padded(n):
    return (n + 127) // 128 * 128


def _words(n):
    return (n + 511) // 512 * 4


def _quantize(x, tiles, straight=True, transposed=False, fmt=0, mult=None, colsum=False, panels=False):
    """(Blocks | None, Blocks | None of the transpose, column sums | None) of x (rows, cols) by one pass. panels: the
    values as the products read them best, (cols / 64, rows, 64)."""
    x, ld = _rows_of(x)
    rows, cols = x.shape
    dev, dtype = x.device, torch.float8_e5m2 if fmt else torch.float8_e4m3fn
    q = s = qt = st = ws = sums = None
    if straight:
        q = torch.empty(*((_padded(cols) // 64, rows, 64) if panels else (rows, _padded(cols))), dtype=dtype, device=dev)
        s = torch.empty((rows + 127) // 128 if tiles else rows, _words(cols), dtype=torch.uint8, device=dev)
    if transposed:
        qt = torch.empty(*((_padded(rows) // 64, cols, 64) if panels else (cols, _padded(rows))), dtype=dtype, device=dev)
        st = torch.empty((cols + 127) // 128 if tiles else cols, _words(rows), dtype=torch.uint8, device=dev)
    if colsum:
        ws = torch.empty((rows + 127) // 128, cols, device=dev)
        sums = torch.empty(cols, device=dev)
    lib = _lib.load()
    with _On(dev):
        _lib.check(lib.siren_fp8_quantize(_p(x), _DTYPES[x.dtype], rows, cols, ld, _p(mult), fmt, int(tiles), int(panels),
                                          _p(q), _p(s), _p(qt), _p(st), _p(ws), _p(sums), _stream(dev)), 'siren_fp8_quantize')
    return (Blocks(q, s, cols) if straight else None), (Blocks(qt, st, rows) if transposed else None), sums


def quantize(x, block='row', dtype=torch.float8_e4m3fn):
    """x (rows, cols), fp32, bf16 or fp16 -> Blocks quantised along the columns, with a scale per 1 x 128 ('row') or per
    128 x 128 ('tile'). dtype: torch.float8_e4m3fn or torch.float8_e5m2."""
    _check_input(x)
    if x.dim() != 2:
        raise ValueError('x must be (rows, cols); got %s' % (tuple(x.shape),))
    if block not in ('row', 'tile'):
        raise ValueError("block must be 'row' or 'tile'; got %r" % (block,))
    if dtype not in _FORMATS:
        raise TypeError('dtype must be torch.float8_e4m3fn or torch.float8_e5m2; got %s' % (dtype,))
    return _quantize(x.detach(), block == 'tile', fmt=_FORMATS[dtype])[0]


def dequantize(b):
    """The fp32 values (rows, cols) that Blocks stand for (elementary torch operations: not a hot path)."""
    rows, kb = b.data.shape[0], b.data.shape[1] // BLOCK
    byte = b.scale[:, :kb].to(torch.int32)
    s = torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)  # byte 0 is 2^-127, a subnormal number
    if b.tiled:
        s = s.repeat_interleave(BLOCK, 0)[:rows]
    return (b.data.float().view(rows, kb, BLOCK) * s[:, :, None]).view(rows, -1)[:, :b.cols]


def _product(a, b, bias, act, omega, out_dtype, deriv=False):
    """act(a b^T + bias) of two Blocks quantised along the summed axis, and omega cos(omega z) in bf16 if asked for."""
    m, n, dev = a.rows, b.rows, a.data.device
    out = torch.empty(m, n, dtype=out_dtype, device=dev)
    # the sine's derivative meets a gradient that is rounded to 3 bits of mantissa next: 8 bits of it are enough
    d = torch.empty(m, n, dtype=torch.bfloat16, device=dev) if deriv else None
    lib, need = _lib.load(), ctypes.c_int64()
    _lib.check(lib.siren_fp8_matmul_ws_bytes(m, n, a.cols, ctypes.byref(need)), 'siren_fp8_matmul_ws_bytes')
    ws = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
    with _On(dev):
        _lib.check(lib.siren_fp8_matmul(_p(a.data), _p(a.scale), m, a.layout, _FORMATS[a.data.dtype], _p(b.data),
                                        _p(b.scale), n, b.layout, a.cols, _p(bias), act, omega, _p(out),
                                        _DTYPES[out_dtype], _p(d), _p(ws), _stream(dev)), 'siren_fp8_matmul')
    return out, d


def _serve(x, w, bias, act, omega):
    """The forward alone, one call of the C ABI: x (m, k) of any of the three types, w Blocks (n, k) with tiles."""
    x, ld = _rows_of(x)
    (m, k), n, dev = x.shape, w.data.shape[0], x.device
    y = torch.empty(m, n, dtype=x.dtype, device=dev)
    lib, need = _lib.load(), ctypes.c_int64()
    _lib.check(lib.siren_fp8_linear_ws_bytes(m, n, k, ctypes.byref(need)), 'siren_fp8_linear_ws_bytes')
    ws = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
    with _On(dev):
        _lib.check(lib.siren_fp8_linear(_p(x), _DTYPES[x.dtype], m, k, ld, _p(w.data), _p(w.scale), n, _p(bias), act, omega,
                                        _p(y), _p(ws), _stream(dev)), 'siren_fp8_linear')
    return y


class _Linear(torch.autograd.Function):
    """y = act(x W^T + b) with gradients. x is read once in the forward and dy once in the backward, each quantised both
    along its rows and along its columns in that pass; the weight's tiles serve both directions."""

    @staticmethod
    def forward(ctx, x, weight, bias, act, omega, fmt):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        ctx.rows, ctx.widths, ctx.fmt = x.shape[0], tuple(weight.shape), fmt
        ctx.types = x.dtype, weight.dtype, None if bias is None else bias.dtype
        if not ctx.rows:  # an empty batch: no products, gradients of zero
            return x.new_empty(0, weight.shape[0])
        qx, qxt, _ = _quantize(x, False, transposed=need_w, panels=True)
        qw, qwt, _ = _quantize(weight, True, transposed=need_x, panels=True)
        y, deriv = _product(qx, qw, _bias32(bias), act, omega, x.dtype, deriv=act == 1 and (need_x or need_w or need_b))
        ctx.save_for_backward(*(qxt[:2] if need_w else ()), *(qwt[:2] if need_x else ()),
                              *((deriv,) if deriv is not None else ()))
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        (n, k), (xt, wt, bt) = ctx.widths, ctx.types
        if not ctx.rows:
            return (dy.new_empty(0, k) if need_x else None, dy.new_zeros(n, k, dtype=wt) if need_w else None,
                    dy.new_zeros(n, dtype=bt) if need_b else None, None, None, None)
        saved = list(ctx.saved_tensors)
        qxt = Blocks(saved.pop(0), saved.pop(0), ctx.rows) if need_w else None
        qwt = Blocks(saved.pop(0), saved.pop(0), n) if need_x else None
        deriv = saved.pop(0) if saved else None
        qd, qdt, sums = _quantize(dy, False, straight=need_x, transposed=need_w, fmt=ctx.fmt, mult=deriv, colsum=need_b,
                                  panels=True)
        dx = _product(qd, qwt, None, 0, 0., xt)[0] if need_x else None
        dw = _product(qdt, qxt, None, 0, 0., wt)[0] if need_w else None
        return dx, dw, (sums.to(bt) if need_b else None), None, None, None


def _bias32(bias):
    return None if bias is None else bias.detach().float().contiguous()


def _check_weight(weight, x):
    if isinstance(weight, Blocks):
        data, scale, k = weight
        if not isinstance(data, torch.Tensor) or not isinstance(scale, torch.Tensor):
            raise TypeError('Blocks hold tensors')
        if data.dtype != torch.float8_e4m3fn or scale.dtype != torch.uint8:
            raise TypeError('an 8-bit weight is e4m3 with uint8 scales; got %s and %s' % (data.dtype, scale.dtype))
        if data.dim() != 2 or scale.dim() != 2 or data.shape[1] != _padded(k) or \
                tuple(scale.shape) != ((data.shape[0] + 127) // 128, _words(k)):
            raise ValueError("an 8-bit weight is quantize(weight, 'tile'): data (n, %d), scale (ceil(n / 128), %d); got %s "
                             'and %s' % (_padded(k), _words(k), tuple(data.shape), tuple(scale.shape)))
        if not data.is_contiguous() or not scale.is_contiguous() or data.data_ptr() % 16 or scale.data_ptr() % 4:
            raise ValueError('an 8-bit weight must be contiguous, its data 16-byte and its scales 4-byte aligned')
        if data.device != x.device or scale.device != x.device:
            raise ValueError('weight on %s but x on %s' % (data.device, x.device))
        return data.shape[0], k
    _check_input(weight, 'weight')
    if weight.dim() != 2:
        raise _lib.SirenUnsupported('fp8.linear takes one weight (out, in); got %s' % (tuple(weight.shape),))
    if weight.device != x.device:
        raise ValueError('weight on %s but x on %s' % (weight.device, x.device))
    return weight.shape[0], weight.shape[1]


def linear(x, weight, bias=None, activation=None, omega=30., grad_dtype=torch.float8_e4m3fn):
    """act(x weight^T + bias): x (..., in) fp32, bf16 or fp16 -> (..., out) in x's type.

    weight: a tensor (out, in) of any of the three types, quantised on the way and differentiable, or Blocks from
    quantize(weight, 'tile') (a weight that stays in 8 bits: forward only). activation: None or 'sine', sin(omega z).
    The backward gives dx, dW and db; its gradients are rounded to grad_dtype (e4m3 or e5m2) and are not differentiable
    again. dW is quantised products of gradients and activations, so its relative error is that of e4m3's 3 bits."""
    _check_input(x)
    if x.dim() < 1:
        raise ValueError('x must be (..., in)')
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be None or 'sine'; got %r" % (activation,))
    if grad_dtype not in _FORMATS:
        raise TypeError('grad_dtype must be torch.float8_e4m3fn or torch.float8_e5m2; got %s' % (grad_dtype,))
    n, k = _check_weight(weight, x)
    if k < 1 or n < 1:
        raise ValueError('weight must have rows and columns; got (%d, %d)' % (n, k))
    if x.shape[-1] != k:
        raise ValueError('x must be (..., %d) for this weight; got %s' % (k, tuple(x.shape)))
    if bias is not None:
        _check_input(bias, 'bias')
        if tuple(bias.shape) != (n,) or bias.device != x.device:
            raise ValueError('bias must be (%d,) on %s; got %s on %s' % (n, x.device, tuple(bias.shape), bias.device))
    act, omega = _ACTIVATIONS[activation], float(omega)
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    packed = isinstance(weight, Blocks)
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad) or
                                    (not packed and weight.requires_grad)):
        if packed:
            raise RuntimeError('fp8.linear: a weight held in 8 bits is forward only; use torch.no_grad(), or pass the '
                               'weight itself to train')
        y = _Linear.apply(x2, weight, bias, act, omega, _FORMATS[grad_dtype])
    else:
        w = weight if packed else _quantize(weight.detach(), True)[0]
        y = _serve(x2.detach(), w, _bias32(bias), act, omega)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], n)
