"""The 8-bit layer products (siren_amd.fp8) against a 64-bit restatement of their definition: the quantiser's bytes
exactly, products within the rounding of a 32-bit sum, gradients from the quantised operands and against differences of
the layer itself. Needs an MI355X."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


# ---- the definition, in 64 bits on the CPU -----------------------------------------------------------------------------
def grid(top, mant, emin):
    """A format as (largest value, mantissa bits, exponent of the smallest normal number)."""
    return top, mant, emin


FORMATS = {E4M3: grid(448., 3, -6), E5M2: grid(57344., 2, -14)}


def round_blocks(v, fmt):
    """(values that 8 bits hold, exponent bytes) of the blocks along v's last axis (numpy float64)."""
    top, mant, emin = FORMATS[fmt]
    fin = np.where(np.isfinite(v), np.abs(v), 0.).max(-1, keepdims=True)
    f, e = np.frexp(fin / top)
    e = np.where(f > 0, np.maximum(np.where(f > 0.5, e, e - 1), -126), -126)
    s = np.ldexp(1., e)
    with np.errstate(invalid='ignore'):
        u = v / s
        step = np.ldexp(1., np.maximum(np.frexp(np.where(np.isfinite(u), u, 0.))[1] - 1, emin) - mant)
        out = np.rint(u / step) * step * s
    if fmt is E4M3:
        out = np.where(np.isfinite(v), out, np.nan)
    return out, (e + 127)[..., 0].astype(np.int64)


def held(x, fmt=E4M3, tiles=False):
    """(rows, cols) -> (values, bytes) quantised along the columns."""
    x = np.asarray(x, np.float64)
    r, c = x.shape
    pc, pr = -c % 128, -r % 128
    if not tiles:
        v, b = round_blocks(np.pad(x, ((0, 0), (0, pc))).reshape(r, -1, 128), fmt)
        return v.reshape(r, -1)[:, :c], b
    t = np.pad(x, ((0, pr), (0, pc)))
    nb, kb = t.shape[0] // 128, t.shape[1] // 128
    v, b = round_blocks(t.reshape(nb, 128, kb, 128).transpose(0, 2, 1, 3).reshape(nb, kb, -1), fmt)
    return v.reshape(nb, kb, 128, 128).transpose(0, 2, 1, 3).reshape(nb * 128, -1)[:r, :c], b


def np64(t):
    return t.detach().double().cpu().numpy()


HALF = {torch.float32: 2. ** -24, torch.bfloat16: 2. ** -8, torch.float16: 2. ** -11}
TINY = {torch.float32: 2. ** -149, torch.bfloat16: 2. ** -133, torch.float16: 2. ** -25}


def product_tol(a, b, out, dtype, extra=0.):
    """A sum of k exact products and a bias in 32 bits, in any order: at most (k + 2) roundings of half a step, each of at
    most the sum of magnitudes; then one rounding to dtype."""
    k = a.shape[1]
    return (k + 2) * 2. ** -24 * (np.abs(a) @ np.abs(b).T + extra) + HALF[dtype] * np.abs(out) + TINY[dtype]


def check(got, want, tol, what):
    got = np64(got)
    assert got.shape == want.shape, what
    bad = np.abs(got - want) > tol
    assert not bad.any(), '%s: %d of %d off, worst %.3g of its tolerance' % (
        what, bad.sum(), bad.size, (np.abs(got - want) / tol).max())


def values(shape, seed, scale=1.):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g) * torch.exp(torch.randn(shape[0], 1, generator=g)) * scale


# ---- the quantiser -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('rows,cols', [(1, 1), (1, 128), (3, 100), (128, 129), (130, 640), (257, 1025)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('block', ['row', 'tile'])
@pytest.mark.parametrize('fmt', [E4M3, E5M2])
def test_quantize_is_the_definition(cuda, rows, cols, dtype, block, fmt):
    from siren_amd import fp8
    x = values((rows, cols), rows * 7 + cols).to(dtype)
    b = fp8.quantize(x.to(cuda), block, fmt)
    want, byte = held(np64(x), fmt, block == 'tile')
    assert b.data.dtype == fmt and b.data.shape == (rows, (cols + 127) // 128 * 128)
    assert b.scale.shape == (((rows + 127) // 128 if block == 'tile' else rows), (cols + 511) // 512 * 4)
    kb = (cols + 127) // 128
    assert np.array_equal(b.scale.cpu().numpy()[:, :kb], byte)
    assert (b.scale[:, kb:] == 127).all() and (b.data[:, cols:].float() == 0).all()
    assert np.array_equal(np64(fp8.dequantize(b)), want)
    assert b.tiled == (block == 'tile' and rows > 1)


def test_quantize_special_values(cuda):
    """Zeros, subnormals, the format's borders and values that are not finite, in blocks of their own."""
    from siren_amd import fp8
    x = torch.zeros(8, 256)
    x[1, :3] = torch.tensor([448., 449., -1.])
    x[2, :4] = torch.tensor([float('inf'), 1., float('-inf'), float('nan')])
    x[3, 0], x[3, 1] = 2. ** -149, -2. ** -126
    x[4, 0], x[4, 1] = torch.finfo(torch.float32).max, 1.
    x[5, :] = float('nan')
    x[6, :128] = torch.arange(128) * 2. ** -9
    x[7, :2] = torch.tensor([-0., 2. ** -120])
    for fmt in (E4M3, E5M2):
        b = fp8.quantize(x.to(cuda), 'row', fmt)
        want, byte = held(x.double().numpy(), fmt)
        assert np.array_equal(b.scale.cpu().numpy()[:, :2], byte)
        # the largest fp32 number, 2^128 (1 - 2^-24), rounds to 2^128, which fp32 values hold as an infinity only
        with np.errstate(over='ignore'):
            want = want.astype(np.float32).astype(np.float64)
        assert np.array_equal(np64(fp8.dequantize(b)), want, equal_nan=True)


@pytest.mark.parametrize('rows,cols', [(1, 130), (200, 70), (128, 128), (129, 1), (1, 1), (300, 515)])
@pytest.mark.parametrize('block', ['row', 'tile'])
def test_both_directions_in_one_pass(cuda, rows, cols, block):
    """The transpose is the quantised transpose."""
    from siren_amd import fp8
    x = values((rows, cols), 5)
    for b, v in zip(fp8.quantize(x.to(cuda), block, transposed=True), (x.numpy(), x.numpy().T)):
        want, byte = held(v, E4M3, block == 'tile')
        assert np.array_equal(np64(fp8.dequantize(b)), want)
        assert np.array_equal(b.scale.cpu().numpy()[:, :byte.shape[1]], byte)
        assert (b.scale[:, byte.shape[1]:] == 127).all() and (b.data[:, v.shape[1]:].float() == 0).all()


@pytest.mark.parametrize('view', ['strided', 'offset', 'transposed', 'expanded', 'wide'])
def test_quantize_reads_views(cuda, view):
    from siren_amd import fp8
    base = values((300, 400), 9).to(cuda)
    x = {'strided': base[:, ::2], 'offset': base[1:, 3:200], 'transposed': base.t(), 'expanded': base[:1].expand(9, 400),
         'wide': base[::3]}[view]
    assert np.array_equal(np64(fp8.dequantize(fp8.quantize(x))), held(np64(x))[0])


# ---- the forward -------------------------------------------------------------------------------------------------------
def layer(m, k, n, dtype, cuda, seed=0):
    x = torch.sin(values((m, k), seed)).to(dtype)
    g = torch.Generator().manual_seed(seed + 1)
    w = (torch.rand(n, k, generator=g) * 2 - 1) * math.sqrt(6 / k) / 30
    b = (torch.rand(n, generator=g) * 2 - 1) / math.sqrt(k)
    return x.to(cuda), w.to(cuda), b.to(cuda)


SIZES = [(1, 1, 1), (1, 256, 512), (2, 128, 128), (3, 100, 257), (15, 257, 130), (17, 64, 1), (32, 256, 1024), (33, 1024, 320),
         (129, 4096, 65), (130, 129, 127), (300, 640, 385), (1000, 384, 513)]


@pytest.mark.parametrize('m,k,n', SIZES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('act', [None, 'sine'])
def test_linear_forward(cuda, m, k, n, dtype, act):
    from siren_amd import fp8
    x, w, b = layer(m, k, n, dtype, cuda, m + k + n)
    y = fp8.linear(x, fp8.quantize(w, 'tile'), b, activation=act)
    assert y.dtype == dtype and y.shape == (m, n)
    xq, wq = held(np64(x))[0], held(np64(w), tiles=True)[0]
    z = xq @ wq.T + np64(b)
    if act is None:
        check(y, z, product_tol(xq, wq, z, dtype, np.abs(np64(b))), 'y')
    else:  # the phase is rounded once more, the sine to 2^-22
        tol = 30 * product_tol(xq, wq, 0 * z, torch.float32, np.abs(np64(b))) + np.abs(30 * z) * 2. ** -23 + 2. ** -22
        check(y, np.sin(30 * z), tol + HALF[dtype] * np.abs(np.sin(30 * z)) + TINY[dtype], 'sin')
    assert torch.equal(y, fp8.linear(x, w, b, activation=act)), 'a weight quantised on the way is the same'
    assert torch.equal(y, fp8.linear(x, fp8.quantize(w, 'tile'), b, activation=act)), 'the same call, the same result'


def test_linear_shapes_bias_and_omega(cuda):
    from siren_amd import fp8
    x, w, b = layer(60, 96, 40, torch.float32, cuda)
    w8 = fp8.quantize(w, 'tile')
    y = fp8.linear(x, w8, b, 'sine', omega=7.)
    assert torch.equal(fp8.linear(x.view(3, 4, 5, 96), w8, b, 'sine', omega=7.).view(60, 40), y)
    assert torch.equal(fp8.linear(x[7], w8, b, 'sine', omega=7.), y[7])
    assert fp8.linear(x[:0], w8, b).shape == (0, 40)
    z = fp8.linear(x, w8)
    assert torch.allclose(torch.sin(7 * (z + b)), y, atol=1e-5)
    assert torch.equal(fp8.linear(x, w8, b.bfloat16()), fp8.linear(x, w8, b.bfloat16().float()))
    strided = torch.empty(60, 200, device=cuda)[:, 3:99].copy_(x)
    assert torch.equal(fp8.linear(strided, w8, b, 'sine', omega=7.), y)


def test_linear_not_finite(cuda):
    """A NaN or an infinity spoils its own row of y and no other."""
    from siren_amd import fp8
    x, w, b = layer(40, 300, 200, torch.float32, cuda)
    y = fp8.linear(x, w, b)
    x[3, 7], x[20, 299] = float('nan'), float('inf')
    z = fp8.linear(x, w, b)
    keep = torch.ones(40, dtype=torch.bool, device=cuda)
    keep[3] = keep[20] = False
    assert torch.isnan(z[~keep]).all() and torch.equal(z[keep], y[keep])


@pytest.mark.parametrize('m,k,n', [(1, 1, 1), (70, 300, 130), (260, 1100, 257), (40, 5000, 30)])
def test_matmul(cuda, m, k, n):
    """Two quantised operands, either in rows or tiles, the first in either format."""
    from siren_amd import fp8
    a, b = values((m, k), 1).to(cuda), values((n, k), 2).to(cuda)
    bias = values((1, n), 3)[0].to(cuda)
    for fmt in (E4M3, E5M2):
        for ba in ('row', 'tile'):
            for bb in ('row', 'tile'):
                aq, bq = held(np64(a), fmt, ba == 'tile')[0], held(np64(b), tiles=bb == 'tile')[0]
                z = aq @ bq.T + np64(bias)
                for dtype in (torch.float32, torch.bfloat16):
                    y = fp8.matmul(fp8.quantize(a, ba, fmt), fp8.quantize(b, bb), bias, dtype=dtype)
                    check(y, z, product_tol(aq, bq, z, dtype, np.abs(np64(bias))), (fmt, ba, bb))
    with pytest.raises(ValueError):
        fp8.matmul(fp8.quantize(a), fp8.quantize(torch.cat([b, b], 1)))
    with pytest.raises(TypeError):
        fp8.matmul(fp8.quantize(a), fp8.quantize(b, dtype=E5M2))
    with pytest.raises(TypeError):
        fp8.matmul(a, b)
    with pytest.raises(ValueError):
        fp8.matmul(fp8.quantize(a), fp8.quantize(b), derivative=True)


def test_linear_refuses(cuda):
    from siren_amd import fp8
    from siren_amd._lib import SirenUnsupported
    x, w, b = layer(5, 200, 300, torch.float32, cuda)
    w8 = fp8.quantize(w, 'tile')
    for bad in (dict(x=x[:, :100]), dict(bias=b[:4]), dict(bias=b.cpu()), dict(activation='relu'), dict(omega=float('nan')),
                dict(weight=fp8.quantize(w)), dict(weight=fp8.Blocks(w8.data[:, :128], w8.scale, 200)),
                dict(weight=fp8.Blocks(w8.data, w8.scale[:, :2], 200)), dict(weight=fp8.Blocks(w8.data, w8.scale, 100)),
                dict(weight=fp8.Blocks(w8.data.t().contiguous().t(), w8.scale, 200))):
        with pytest.raises((ValueError, RuntimeError)):
            fp8.linear(**{**dict(x=x, weight=w8, bias=b), **bad})
    for bad in (dict(x=x.double()), dict(x=x.int()), dict(weight=w.double()), dict(grad_dtype=torch.float16),
                dict(weight=fp8.quantize(w, 'tile', E5M2)), dict(weight=fp8.Blocks(w8.data, w8.scale.int(), 200))):
        with pytest.raises(TypeError):
            fp8.linear(**{**dict(x=x, weight=w, bias=b), **bad})
    with pytest.raises(SirenUnsupported):
        fp8.linear(x, w[None])
    with pytest.raises(ValueError):
        fp8.quantize(x, 'column')
    with pytest.raises(ValueError):
        fp8.quantize(x[0])


# ---- gradients ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('m,k,n', [(1, 1, 1), (1, 256, 300), (32, 256, 1024), (33, 130, 64), (129, 257, 130), (1500, 192, 320)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('fmt', [E4M3, E5M2])
def test_linear_gradients(cuda, m, k, n, dtype, fmt):
    """dx, dW and db are the products of the operands as 8 bits hold them."""
    from siren_amd import fp8
    x, w, b = layer(m, k, n, dtype, cuda, 3)
    dy = values((m, n), 4, 1 / 64).to(dtype).to(cuda)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = fp8.linear(x, w, b, grad_dtype=fmt)
    with torch.no_grad():
        assert torch.equal(y, fp8.linear(x, w, b))
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert dx.dtype == dtype and dw.dtype == torch.float32 and db.dtype == torch.float32
    d = np64(dy)
    wq, dq = held(np64(w), tiles=True)[0], held(d, fmt)[0]
    check(dx, dq @ wq, product_tol(dq, wq.T, dq @ wq, dtype), 'dx')
    dqt, xqt = held(d.T, fmt)[0], held(np64(x).T)[0]
    check(dw, dqt @ xqt.T, product_tol(dqt, xqt, dqt @ xqt.T, torch.float32), 'dw')
    check(db, d.sum(0), 24 * 2. ** -24 * np.abs(d).sum(0) + 2. ** -149, 'db')
    # one gradient at a time is the same gradient
    for i, g in enumerate((dx, dw, db)):
        ts = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(fp8.linear(*ts, grad_dtype=fmt), ts[i], dy)[0], g)


def test_sine_gradients(cuda):
    """The sine's gradient is dy omega cos(omega z), the cosine held in bf16, then the linear layer's."""
    from siren_amd import fp8
    m, k, n = 200, 192, 260
    x, w, b = layer(m, k, n, torch.float32, cuda, 8)
    dy = values((m, n), 4, 1 / 64).to(cuda)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(fp8.linear(x, w, b, 'sine'), leaves, dy)
    xq, wq = held(np64(x))[0], held(np64(w), tiles=True)[0]
    z = xq @ wq.T + np64(b)
    _, deriv = fp8.matmul(fp8.quantize(x), fp8.quantize(w, 'tile'), b, 'sine', derivative=True)
    tol = 30 * (30 * product_tol(xq, wq, 0 * z, torch.float32, np.abs(np64(b))) + np.abs(30 * z) * 2. ** -23 + 2. ** -22)
    check(deriv, 30 * np.cos(30 * z), tol + 2. ** -8 * np.abs(30 * np.cos(30 * z)), 'derivative')
    g = (dy * deriv.float()).cpu().double().numpy()
    gq, gqt, xqt = held(g)[0], held(g.T)[0], held(np64(x).T)[0]
    check(dx, gq @ wq, product_tol(gq, wq.T, gq @ wq, torch.float32), 'dx')
    check(dw, gqt @ xqt.T, product_tol(gqt, xqt, gqt @ xqt.T, torch.float32), 'dw')
    check(db, g.sum(0), 24 * 2. ** -24 * np.abs(g).sum(0) + 2. ** -149, 'db')


@pytest.mark.parametrize('act', [None, 'sine'])
def test_gradients_against_differences(cuda, act):
    """Along random directions the gradients are those of the layer without 8 bits (central differences in 64), up to what
    rounding each operand can do: an e4m3 value is off by 2^-4 of itself or 2^-10 of its block's scale, at most
    2 amax / 448; a bf16 cosine by 2^-8; the phase's error moves the sine's own derivative by omega^2 |dz|."""
    from siren_amd import fp8
    m, k, n = 24, 140, 150
    x, w, b = layer(m, k, n, torch.float32, cuda, 21)
    dy = values((m, n), 22, 1 / 8).to(cuda)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    got = [np64(g) for g in torch.autograd.grad(fp8.linear(x, w, b, act), leaves, dy)]
    X, W, B, D = (np64(t) for t in (x, w, b, dy))

    def off(a):
        return 2. ** -4 * np.abs(a) + 2. ** -10 * np.abs(a).max() / 224

    z = X @ W.T + B
    dz = off(X) @ np.abs(W).T + np.abs(X) @ off(W).T + off(X) @ off(W).T + 1e-5
    if act == 'sine':
        G = D * 30 * np.cos(30 * z)
        eg = np.abs(D) * (30 * np.minimum(30 * dz, 2.) + 30 * 2. ** -8)
    else:
        G, eg = D, 0 * D
    eq = eg + 2. ** -4 * (np.abs(G) + eg) + 2. ** -10 * (np.abs(G) + eg).max() / 224
    tols = [eq @ np.abs(W) + np.abs(G) @ off(W) + eq @ off(W), eq.T @ np.abs(X) + np.abs(G).T @ off(X) + eq.T @ off(X), eg.sum(0)]

    def loss(X, W, B):
        y = X @ W.T + B
        return (D * (np.sin(30 * y) if act == 'sine' else y)).sum()

    rng = np.random.default_rng(0)
    for i, (g, t) in enumerate(zip(got, tols)):
        for _ in range(4):
            v = rng.normal(size=g.shape)
            h = 1e-5
            lo, hi = [X, W, B], [X, W, B]
            lo[i], hi[i] = lo[i] - h * v, hi[i] + h * v
            diff = (loss(*hi) - loss(*lo)) / (2 * h)
            bound = (t * np.abs(v)).sum() + 1e-4 * np.abs(diff) + 1e-6 * np.abs(G).sum()
            assert abs((g * v).sum() - diff) <= bound, (i, (g * v).sum(), diff, bound)


def test_empty_batch_and_broadcast_gradient(cuda):
    from siren_amd import fp8
    x, w, b = layer(9, 40, 30, torch.float32, cuda)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(fp8.linear(x[:0], w, b).sum(), leaves)
    assert not dx.any() and not dw.any() and not db.any()
    one = torch.autograd.grad(fp8.linear(x, w, b).sum(), leaves)  # dy is one number, expanded
    two = torch.autograd.grad(fp8.linear(x, w, b), leaves, torch.ones(9, 30, device=cuda))
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    shared = fp8.linear(x, w, b) + fp8.linear(x * 2, w, b)  # a weight used twice: its gradients add
    dw2, = torch.autograd.grad(shared, w, torch.ones(9, 30, device=cuda))
    assert torch.allclose(dw2, 3 * two[1], rtol=0.2, atol=1e-3)


def test_second_derivatives_and_packed_gradients_are_refused(cuda):
    from siren_amd import fp8
    x, w, b = layer(9, 40, 30, torch.float32, cuda)
    w8 = fp8.quantize(w, 'tile')
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match='forward only'):
        fp8.linear(x, w8, b)
    with torch.no_grad():
        fp8.linear(x, w8, b)
    g, = torch.autograd.grad(fp8.linear(x, w, b).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---- streams, graphs, long offsets -------------------------------------------------------------------------------------
def test_streams_and_graphs(cuda):
    """Calls on a side stream and captured calls replayed on new inputs; two graphs share nothing."""
    from siren_amd import fp8
    x, w, b = layer(70, 1100, 200, torch.float32, cuda)
    w8 = fp8.quantize(w, 'tile')
    want = [fp8.linear(x * s, w8, b, 'sine') for s in (1., 0.5, 0.25)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(fp8.linear(x, w8, b, 'sine'), want[0])
    torch.cuda.synchronize()
    graphs, ins, outs = [], [], []
    for s in (1., 0.5):
        xin = (x * s).clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = fp8.linear(xin, w8, b, 'sine')
        graphs.append(g), ins.append(xin), outs.append(y)
    for _ in range(3):
        graphs[0].replay(), graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        torch.randn(1000, device=cuda).sum().item()
    ins[0].copy_(x * 0.25)
    graphs[0].replay()
    assert torch.equal(outs[0], want[2])


def test_captured_training_step(cuda):
    from siren_amd import fp8
    x, w, b = layer(260, 300, 140, torch.float32, cuda)
    dy = values((260, 140), 2).to(cuda)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(fp8.linear(x, w, b, 'sine'), leaves, dy)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(fp8.linear(x, w, b, 'sine'), leaves, dy)
    for _ in range(3):
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_capture_beside_an_eager_graph_is_refused(cuda):
    """A capture whose leaf an eager graph still holds is refused before the engine could meet it, and works once that graph
    is gone. (A graph made on the capturing stream itself is no obstacle.)"""
    from siren_amd import fp8
    x, w, b = layer(40, 64, 64, torch.float32, cuda)
    w.requires_grad_(True)
    eager = fp8.linear(x, w, b)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match='eager graph'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fp8.linear(x, w, b)
    want, = torch.autograd.grad(eager.sum(), w)
    del eager
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = fp8.linear(x, w, b) + fp8.linear(x, w, b)  # the capture's own graph of the leaf is no obstacle
        got, = torch.autograd.grad(y, w, torch.ones_like(y))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, 2 * want)


def test_offsets_past_32_bits(cuda):
    """Rows whose bytes, and outputs whose elements, begin past 2^32."""
    from siren_amd import fp8
    m, k, n = (1 << 21) + 3, 260, 2100
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda)
    g = torch.Generator(device='cuda').manual_seed(0)
    some = torch.cat([torch.arange(5), torch.tensor([m // 2]), torch.arange(m - 200, m)]).to(cuda)
    x[some] = torch.randn(some.numel(), k, generator=g, device=cuda).bfloat16()
    w8 = fp8.quantize(torch.randn(n, k, generator=g, device=cuda), 'tile')
    assert m * n > 1 << 32
    y = fp8.linear(x, w8)
    assert torch.equal(y[some], fp8.linear(x[some], w8))
    assert not y[1000:2000].any()


# ---- in the modules ----------------------------------------------------------------------------------------------------
def test_rows_of_a_batch_do_not_depend_on_it(cuda):
    """One row, a few and many take different kernels; a row's result may differ by the order of its sums only."""
    from siren_amd import fp8
    x, w, b = layer(700, 1000, 300, torch.float32, cuda)
    w8 = fp8.quantize(w, 'tile')
    y = fp8.linear(x, w8, b)
    xq, wq = held(np64(x))[0], held(np64(w), tiles=True)[0]
    tol = 2 * product_tol(xq, wq, np64(y), torch.float32, np.abs(np64(b)))
    for m in (1, 2, 5, 16, 17, 31, 32, 33, 64, 65, 128, 129, 257):
        check(fp8.linear(x[:m], w8, b), np64(y)[:m], tol[:m], m)


@pytest.mark.parametrize('m', [3, 40, 600])
def test_sine_of_what_is_not_finite(cuda, m):
    """sin(omega z) and its derivative of an infinite or NaN z are NaN, and a huge one's stay within 1 and omega."""
    from siren_amd import fp8
    w = torch.ones(5, 70, device=cuda)
    bias = torch.tensor([math.inf, -math.inf, math.nan, 1e38, 0.], device=cuda)
    x = torch.full((m, 70), 0.01, device=cuda)
    y, d = fp8.matmul(fp8.quantize(x), fp8.quantize(w, 'tile'), bias, 'sine', omega=2., derivative=True)
    for got, top in ((y, 1.), (d.float(), 2.), (fp8.linear(x, fp8.quantize(w, 'tile'), bias, 'sine', omega=2.), 1.)):
        assert bool(got[:, :3].isnan().all())
        assert bool((got[:, 3:].abs() <= top).all())


@pytest.mark.parametrize('m', [5, 200])
@pytest.mark.parametrize('act', [None, 'sine'])
def test_graph_is_used_as_any_other(cuda, m, act):
    """Parts of the gradients, a graph kept for two backward passes and refused a third, leaves that accumulate, hooks on what
    is saved and recomputation: the same bytes each time."""
    from torch.utils.checkpoint import checkpoint
    from siren_amd import fp8
    x, w, b = (torch.randn(*s, device=cuda, requires_grad=True) for s in ((m, 130), (70, 130), (70,)))
    dy = torch.randn(m, 70, device=cuda)
    y = fp8.linear(x, w, b, act)
    want = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    for i, leaf in enumerate((x, w, b)):
        assert torch.equal(torch.autograd.grad(y, (leaf,), dy, retain_graph=True)[0], want[i])
    y.backward(dy)
    with pytest.raises(RuntimeError, match='second time'):
        y.backward(dy)
    assert all(torch.equal(leaf.grad, g) for leaf, g in zip((x, w, b), want))
    fp8.linear(x, w, b, act).backward(dy)
    assert all(torch.equal(leaf.grad, 2 * g) for leaf, g in zip((x, w, b), want))
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.numel()) or t, lambda t: t):
        y = fp8.linear(x, w, b, act)
    assert len(seen) == (2 if act else 1)
    assert all(torch.equal(p, g) for p, g in zip(torch.autograd.grad(y, (x, w, b), dy), want))
    y = checkpoint(lambda *a: fp8.linear(*a, act), x, w, b, use_reentrant=False)
    assert all(torch.equal(p, g) for p, g in zip(torch.autograd.grad(y, (x, w, b), dy), want))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,cols,ld', [(200, 3, 3), (131, 6, 7), (129, 131, 131), (40, 66, 1 << 25), (3, 2, (1 << 25) + 1)])
def test_quantize_at_any_address(cuda, dtype, rows, cols, ld):
    """Rows that begin anywhere, narrow ones, and ones too far apart for 32-bit offsets: both layouts, and what a sine layer's
    backward multiplies and sums on the way, as of a plain copy."""
    from siren_amd import fp8
    if dtype is torch.float32 and ld > 1000:
        rows = min(rows, 20)  # a few GB
    base = torch.zeros((rows - 1) * ld + cols + 3, dtype=dtype, device=cuda)
    for shift in range(3):
        x = base[shift:].as_strided((rows, cols), (ld, 1))
        x.copy_(torch.randn(rows, cols, device=cuda))
        for block in ('row', 'tile'):
            for a, b in zip(fp8.quantize(x, block, transposed=True), fp8.quantize(x.clone(), block, transposed=True)):
                assert torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8)) and torch.equal(a.scale, b.scale)
            want = held(np64(x), tiles=block == 'tile')[0]
            assert np.array_equal(np64(fp8.dequantize(fp8.quantize(x, block))), want)
        w = torch.randn(cols, 9, device=cuda, requires_grad=True)
        b = torch.randn(cols, device=cuda, requires_grad=True)
        h = torch.randn(rows, 9, device=cuda).to(dtype).requires_grad_(True)
        grads = [torch.autograd.grad(fp8.linear(h, w, b, 'sine'), (h, w, b), dy) for dy in (x, x.clone())]
        assert all(torch.equal(p, q) for p, q in zip(*grads))


@pytest.mark.parametrize('m,n,k', [(33, 200, 700), (200, 200, 1024), (65, 64, 30000), (700, 700, 5000), (2000, 1000, 4096),
                                   (833, 321, 50001), (1024, 1024, 131072), (1000, 1023, 140000)])
def test_long_sums_are_exact(cuda, m, n, k):
    """Small whole numbers, which e4m3 holds and whose sums 32 bits hold: every way of splitting the sum gives them exactly."""
    from siren_amd import fp8
    g = torch.Generator(device=cuda).manual_seed(k)
    a = torch.randint(-3, 4, (m, k), generator=g, device=cuda)
    b = torch.randint(-3, 4, (n, k), generator=g, device=cuda)
    a[:, ::128], b[:, ::128] = 4, 4  # no block's scale is below 1/64: all values stay whole
    out = fp8.matmul(fp8.quantize(a.float()), fp8.quantize(b.float()))
    want = sum(a[:, c:c + 16384].double() @ b[:, c:c + 16384].double().t().contiguous() for c in range(0, k, 16384))
    assert torch.equal(out.double(), want)


def test_forward_mode_is_refused(cuda):
    import torch.autograd.forward_ad as fwd
    from siren_amd import fp8
    x, w, b = torch.randn(5, 130, device=cuda), torch.randn(70, 130, device=cuda), torch.randn(70, device=cuda)
    w8 = fp8.quantize(w, 'tile')
    with fwd.dual_level():
        for call in (lambda: fp8.linear(fwd.make_dual(x, x), w, b), lambda: fp8.linear(x, fwd.make_dual(w, w), b),
                     lambda: fp8.linear(x, w, fwd.make_dual(b, b)), lambda: fp8.linear(fwd.make_dual(x, x), w8),
                     lambda: fp8.quantize(fwd.make_dual(x, x))):
            with pytest.raises(RuntimeError, match='tangent'):
                call()
        fp8.linear(x, w, b)


def test_saved_tensors_elsewhere(cuda):
    """Hooks that keep what is saved on the host and bring it back: the same gradients; brought back wrong, an error."""
    from siren_amd import fp8
    x, w, b = (torch.randn(*s, device=cuda, requires_grad=True) for s in ((50, 130), (70, 130), (70,)))
    dy = torch.randn(50, 70, device=cuda)
    want = torch.autograd.grad(fp8.linear(x, w, b, 'sine'), (x, w, b), dy)
    with torch.autograd.graph.save_on_cpu():
        y = fp8.linear(x, w, b, 'sine')
    assert all(torch.equal(p, g) for p, g in zip(torch.autograd.grad(y, (x, w, b), dy), want))
    for wrong in (lambda t: t.cpu(), lambda t: t[:-1], lambda t: t.float(), lambda t: torch.cat([t, t])[::2]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, wrong):
            y = fp8.linear(x, w, b, 'sine')
        with pytest.raises(RuntimeError, match='saved tensor came back'):
            torch.autograd.grad(y, (x, w, b), dy)


@pytest.mark.parametrize('m', [5, 200])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('needs', [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (1, 0, 1)])
def test_gradients_of_some_leaves(cuda, m, dtype, needs):
    """Each leaf's gradient is the same bytes whichever others there are."""
    from siren_amd import fp8
    made = [torch.randn(*s, device=cuda) for s in ((m, 130), (70, 130), (70,))]
    made[0] = made[0].to(dtype)
    dy = torch.randn(m, 70, device=cuda).to(dtype)
    for act in (None, 'sine'):
        all_ = [t.clone().requires_grad_(True) for t in made]
        want = torch.autograd.grad(fp8.linear(*all_, act), all_, dy)
        some = [t.clone().requires_grad_(bool(n)) for t, n in zip(made, needs)]
        fp8.linear(*some, act).backward(dy)
        for t, g, n in zip(some, want, needs):
            assert torch.equal(t.grad, g) if n else t.grad is None


@pytest.mark.parametrize('m', [1, 4, 5, 9, 16, 17, 32, 33])
@pytest.mark.parametrize('k,n', [(513, 40), (1024, 300), (1025, 16384), (2048, 16385), (2049, 17), (4100, 70), (8192, 33), (8193, 129)])
def test_few_rows_of_long_sums(cuda, m, k, n):
    """Small whole numbers again: however few rows share out a long sum, it is exact; and a sine of it as a plain product's."""
    from siren_amd import fp8
    g = torch.Generator(device=cuda).manual_seed(m * k + n)
    x = torch.randint(-3, 4, (m, k), generator=g, device=cuda).float()
    w = torch.randint(-3, 4, (n, k), generator=g, device=cuda).float()
    x[:, ::128], w[:, ::128] = 4., 4.
    b = torch.randint(-9, 9, (n,), generator=g, device=cuda).float()
    w8 = fp8.quantize(w, 'tile')
    want = x.double() @ w.double().t().contiguous() + b
    assert torch.equal(fp8.linear(x, w8, b).double(), want)
    y = fp8.linear(x.bfloat16(), w8, b)
    assert y.dtype is torch.bfloat16 and torch.equal(y, want.float().bfloat16())
    plain = fp8.matmul(fp8.quantize(x), w8, b, 'sine', omega=0.01)
    assert torch.equal(fp8.linear(x, w8, b, 'sine', omega=0.01), plain)


def test_negated_views(cuda):
    """A view that torch negates on reading (of a conjugate's imaginary part) counts with its sign."""
    from siren_amd import fp8
    x, w, b = torch.randn(40, 130, device=cuda), torch.randn(70, 130, device=cuda), torch.randn(70, device=cuda)
    neg = [torch._neg_view(t) for t in (x, w, b)]
    assert all(t.is_neg() for t in neg)
    for rows in (3, 40):
        assert torch.equal(fp8.linear(neg[0][:rows], neg[1], neg[2]), fp8.linear(-x[:rows], -w, -b))
        leaves = [t.detach().requires_grad_(True) for t in (neg[0][:rows], neg[1], neg[2])]
        plain = [t.clone().requires_grad_(True) for t in (-x[:rows], -w, -b)]
        dy = torch.randn(rows, 70, device=cuda)
        got = torch.autograd.grad(fp8.linear(*leaves, 'sine'), leaves, torch._neg_view(dy))
        want = torch.autograd.grad(fp8.linear(*plain, 'sine'), plain, -dy)
        assert all(torch.equal(g, v) for g, v in zip(got, want))
    assert torch.equal(fp8.dequantize(fp8.quantize(neg[0])), fp8.dequantize(fp8.quantize(-x)))


def test_sine_at_any_phase(cuda):
    """sin(omega z) of phases from none to 1e12, each exact in its own 32 bits, and no row's result by its neighbours'."""
    from siren_amd import fp8
    omega, n = 30., 64
    w = torch.zeros(n, 128, device=cuda)
    w8 = fp8.quantize(w, 'tile')
    edge = 2. ** 22 * 2 * math.pi / omega
    bias = torch.cat([torch.logspace(-6, 10.5, 40, dtype=torch.float64), edge * (1 + torch.linspace(-3e-7, 3e-7, 24).double())])
    bias = bias.float().to(cuda)
    x = torch.zeros(70, 128, device=cuda)
    for m in (1, 20, 70):
        y = fp8.linear(x[:m], w8, bias, 'sine', omega=omega)
        want = np.sin(np64(bias) * omega)
        # v_sin_f32's own error and the turns' last bit (2^-24 of a turn); past 2^22 turns, 2^-53 of the product in 64 bits
        turns = np.abs(np64(bias)) * omega / (2 * math.pi)
        tol = 1e-6 + 2 * math.pi * (turns * 2. ** -52)
        assert (np.abs(np64(y) - want) <= tol).all()
    alone = torch.cat([fp8.linear(x[:1], fp8.quantize(w[i:i + 1], 'tile'), bias[i:i + 1], 'sine', omega=omega) for i in range(n)], 1)
    assert torch.equal(alone, fp8.linear(x[:1], w8, bias, 'sine', omega=omega))


def test_a_layer_whose_backward_would_not_fit_is_refused_at_once(cuda):
    """dx and dW have the layer's inputs as their columns (fewer than 2^22), dW the rows as its sum (2^24 - 128 at most): the
    forward of what a gradient would be refused for is refused, that of a layer without those gradients is not."""
    from siren_amd import fp8
    k = 1 << 22
    x, w = torch.ones(1, k, device=cuda), torch.zeros(1, k, device=cuda)
    w[0, :5] = 1.
    assert fp8.linear(x, w).tolist() == [[5.]]
    for a, b in ((x.clone().requires_grad_(True), w), (x, w.clone().requires_grad_(True))):
        with pytest.raises(ValueError, match='gradient'):
            fp8.linear(a, b)
    b = torch.ones(1, device=cuda, requires_grad=True)
    y = fp8.linear(x, w, b)  # a bias's gradient alone has no such product
    assert torch.autograd.grad(y.sum(), b)[0].tolist() == [1.]
    # one input less: a result of 2^22 - 1 columns, exact in ones
    leaves = [x[:, 1:].clone().requires_grad_(True), w[:, 1:].clone().requires_grad_(True)]
    dx, dw = torch.autograd.grad(fp8.linear(*leaves).sum(), leaves)
    assert torch.equal(dx, leaves[1].detach()) and torch.equal(dw, leaves[0].detach())
    rows, w = (1 << 24) - 128, torch.ones(1, 1, device=cuda, requires_grad=True)
    x = torch.ones(rows + 1, 1, device=cuda)
    with pytest.raises(ValueError, match='gradient of the weight'):
        fp8.linear(x, w)
    assert bool((fp8.linear(x, w.detach()) == 1).all())
    y = fp8.linear(x[:rows], w)
    assert torch.autograd.grad(y, w, torch.ones_like(y))[0].tolist() == [[float(rows)]]  # whole numbers below 2^24


@pytest.mark.parametrize('m', [3, 40, 300])
@pytest.mark.parametrize('fmt', [E4M3, E5M2])
def test_products_at_the_small_end(cuda, m, fmt):
    """Blocks of magnitudes from 2^-139 to 2^-90 against others near 2^100: a bf16 operand holds values under 2^-126 to half of
    2^-133, all others exactly; the sums are 32-bit ones of that. The scale bytes from which on nothing is lost are 3 and, for
    e5m2, 10."""
    from siren_amd import fp8
    g = torch.Generator().manual_seed(m)
    k, n, first = 384, 70, 3 if fmt is E4M3 else 10
    a = torch.randn(m, k, generator=g) * torch.exp2(torch.randint(-137, -90, (m, 3), generator=g).float()).repeat_interleave(128, 1)
    b = torch.randn(n, k, generator=g) * 2. ** 100
    aq, byte = held(np64(a), fmt)
    bq = held(np64(b), tiles=True)[0]
    assert byte.min() == 1 and byte.max() > first
    small = (np.abs(aq) < 2. ** -126) & np.repeat(byte < first, 128, 1)
    want = aq @ bq.T
    tol = product_tol(aq, bq, want, torch.float32) + (1 + 2. ** -10) * 2. ** -134 * (small @ np.abs(bq).T)
    qa, qb = fp8.quantize(a.to(cuda), dtype=fmt), fp8.quantize(b.to(cuda), 'tile')
    check(fp8.matmul(qa, qb), want, tol, 'small first operand')
    lossless = torch.from_numpy((byte >= first).all(1))
    check(fp8.matmul(qa, qb)[lossless.to(cuda)], want[lossless.numpy()], product_tol(aq, bq, want, torch.float32)[lossless.numpy()],
          'bytes from %d on' % first)
    if fmt is E4M3:
        check(fp8.linear(a.to(cuda), qb), want, tol, 'layer')
        check(fp8.matmul(qb, qa), want.T, tol.T, 'small second operand')


@pytest.mark.parametrize('m', [3, 40])
def test_products_at_the_large_end(cuda, m):
    """A block whose largest value rounds to 2^128 holds an infinity there, as dequantize shows it, and spoils its own row; the
    largest that does not, 2^128 (1 - 2^-4), is taken exactly."""
    from siren_amd import fp8
    a = torch.zeros(m, 200)
    a[:, 0] = 2. ** 127 + 2. ** 126 + 2. ** 125 + 2. ** 124  # 2^128 (1 - 2^-4), an e4m3 number times a power of two
    a[:, 1], a[1, 0] = 2. ** 121, torch.finfo(torch.float32).max
    b = torch.zeros(5, 200)
    b[:, :2], b[3, 0] = 2. ** -100, 0.
    qa, qb = fp8.quantize(a.to(cuda)), fp8.quantize(b.to(cuda))
    assert bool(torch.isinf(fp8.dequantize(qa)[1, 0]))
    want = (fp8.dequantize(qa).double().cpu() @ fp8.dequantize(qb).double().cpu().t()).float()
    assert torch.isinf(want[1, :3]).all() and torch.isnan(want[1, 3]) and torch.isfinite(want[0]).all()
    for got in (fp8.matmul(qa, qb), fp8.linear(a.to(cuda), fp8.quantize(b.to(cuda), 'tile'))):
        assert torch.equal(got.cpu().nan_to_num(1., 2.), want.nan_to_num(1., 2.))


@pytest.mark.parametrize('m', [7, 200, 1500])
def test_sine_bias_gradient_is_the_formulas(cuda, m):
    """db of a sine layer against dy omega cos(omega z) in 64 bits: its terms are products of dy and a bf16 cosine, off by half a
    bf16 step (2^-8) and by the phase's error, nothing of them is in 8 bits, and their sum is a 32-bit one."""
    from siren_amd import fp8
    k, n = 192, 130
    x, w, b = layer(m, k, n, torch.float32, cuda, 5)
    dy = values((m, n), 6, 1 / 64).to(cuda)
    b.requires_grad_(True)
    db, = torch.autograd.grad(fp8.linear(x, w, b, 'sine'), b, dy)
    xq, wq = held(np64(x))[0], held(np64(w), tiles=True)[0]
    z = xq @ wq.T + np64(b)
    d = 30 * np.cos(30 * z)
    phase = 30 * product_tol(xq, wq, 0 * z, torch.float32, np.abs(np64(b))) + np.abs(30 * z) * 2. ** -23 + 2. ** -22
    off = 30 * phase + 2. ** -8 * np.abs(d)
    want, mag = (np64(dy) * d).sum(0), (np.abs(np64(dy)) * (np.abs(d) + off)).sum(0)
    check(db, want, (np.abs(np64(dy)) * off).sum(0) + 24 * 2. ** -24 * mag + 2. ** -149, 'db')
