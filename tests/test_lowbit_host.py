"""Refusals of the 8-bit training entry points that need no GPU: the C ABI validates before any device work, and the Python
entry points refuse CPU tensors and wrong arguments."""
import ctypes

import pytest
import torch


@pytest.fixture(scope='module')
def lib():
    import __graft_entry__
    __graft_entry__.build()
    from siren_amd import _lib
    return _lib.load()


P = ctypes.c_void_p
OK, EINVAL = 0, 1


def test_quantize_validates(lib):
    def call(x=P(64), dtype=0, rows=4, cols=8, ld=8, mult=None, fmt=0, tiles=0, q=P(64), s=P(64), qt=None, st=None,
             ws=None, sums=None):
        return lib.siren_fp8_quantize(x, dtype, rows, cols, ld, mult, fmt, tiles, 0, q, s, qt, st, ws, sums, None)
    assert call(rows=0) == OK and call(cols=0, ld=0) == OK
    for bad in (dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(cols=-1), dict(ld=7), dict(fmt=2), dict(s=None), dict(q=None),
                dict(qt=P(64)), dict(st=P(64)), dict(rows=129, sums=P(64)), dict(x=None), dict(q=None, s=None), dict(q=P(72)),
                dict(x=P(66)), dict(dtype=1, x=P(65)), dict(qt=P(8), st=P(64)),
                dict(rows=1 << 40, cols=1 << 30, ld=1 << 30), dict(rows=1 << 29, cols=128, ld=128), dict(mult=P(72)),
                dict(rows=1 << 31, qt=P(64), st=P(64)), dict(rows=2, cols=1 << 27, ld=1 << 27, sums=P(64))):
        assert call(**bad) == EINVAL, bad
        assert lib.siren_last_error()


def test_quantize_sources_validate(lib):
    def source(**kw):
        f = dict(x=64, dtype=0, format=0, rows=4, cols=8, ld=8, mult=None, tiles=0, panels=0, q=64, s=64, qt=None, st=None,
                 colsum_ws=None, colsum=None)
        f.update(kw)
        return tuple(f[name] for name, _ in Source._fields_)

    class Source(ctypes.Structure):
        _fields_ = [('x', P), ('dtype', ctypes.c_int32), ('format', ctypes.c_int32), ('rows', ctypes.c_int64),
                    ('cols', ctypes.c_int64), ('ld', ctypes.c_int64), ('mult', P), ('tiles', ctypes.c_int32),
                    ('panels', ctypes.c_int32)] + [(n, P) for n in ('q', 's', 'qt', 'st', 'colsum_ws', 'colsum')]

    def call(*sources, count=None):
        held = (Source * len(sources))(*sources)
        return lib.siren_fp8_quantize_sources(ctypes.byref(held), len(sources) if count is None else count, None)
    assert call(source(rows=0)) == OK and call(source(rows=0), source(cols=0)) == OK
    assert lib.siren_fp8_quantize_sources(None, 1, None) == EINVAL
    for count in (0, 3, -1):
        assert call(source(rows=0), source(rows=0), count=count) == EINVAL
    # a wrong second one is refused before the first is begun
    for bad in (dict(dtype=3), dict(s=None), dict(ld=7), dict(q=None, s=None), dict(x=None), dict(panels=4)):
        assert call(source(), source(**bad)) == EINVAL and call(source(**bad), source()) == EINVAL, bad


def test_products_validate(lib):
    def call(a=P(64), sa=P(64), m=4, b=P(64), sb=P(64), n=4, k=8, bias=None, act=0, omega=30., out=P(64), dtype=0, deriv=None,
             ws=None, fmt=0):
        return lib.siren_fp8_matmul(a, sa, m, 0, fmt, b, sb, n, 1, k, bias, act, omega, out, dtype, deriv, ws, None)
    assert call(m=0) == OK and call(n=0) == OK
    for bad in (dict(m=-1), dict(n=-1), dict(k=0), dict(fmt=2), dict(act=2), dict(dtype=9), dict(a=None), dict(sa=None),
                dict(b=None), dict(sb=None), dict(out=None), dict(a=P(8)), dict(b=P(8)), dict(sa=P(2)), dict(sb=P(2)),
                dict(out=P(8)), dict(bias=P(2)), dict(deriv=P(64)), dict(act=1, omega=float('nan')),
                dict(act=1, omega=float('inf')), dict(act=1, deriv=P(4)), dict(k=1 << 20), dict(m=1 << 40, n=1 << 40)):
        assert call(**bad) == EINVAL, bad  # k = 2^20 with 4 x 4 outputs is split: it needs ws
    c = ctypes.c_int64(-7)
    for fn in (lib.siren_fp8_matmul_ws_bytes, lib.siren_fp8_linear_ws_bytes):
        assert fn(4, 4, 0, ctypes.byref(c)) == EINVAL and fn(-1, 4, 4, ctypes.byref(c)) == EINVAL and c.value == -7
        assert fn(4, 4, 4, None) == EINVAL
        assert fn(0, 4, 4, ctypes.byref(c)) == OK and c.value == 0
        c.value = -7
    assert lib.siren_fp8_matmul_ws_bytes(1 << 18, 1024, 1024, ctypes.byref(c)) == OK and c.value == 0
    assert lib.siren_fp8_matmul_ws_bytes(1024, 1024, 1 << 18, ctypes.byref(c)) == OK and c.value % (4 << 20) == 0 and c.value

    def lin(x=P(64), m=40, k=8, ld=8, w=P(64), sw=P(64), n=4, y=P(64), ws=P(64), deriv=None):
        return lib.siren_fp8_linear(x, 0, m, k, ld, w, sw, n, None, 0, 30., y, deriv, ws, None)
    assert lin(m=0) == OK and lin(n=0) == OK
    for bad in (dict(m=-1), dict(k=0), dict(x=None), dict(w=None), dict(sw=None), dict(y=None), dict(ws=None), dict(ws=P(8)),
                dict(w=P(4)), dict(sw=P(1)), dict(ld=3), dict(x=P(66)), dict(y=P(4)), dict(deriv=P(64))):
        assert lin(**bad) == EINVAL, bad


def test_adamw_validates(lib):
    def call(count=1, p=64, g=64, n=5, dtype=0, bits=32, m=P(64), v=P(64), sm=None, sv=None, step=P(64), lr=1e-3, b1=.9, b2=.99,
             eps=1e-8, wd=0., scratch=P(64), arrays=True):
        ps, gs = (P * 1)(p), (P * 1)(g)
        ns, ts = (ctypes.c_int64 * 1)(n), (ctypes.c_int32 * 1)(dtype)
        a = (ps, gs, ns, ts) if arrays else (None,) * 4
        return lib.siren_adamw_step(count, *a, bits, m, v, sm, sv, step, lr, b1, b2, eps, wd, 0., 0, scratch, None)
    for bad in (dict(count=-1), dict(bits=16), dict(b1=1.), dict(b2=-.1), dict(eps=-1.), dict(eps=float('nan')),
                dict(lr=float('inf')), dict(wd=float('nan')), dict(step=None), dict(step=P(4)), dict(scratch=None),
                dict(arrays=False), dict(dtype=3), dict(n=-1), dict(p=None), dict(p=66), dict(g=66), dict(m=None), dict(v=None),
                dict(m=P(8)), dict(bits=8), dict(bits=8, sm=P(64)), dict(n=1 << 45)):
        assert call(**bad) == EINVAL, bad
    c = ctypes.c_int64(-7)
    assert lib.siren_adamw_scratch_bytes(-1, ctypes.byref(c)) == EINVAL and c.value == -7
    assert lib.siren_adamw_scratch_bytes(1000, None) == EINVAL
    assert lib.siren_adamw_scratch_bytes(1000, ctypes.byref(c)) == OK and c.value > 64


def test_python_entry_points_refuse_the_cpu():
    from siren_amd import fp8, optim
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match='ROCm'):
        fp8.linear(x, w)
    with pytest.raises(RuntimeError, match='ROCm'):
        fp8.quantize(x)
    with pytest.raises(TypeError):
        fp8.linear([1.], w)
    with pytest.raises(RuntimeError, match='ROCm'):
        optim.adamw_step([x], [x], x, x, x)
    with pytest.raises(RuntimeError, match='ROCm'):
        optim.FusedAdamW([x])
    with pytest.raises(ValueError):
        optim.FusedAdamW([])
    with pytest.raises(ValueError):
        optim.adamw_step([], [], x, x, x)


def test_dequantize_is_the_layout():
    """Blocks by hand: two rows of 200 columns, scales per row and per tile."""
    from siren_amd import fp8
    data = torch.zeros(2, 256)
    data[0, :200], data[1, :200] = 1., -2.
    data = data.to(torch.float8_e4m3fn)
    row = torch.tensor([[127, 128, 127, 127], [126, 129, 127, 127]], dtype=torch.uint8)
    got = fp8.dequantize(fp8.Blocks(data, row, 200))
    want = torch.cat([torch.tensor([[1.], [-1.]]).expand(2, 128), torch.tensor([[2.], [-8.]]).expand(2, 72)], 1)
    assert torch.equal(got, want)
    tile = fp8.dequantize(fp8.Blocks(data, row[:1], 200))
    assert torch.equal(tile, torch.cat([torch.tensor([[1.], [-2.]]).expand(2, 128), torch.tensor([[2.], [-4.]]).expand(2, 72)], 1))


def test_modules_take_the_precision():
    from siren_amd.meta_modules import HyperNetwork
    from siren_amd.modules import FCBlock, SingleBVPNet
    torch.manual_seed(0)
    a = SingleBVPNet(verbose=False)
    torch.manual_seed(0)
    b = SingleBVPNet(precision='fp8', verbose=False)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    assert list(a.state_dict()) == list(b.state_dict())
    with pytest.raises(RuntimeError, match='ROCm'):
        b({'coords': torch.zeros(1, 4, 2)})
    hyper = HyperNetwork(64, 1, 64, a, precision='fp8')
    with pytest.raises(RuntimeError, match='ROCm'):
        hyper(torch.zeros(2, 64))
    assert [l[0].precision for l in FCBlock(2, 1, 1, 64, nonlinearity='relu', precision='fp8').net] == ['fp32', 'fp8', 'fp32']
    assert [l[0].precision for l in FCBlock(2, 1, 1, 64, nonlinearity='relu').net] == ['fp32'] * 3
    with pytest.raises(ValueError):
        SingleBVPNet(precision='fp4', verbose=False)


def test_longest_sums(lib):
    """The longest sum is 2^24 - 128: a tile's 256 rows of k bytes, rounded up to 128, are addressed by 32-bit offsets. A
    result has fewer than 2^22 columns. The refusal names the bound that it enforces."""
    c = ctypes.c_int64(0)
    for fn in (lib.siren_fp8_matmul_ws_bytes, lib.siren_fp8_linear_ws_bytes):
        assert fn(4, 4, (1 << 24) - 128, ctypes.byref(c)) == OK and fn(4, (1 << 22) - 1, 8, ctypes.byref(c)) == OK
        for bad in ((4, 4, (1 << 24) - 127), (4, 4, (1 << 24) - 1), (4, 1 << 22, 8)):
            assert fn(*bad, ctypes.byref(c)) == EINVAL, bad
            assert b'2^24 - 128' in lib.siren_last_error() and b'2^22' in lib.siren_last_error()


@pytest.mark.parametrize('n', [(1 << 63) - 1, (1 << 63) - 60, (1 << 63) - 128, 1 << 62, 1 << 56])
def test_sizes_at_the_end_of_64_bits(lib, n):
    """No size wraps on its way to a check: each is refused."""
    c = ctypes.c_int64(-7)
    for fn in (lib.siren_fp8_matmul_ws_bytes, lib.siren_fp8_linear_ws_bytes):
        for size in ((n, 4, 4), (4, n, 4), (4, 4, n), (n, n, n)):
            assert fn(*size, ctypes.byref(c)) == EINVAL and c.value == -7, size
    for rows, cols in ((n, 4), (4, n), (n, n)):
        assert lib.siren_fp8_quantize(P(64), 0, rows, cols, cols, None, 0, 0, 0, P(64), P(64), None, None, None, None, None) == EINVAL
        assert lib.siren_fp8_quantize(P(64), 0, rows, cols, cols, None, 0, 0, 0, P(64), P(64), P(64), P(64), P(64), P(64),
                                      None) == EINVAL
    many = 300  # their blocks' sum does not wrap either
    ps, ns, ts = (P * many)(*[64] * many), (ctypes.c_int64 * many)(*[n] * many), (ctypes.c_int32 * many)()
    assert lib.siren_adamw_step(many, ps, ps, ns, ts, 32, P(64), P(64), None, None, P(64), 1e-3, .9, .99, 1e-8, 0., 0., 0, P(64),
                                None) == EINVAL


def test_adamw_with_counts_validates(lib):
    def call(counts, step=P(64), count=1, scratch=P(64)):
        return lib.siren_adamw_step_each(count, (P * 1)(64), (P * 1)(64), (ctypes.c_int64 * 1)(5), (ctypes.c_int32 * 1)(0), 32, P(64),
                                         P(64), None, None, step, counts, 1e-3, .9, .99, 1e-8, 0., 0., 0, scratch, None)
    for bad in (dict(counts=P(4)), dict(counts=P(65)), dict(counts=P(64), step=None), dict(counts=P(64), scratch=None),
                dict(counts=P(64), count=-1), dict(counts=None, count=1 << 33)):
        assert call(**bad) == EINVAL, bad
    a, b = ctypes.c_int64(0), ctypes.c_int64(0)
    assert lib.siren_adamw_scratch_bytes(1000, ctypes.byref(a)) == OK and lib.siren_adamw_scratch_bytes(2000, ctypes.byref(b)) == OK
    assert b.value - a.value >= 8 * 1000 and a.value % 16 == 0  # room for each tensor's own corrections


def test_zero_grad_of_a_bucket():
    """Gradients that are views of one buffer are cleared in place and stay its views."""
    from types import SimpleNamespace
    from siren_amd import optim
    bucket = torch.ones(10)
    p, q, r = torch.zeros(4, requires_grad=True), torch.zeros(6, requires_grad=True), torch.zeros(2, requires_grad=True)
    p.grad, q.grad = bucket[:4], bucket[4:].view_as(q)
    optim.FusedAdamW.zero_grad(SimpleNamespace(params=[p, q, r]), set_to_none=False)
    assert not bucket.any() and p.grad.data_ptr() == bucket.data_ptr() and r.grad is None
    x = torch.ones(4, requires_grad=True)  # one that is a graph's result is cut off from it
    p.grad = x * 2
    optim.FusedAdamW.zero_grad(SimpleNamespace(params=[p]), set_to_none=False)
    assert p.grad.grad_fn is None and not p.grad.any()
    optim.FusedAdamW.zero_grad(SimpleNamespace(params=[p, q]))
    assert p.grad is None and q.grad is None


@pytest.mark.parametrize('bits', [32, 8])
def test_a_state_is_taken_whole_or_not(bits):
    """load_state_dict of a state that lacks a tensor, or holds one of another size or type, changes nothing."""
    from siren_amd import optim

    def build(fill, n=256, count=2):
        opt = object.__new__(optim.FusedAdamW)
        opt.state_bits, opt.seed, dtype = bits, fill, torch.float32 if bits == 32 else torch.float8_e4m3fn
        opt.exp_avg, opt.exp_avg_sq = (torch.full((n,), float(fill)).to(dtype) for _ in range(2))
        opt.scales = None if bits == 32 else tuple(torch.full((n // 128,), fill, dtype=torch.uint8) for _ in range(2))
        opt.steps, opt.counts = torch.full((1,), fill), torch.full((count,), fill)
        return opt

    def bytes_of(opt):
        return [opt.seed] + [t.contiguous().view(torch.uint8).tolist() for t in opt.state_dict().values() if isinstance(t, torch.Tensor)]

    mine, good = build(1), build(2).state_dict()
    before = bytes_of(mine)
    for key in good:
        if key != 'counts':  # that one is made up
            with pytest.raises(KeyError):
                mine.load_state_dict({k: v for k, v in good.items() if k != key})
            assert bytes_of(mine) == before, key
        if isinstance(good[key], torch.Tensor):
            for bad in (good[key].float()[:1].expand(3), good[key].to(torch.float64)):
                with pytest.raises(ValueError):
                    mine.load_state_dict({**good, key: bad})
                assert bytes_of(mine) == before, key
    with pytest.raises(ValueError):  # as many values, other tensors
        mine.load_state_dict(build(2, count=3).state_dict())
    assert bytes_of(mine) == before
    mine.load_state_dict(good)
    assert bytes_of(mine) == bytes_of(build(2))


@pytest.mark.parametrize('rows,cols', [(0, 200), (0, 0), (3, 0)])
@pytest.mark.parametrize('tile', [False, True])
def test_dequantize_nothing(rows, cols, tile):
    """What quantize returns for no rows or no columns is no values."""
    from siren_amd import fp8
    b = fp8.Blocks(torch.zeros(rows, (cols + 127) // 128 * 128).to(torch.float8_e4m3fn),
                   torch.zeros((rows + 127) // 128 if tile else rows, (cols + 511) // 512 * 4, dtype=torch.uint8), cols)
    assert fp8.dequantize(b).shape == (rows, cols)
