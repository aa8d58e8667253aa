"""The many-tensor AdamW step (siren_amd.optim.adamw_step, FusedAdamW) against torch.optim.AdamW and against a restatement
of its definition: 32-bit moments in 64 bits, 8-bit moments code for code. Needs an MI355X."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [198401, 1, 127, 128, 129, 0, 4099, 2048, 2049, 65536]


def make(sizes, dtype, seed=0, scale=1.):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        out.append((torch.randn(n, generator=g) * scale * 10. ** float(torch.randn(1, generator=g).clamp(-2, 2))).to(dtype))
    return out


def flat(ts):
    return np.concatenate([np.pad(t.detach().float().cpu().numpy().reshape(-1), (0, -t.numel() % 128)) for t in ts])


# ---- the definition ----------------------------------------------------------------------------------------------------
def mix(z):
    with np.errstate(over='ignore'):
        z = z + np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    return z ^ (z >> np.uint64(31))


def hold(x, bits16):
    """(codes, bytes) of a flat fp32 state: per block of 128 the smallest 2^e >= 2^-126 with max |x| <= 448 2^e; a magnitude
    lies between two e4m3 values and takes the upper one if its 16 random bits, added at 2^-16 of their distance,
    carry. Magnitudes are cut to 20 bits below the code first, as a number of fp32's precision is."""
    b = x.reshape(-1, 128)
    bad = ~np.isfinite(b).all(1)
    safe = np.where(bad[:, None], np.float32(0), b)
    f, e = np.frexp(np.abs(safe).max(1).astype(np.float64) / 448)
    e = np.where(f > 0, np.maximum(np.where(f > 0.5, e, e - 1), -126), -126)
    y = np.abs(safe).astype(np.float64) * np.ldexp(1., -e)[:, None]
    ey = np.where(y > 0, np.maximum(np.frexp(y)[1] - 1, -6), -6)  # exponent of y's e4m3 binade
    part = y / np.ldexp(1., ey - 3)                 # in units of the binade's spacing
    part = np.rint(part * 2 ** 20)                  # fp32 holds 20 bits below the code; subnormal codes round there
    up = np.floor((part + bits16.reshape(-1, 128).astype(np.float64) * 16) / 2 ** 20)
    code = np.where(ey == -6, up, up + 8 * (ey + 6)).astype(np.int64)
    return np.where(bad[:, None], 0, code).reshape(-1), np.where(bad, 255, e + 127)


def value(code, byte):
    mant, ex = code & 7, (code >> 3) & 15
    v = np.where(ex == 0, np.ldexp(mant / 8., -6), np.ldexp(1 + mant / 8., ex - 7)) * np.where(code & 128, -1., 1.)
    s = np.where(byte == 255, np.nan, np.ldexp(1., np.asarray(byte, np.int64) - 127))
    return (v.reshape(-1, 128) * s[:, None]).reshape(-1).astype(np.float32)


def oracle8(g, m, u, t, seed, c, b1, b2):
    """One step of the 8-bit moments in fp32, each operation rounded by itself: (m, u) before rounding, codes, bytes."""
    f = np.float32
    g = g * f(c)
    m = m + (g - m) * f(1 - b1)
    v = (u * u) * f(b2) + (g * g) * f(1 - b2)
    u = np.sqrt(v)
    i = np.arange(m.size // 2, dtype=np.uint64)
    with np.errstate(over='ignore'):
        h = mix(mix(np.uint64(seed) ^ mix(np.uint64(t))) + i)
    rm = np.stack([h & np.uint64(0xFFFF), (h >> np.uint64(32)) & np.uint64(0xFFFF)], 1).reshape(-1)
    ru = np.stack([(h >> np.uint64(16)) & np.uint64(0xFFFF), h >> np.uint64(48)], 1).reshape(-1)
    cm, bm = hold(m, rm)
    cu, bu = hold(u, ru)
    cu = np.where((u > 0) & (np.repeat(bu, 128) != 255), np.maximum(cu, 1), cu)
    cm = np.where((m < 0) & (np.repeat(bm, 128) != 255), cm | 128, cm)
    return m, u, cm, bm, cu, bu


def update(p, m, u, t, lr, b1, b2, eps, wd):
    p, m, u = (a.astype(np.float64) for a in (p, m, u))
    step = lr / (1 - b1 ** t) * m / (u / math.sqrt(1 - b2 ** t) + eps)
    return p * (1 - lr * wd) - step, step


HALF = {torch.float32: 2. ** -24, torch.bfloat16: 2. ** -8, torch.float16: 2. ** -11}


def check_params(got, want, step, dtype, what=''):
    """The update's factors are rounded about ten times at 2^-23 or better (two of them by 1-ulp reciprocal and root),
    p (1 - lr wd) twice at half a step, the sum once, then once to dtype."""
    tol = 3 * 2. ** -24 * np.abs(want) + 12 * 2. ** -23 * np.abs(step) + HALF[dtype] * np.abs(want) + 2. ** -25 * (dtype != torch.float32) + 1e-37
    bad = np.abs(got - want) > tol
    assert not bad.any(), '%s: %d off, worst %.3g' % (what, bad.sum(), (np.abs(got - want) / tol).max())


# ---- 32 bits -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('max_norm', [None, 1., 1e9])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_states_in_32_bits(cuda, max_norm, dtype):
    from siren_amd.optim import FusedAdamW
    params = [t.to(cuda).requires_grad_(True) for t in make(SIZES, dtype, 1, 0.05)]
    opt = FusedAdamW(params, lr=1e-3, weight_decay=0.1, max_norm=max_norm)
    m = v = np.zeros(opt.exp_avg.numel())
    for t in range(1, 5):
        grads = make(SIZES, dtype, 10 + t, 0.1)
        for p, g in zip(params, grads):
            p.grad = g.to(cuda)
        before = flat(params)
        opt.step()
        g = flat(grads).astype(np.float64)
        norm = math.sqrt((g ** 2).sum())
        c = 1. if max_norm is None else min(1., max_norm / (norm + 1e-6))
        if max_norm is not None:
            assert abs(float(opt.grad_norm()) - norm) <= 2. ** -23 * norm
        g = g * np.float64(np.float32(c))
        # from the kernel's own previous state: a step's error, not the run's
        m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g ** 2
        gm, gv = (s.cpu().numpy().astype(np.float64) for s in (opt.exp_avg, opt.exp_avg_sq))
        # each of the four or five operations rounds at half a step of a magnitude that these sums bound; 1 - b2 as an
        # fp32 number is 2^-24 off itself, and so on
        assert (np.abs(gm - m) <= 6 * 2. ** -24 * (np.abs(m) + np.abs(g)) * t + 1e-44).all()
        assert (np.abs(gv - v) <= 6 * 2. ** -24 * v * t + 1e-44).all()
        want, step = update(before, gm, np.sqrt(gv), t, 1e-3, 0.9, 0.999, 1e-8, 0.1)
        check_params(flat(params), want, step, dtype, t)
        assert int(opt.steps) == t
        m, v = gm, gv


def test_against_torch(cuda):
    """torch.optim.AdamW after clip_grad_norm_, on a network's tensors, 20 steps."""
    from siren_amd.optim import FusedAdamW
    shapes = [(256, 2), (256,), (256, 256), (256,), (1, 256), (1,)]
    g = torch.Generator().manual_seed(0)
    start = [torch.randn(*s, generator=g) * 0.1 for s in shapes]
    a, b = ([t.clone().to(cuda).requires_grad_(True) for t in start] for _ in range(2))
    mine = FusedAdamW(a, lr=1e-3, weight_decay=0.05, max_norm=1.)
    theirs = torch.optim.AdamW(b, lr=1e-3, weight_decay=0.05)
    for k in range(20):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape, generator=g).to(cuda)
            q.grad = p.grad.clone()
        torch.nn.utils.clip_grad_norm_(b, 1.)
        mine.step(), theirs.step()
    for p, q in zip(a, b):  # 20 steps of at most lr each, every one within some 20 roundings
        assert (p - q).abs().max() <= 20 * (1e-3 * 20 * 2. ** -23 + 4 * 2. ** -24)


# ---- 8 bits ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('max_norm', [None, 1.])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_states_in_8_bits(cuda, max_norm, dtype):
    from siren_amd.optim import FusedAdamW
    params = [t.to(cuda).requires_grad_(True) for t in make(SIZES, dtype, 1, 0.05)]
    opt = FusedAdamW(params, lr=1e-3, weight_decay=0.1, max_norm=max_norm, state_bits=8, seed=77)
    m = u = np.zeros(opt.exp_avg.numel(), np.float32)
    for t in range(1, 6):
        grads = make(SIZES, dtype, 10 + t, 0.1)
        for p, g in zip(params, grads):
            p.grad = g.to(cuda)
        before = flat(params)
        opt.step()
        g = flat(grads)
        c = 1. if max_norm is None else min(1., max_norm / (math.sqrt((g.astype(np.float64) ** 2).sum()) + 1e-6))
        mn, un, cm, bm, cu, bu = oracle8(g, m, u, t, 77, c, 0.9, 0.999)
        assert np.array_equal(opt.scales[0].cpu().numpy(), bm) and np.array_equal(opt.scales[1].cpu().numpy(), bu)
        assert np.array_equal(opt.exp_avg.view(torch.uint8).cpu().numpy(), cm)
        assert np.array_equal(opt.exp_avg_sq.view(torch.uint8).cpu().numpy(), cu)
        want, step = update(before, mn, un, t, 1e-3, 0.9, 0.999, 1e-8, 0.1)
        check_params(flat(params), want, step, dtype, t)
        m, u = value(cm, bm), value(cu, bu)


def test_moments_in_8_bits_follow_those_in_32(cuda):
    """Rounding at random is right on average: under a constant gradient (its sign alternating over the elements) m's mean
    follows 1 - b1^t, and the mean of sqrt(v) 1 - b2^t's root, where nearest rounding would leave them behind."""
    from siren_amd.optim import FusedAdamW
    n, steps = 1 << 16, 300
    p = torch.zeros(n, device=cuda, requires_grad=True)
    opt = FusedAdamW([p], lr=0., weight_decay=0., state_bits=8, seed=3)
    sign = torch.where(torch.arange(n, device=cuda) % 2 == 0, 1., -1.)
    p.grad = sign * 0.7
    for _ in range(steps):
        opt.step()
    s = [torch.exp2(b.float() - 127).repeat_interleave(128) for b in opt.scales]
    m, u = opt.exp_avg.float() * s[0] * sign, opt.exp_avg_sq.float() * s[1]
    # a code's spacing is at most 1/8 of its value, a rounding's deviation at most half of that; m forgets within some
    # 1 / (1 - b1^2) steps: an element's deviation is below 0.0625 * sqrt(1 / 0.19) = 0.15, the mean's below 0.15 / 256,
    # five of which are 0.3 %
    assert abs(float(m.mean()) / (0.7 * (1 - 0.9 ** steps)) - 1) < 0.003
    # v = u^2 is unbiased up to u's own variance, which adds at most (1/16)^2 = 0.4 % of v a step where v grows by
    # 0.1 % at least of itself: v's mean is over what 32 bits give, by a factor that the balance of decay 0.001 and
    # variance bounds: at most exp(300 * (1/16)^2 / 3) with u uniform between codes
    want = 0.49 * (1 - 0.999 ** steps)
    ratio = float((u * u).mean()) / want
    assert 0.97 < ratio < math.exp(steps / 256 / 3), ratio


def test_not_finite_gradients(cuda):
    """A NaN or infinite gradient spoils its tensor's element (32 bits) or its block of 128 (8 bits), and stays visible."""
    from siren_amd.optim import FusedAdamW
    for bits in (32, 8):
        p = torch.ones(1000, device=cuda, requires_grad=True)
        opt = FusedAdamW([p], lr=1e-2, state_bits=bits)
        p.grad = torch.full_like(p, 0.1)
        p.grad[130], p.grad[700] = float('nan'), float('inf')
        opt.step()
        p.grad = torch.full_like(p, 0.1)
        opt.step()
        lost = torch.isnan(p)
        block = torch.arange(1000, device=cuda) // 128
        want = torch.zeros(1000, dtype=torch.bool, device=cuda)
        want[130] = want[700] = True
        if bits == 8:
            want = (block == 130 // 128) | (block == 700 // 128)
            assert opt.scales[0].tolist()[1] == 255 and opt.scales[0].tolist()[5] == 255
        assert torch.equal(lost, want)
        opt = FusedAdamW([p.detach().clone().nan_to_num_(1.).requires_grad_(True)], max_norm=1., state_bits=bits)
        opt.params[0].grad = torch.full((1000,), float('nan'), device=cuda)
        opt.step()  # a NaN norm is no factor of 1
        assert torch.isnan(opt.grad_norm()) and torch.isnan(opt.params[0]).all()


@pytest.mark.parametrize('bits', [32, 8])
def test_many_tensors_views_and_missing_gradients(cuda, bits):
    """More tensors than one launch takes, of mixed types, at odd addresses, some without a gradient: the same as each
    tensor's own step (without clipping tensors do not see each other), nothing around them written."""
    from siren_amd.optim import FusedAdamW
    rng = np.random.default_rng(0)
    sizes = [int(s) for s in rng.integers(1, 700, 300)]
    types = [[torch.float32, torch.bfloat16, torch.float16][i % 3] for i in range(300)]

    def build():
        stores, params = [], []
        g = torch.Generator().manual_seed(5)
        for i, (n, dt) in enumerate(zip(sizes, types)):
            store = torch.full((n + 8,), 9., dtype=dt, device=cuda)
            at = i % 5
            p = store[at:at + n]
            p.copy_(torch.randn(n, generator=g))
            grad = torch.randn(n + 8, generator=g).to(dt).to(cuda)[i % 3:i % 3 + n]
            p.requires_grad_(True)
            p.grad = None if i % 7 == 3 else grad
            stores.append((store, at, n)), params.append(p)
        return stores, params

    s1, p1 = build()
    s2, p2 = build()
    opt = FusedAdamW(p1, lr=1e-2, state_bits=bits, seed=9)
    opt.step(), opt.step()
    for i, p in enumerate(p2):
        if bits == 8:
            break  # the random bits go by the element's place in the list: compared below
        own = FusedAdamW([p], lr=1e-2, state_bits=bits, seed=9)
        own.step(), own.step()
        assert torch.equal(p, p1[i]), i
    for (store, at, n), p in zip(s1, p1):
        assert (store[:at] == 9).all() and (store[at + n:] == 9).all()
    off = 0
    for i, (n, q) in enumerate(zip(sizes, p2)):
        span = slice(off, off + (n + 127) // 128 * 128)
        if i % 7 == 3:
            assert torch.equal(p1[i], q.detach()) if bits == 8 else True
            assert not opt.exp_avg[span].float().any() and not opt.exp_avg_sq[span].float().any()
        else:
            assert opt.exp_avg[span].float().any()
        off = span.stop
    if bits == 8:  # one step of all against the definition
        s3, p3 = build()
        opt = FusedAdamW(p3, lr=1e-2, state_bits=8, seed=9)
        opt.step()
        g = flat([torch.zeros_like(p) if p.grad is None else p.grad for p in p3])
        zero = np.zeros(g.size, np.float32)
        _, _, cm, bm, cu, bu = oracle8(g, zero, zero, 1, 9, 1., 0.9, 0.999)
        assert np.array_equal(opt.exp_avg.view(torch.uint8).cpu().numpy(), cm)
        assert np.array_equal(opt.exp_avg_sq.view(torch.uint8).cpu().numpy(), cu)
        assert np.array_equal(opt.scales[1].cpu().numpy(), bu)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('max_norm', [None, 0.5])
def test_captured_step_advances(cuda, bits, max_norm):
    """A captured step counts its replays: three replays are three eager steps; two optimisers' graphs do not meet."""
    from siren_amd.optim import FusedAdamW

    def build(seed):
        ps = [t.to(cuda).requires_grad_(True) for t in make([3000, 17, 128], torch.float32, seed)]
        for p, g in zip(ps, make([3000, 17, 128], torch.float32, seed + 50)):
            p.grad = g.to(cuda)
        return FusedAdamW(ps, lr=1e-2, state_bits=bits, seed=seed, max_norm=max_norm)

    eager, captured, graphs = [build(1), build(2)], [build(1), build(2)], []
    for o in captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o.step()
        graphs.append(g)
    assert int(captured[0].steps) == 0  # recording does not run
    for k in range(3):
        for o in eager:
            o.step()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, captured):
            assert int(b.steps) == k + 1
            assert all(torch.equal(p, q) for p, q in zip(a.params, b.params))
            assert torch.equal(a.exp_avg.view(torch.uint8), b.exp_avg.view(torch.uint8))
        torch.randn(1000, device=cuda).sum().item()


def test_state_dict_resumes(cuda):
    from siren_amd.optim import FusedAdamW
    for bits in (32, 8):
        runs = []
        for resume in (False, True):
            ps = [t.to(cuda).requires_grad_(True) for t in make([500, 20], torch.float32, 4)]
            opt = FusedAdamW(ps, lr=1e-2, state_bits=bits, seed=6)
            for k in range(6):
                if resume and k == 3:
                    saved = {n: v.clone() if isinstance(v, torch.Tensor) else v for n, v in opt.state_dict().items()}
                    ps = [p.detach().clone().requires_grad_(True) for p in ps]
                    opt = FusedAdamW(ps, lr=1e-2, state_bits=bits)
                    opt.load_state_dict(saved)
                for p, g in zip(ps, make([500, 20], torch.float32, 30 + k)):
                    p.grad = g.to(cuda)
                opt.step()
            runs.append(ps)
        assert all(torch.equal(p, q) for p, q in zip(*runs))


def test_autograd_notices_a_step(cuda):
    """A graph that saved a parameter refuses its backward after a step, as with torch's optimisers; a parameter without a
    gradient was not touched."""
    from siren_amd.optim import FusedAdamW
    p, q = (torch.ones(5, device=cuda, requires_grad=True) for _ in range(2))
    opt = FusedAdamW([p, q], max_norm=1.)
    opt.step()  # nothing has a gradient
    assert float(opt.grad_norm()) == 0. and (p == 1).all() and int(opt.steps) == 1
    p.grad = torch.ones_like(p)
    saved, other = (p * p).sum(), (q * q).sum()
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        saved.backward()
    other.backward()
    assert torch.equal(q.grad, 2 * torch.ones_like(q))


def test_refusals(cuda):
    from siren_amd.optim import FusedAdamW, adamw_step
    p = torch.ones(300, device=cuda)
    opt = FusedAdamW([p.requires_grad_(True)])
    p = p.detach()
    m, v, t = opt.exp_avg, opt.exp_avg_sq, opt.steps
    ok = dict(params=[p], grads=[p.clone()], exp_avg=m, exp_avg_sq=v, step=t)
    adamw_step(**ok)
    for change in (dict(params=[]), dict(grads=[]), dict(grads=[p.half()]), dict(grads=[p[:5]]), dict(exp_avg=m[:128]),
                   dict(exp_avg=m.half()), dict(step=t.int()), dict(max_norm=0.), dict(betas=(1., 0.9)), dict(eps=-1.),
                   dict(lr=float('nan')), dict(params=[p[::2]], grads=[p[::2].clone()]),
                   dict(params=[p, p], grads=[p.clone(), p.clone()], exp_avg=torch.zeros(768, device=cuda),
                        exp_avg_sq=torch.zeros(768, device=cuda)),
                   dict(scales=(torch.ones(3, dtype=torch.uint8, device=cuda),) * 2)):
        with pytest.raises(ValueError):
            adamw_step(**{**ok, **change})
    with pytest.raises(RuntimeError):
        adamw_step(**{**ok, 'params': [p.cpu()], 'grads': [p.cpu()]})
    with pytest.raises(RuntimeError):
        adamw_step(**{**ok, 'params': [p.double()], 'grads': [p.double()]})
    with pytest.raises(ValueError):
        FusedAdamW([p], state_bits=16)
    with pytest.raises(ValueError):
        opt.load_state_dict(FusedAdamW([p], state_bits=8).state_dict())


@pytest.mark.parametrize('eps', [0., 1e-25, 1e-8])
def test_subnormal_second_moments(cuda, eps):
    """Gradients of 1e-19 to 1e-20: v is a subnormal number, its root is not, and the step is lr all the same."""
    from siren_amd.optim import FusedAdamW
    p = torch.ones(700, device=cuda).requires_grad_(True)
    opt = FusedAdamW([p], lr=1e-2, eps=eps, weight_decay=0.)
    p.grad = torch.logspace(-19, -20, 700).to(cuda)
    opt.step()
    m, v = opt.exp_avg[:700].cpu().numpy(), opt.exp_avg_sq[:700].cpu().numpy()
    assert (v > 0).all() and (v < 2. ** -126).all()
    want, step = update(np.ones(700), m, np.sqrt(v.astype(np.float64)), 1, 1e-2, 0.9, 0.999, eps, 0.)
    check_params(p.detach().cpu().numpy().astype(np.float64), want, step, torch.float32)


def test_inference_parameters_are_refused_unchanged(cuda):
    from siren_amd import optim
    with torch.inference_mode():
        p = torch.ones(300, device=cuda)
        g = torch.ones(300, device=cuda)
    opt = optim.FusedAdamW([torch.ones(300, device=cuda)])
    with pytest.raises(RuntimeError, match='nference'):
        optim.adamw_step([p], [g], opt.exp_avg, opt.exp_avg_sq, opt.steps)
    assert bool((p == 1).all()) and int(opt.steps) == 0


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_tensors_at_any_address(cuda, bits, dtype):
    """Parameters and gradients that begin one to three elements into their storage give the same bytes as aligned ones."""
    from siren_amd import optim
    sizes, out = [700, 4099, 130, 5, 3, 1], []
    values, slopes = make(sizes, dtype, 3, 0.05), make(sizes, dtype, 4, 0.1)
    for shift in range(4):
        def place(ts):
            held = [torch.empty(t.numel() + 8, dtype=dtype, device=cuda).fill_(7.) for t in ts]
            for h, t in zip(held, ts):
                h[shift:shift + t.numel()] = t.to(cuda)
            return held, [h[shift:shift + t.numel()] for h, t in zip(held, ts)]
        (hp, ps), (_, gs) = place(values), place(slopes)
        opt = optim.FusedAdamW(ps, max_norm=0.5, state_bits=bits)
        optim.adamw_step(ps, gs, opt.exp_avg, opt.exp_avg_sq, opt.steps, max_norm=0.5, scales=opt.scales)
        for h, p in zip(hp, ps):
            assert bool((h[:shift] == 7).all()) and bool((h[shift + p.numel():] == 7).all())
        out.append(torch.cat([p.float() for p in ps] + [opt.exp_avg.float(), opt.exp_avg_sq.float()]))
    assert all(torch.equal(o, out[0]) for o in out)


def test_negated_views(cuda):
    from siren_amd import optim
    p, g = torch.randn(300, device=cuda), torch.randn(300, device=cuda)
    a, b = p.clone(), p.clone()
    for q, grad in ((a, torch._neg_view(g)), (b, -g)):
        opt = optim.FusedAdamW([q])
        optim.adamw_step([q], [grad], opt.exp_avg, opt.exp_avg_sq, opt.steps)
    assert torch.equal(a, b) and not torch.equal(a, p)
    with pytest.raises(ValueError, match='negated'):
        optim.adamw_step([torch._neg_view(p)], [g], opt.exp_avg, opt.exp_avg_sq, opt.steps)


def missing(i, t):
    """Whether tensor i has no gradient in step t: one always has, one never, one begins late, others pause."""
    return [False, True, t <= 7, t % 2 == 0, 3 <= t <= 9, t != 5][i % 6]


@pytest.mark.parametrize('max_norm', [None, 1.])
def test_missing_gradients_against_torch(cuda, max_norm):
    """A parameter's bias corrections count its own steps, as torch.optim.AdamW's do: one whose first gradient comes late, ones
    that pause, one that never has any. More tensors than a launch takes."""
    from siren_amd.optim import FusedAdamW
    g = torch.Generator().manual_seed(0)
    sizes = [7, 130, 300, 5000, 33, 2] * 40
    start = [torch.randn(s, generator=g).clamp(-4, 4) * 0.1 for s in sizes]
    a, b = ([t.clone().to(cuda).requires_grad_(True) for t in start] for _ in range(2))
    mine = FusedAdamW(a, lr=1e-3, weight_decay=0.05, max_norm=max_norm)
    theirs = torch.optim.AdamW(b, lr=1e-3, weight_decay=0.05)
    for t in range(1, 21):
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad = None if missing(i, t) else torch.randn(p.shape, generator=g).to(cuda)
            q.grad = None if p.grad is None else p.grad.clone()
        if max_norm is not None:
            torch.nn.utils.clip_grad_norm_(b, max_norm)
        mine.step(), theirs.step()
    assert mine.counts.tolist() == [sum(not missing(i, t) for t in range(1, 21)) for i in range(len(sizes))]
    assert int(mine.steps) == 20
    # 20 steps, each of at most (1 - b1) / sqrt(1 - b2) = 3.2 lr and within some 20 roundings, of parameters below 1
    for p, q in zip(a, b):
        assert (p - q).abs().max() <= 20 * (4e-3 * 20 * 2. ** -23 + 4 * 2. ** -24)


@pytest.mark.parametrize('max_norm', [None, 1.])
@pytest.mark.parametrize('bits', [32, 8])
def test_missing_gradients_keep_what_is_theirs(cuda, bits, max_norm):
    """Mixed types: without a gradient a parameter and its moments stay as they were; with one, moments, codes and step are the
    definition's, the corrections by the parameter's own count. Captured and replayed it is the same."""
    from siren_amd.optim import FusedAdamW
    types = [torch.float32, torch.bfloat16, torch.float32, torch.float16, torch.float32, torch.bfloat16]
    sizes = [300, 5, 4099, 129, 1, 640]

    def build():
        ps = [t.to(d).to(cuda).requires_grad_(True) for t, d in zip(make(sizes, torch.float32, 1, 0.05), types)]
        return FusedAdamW(ps, lr=1e-3, weight_decay=0.1, max_norm=max_norm, state_bits=bits, seed=5)

    opt, replayed = build(), build()
    m = u = np.zeros(opt.exp_avg.numel(), np.float32)
    count = [0] * 6
    for t in range(1, 9):
        grads = [x.to(d) for x, d in zip(make(sizes, torch.float32, 10 + t, 0.1), types)]
        for o in (opt, replayed):
            for i, (p, g) in enumerate(zip(o.params, grads)):
                p.grad = None if missing(i, t) else g.to(cuda)
        before = [p.detach().clone() for p in opt.params]
        old = [s.clone() for s in (opt.exp_avg.view(torch.uint8), opt.exp_avg_sq.view(torch.uint8))]
        opt.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            replayed.step()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(*([*o.params, o.exp_avg.view(torch.uint8), o.exp_avg_sq.view(torch.uint8), o.counts] for o in (opt, replayed))):
            assert torch.equal(x, y), t
        g = flat([x * 0 if missing(i, t) else x for i, x in enumerate(grads)])
        c = 1. if max_norm is None else min(1., max_norm / (math.sqrt((g.astype(np.float64) ** 2).sum()) + 1e-6))
        mn, un, cm, bm, cu, bu = oracle8(g, m, u, t, 5, c, 0.9, 0.999)
        at = 0
        for i, (p, q) in enumerate(zip(opt.params, before)):
            span = slice(at, at + (p.numel() + 127) // 128 * 128)
            at = span.stop
            raw = [s.view(torch.uint8).view(-1, 4 if bits == 32 else 1)[span] for s in (opt.exp_avg, opt.exp_avg_sq)]
            if missing(i, t):
                assert torch.equal(p, q)
                assert all(torch.equal(x, s.view(-1, 4 if bits == 32 else 1)[span]) for x, s in zip(raw, old))
                continue
            count[i] += 1
            if bits == 8:
                codes = [x.flatten().cpu().numpy() for x in raw]
                assert np.array_equal(codes[0], cm[span]) and np.array_equal(codes[1], cu[span]), (t, i)
            mt, ut = (mn[span], un[span]) if bits == 8 else (opt.exp_avg[span].cpu().numpy(), opt.exp_avg_sq[span].sqrt().cpu().numpy())
            want, step = update(flat([q]), mt, ut, count[i], 1e-3, 0.9, 0.999, 1e-8, 0.1)
            check_params(flat([p]), want, step, types[i], (t, i))
        assert opt.counts.tolist() == count
        if bits == 8:
            m, u = (value(s.view(torch.uint8).cpu().numpy().astype(np.int64), b.cpu().numpy())
                    for s, b in zip((opt.exp_avg, opt.exp_avg_sq), opt.scales))


def test_counts_are_checked_saved_and_made_up(cuda):
    from siren_amd.optim import FusedAdamW, adamw_step
    ps = [torch.ones(300, device=cuda), torch.ones(5, device=cuda)]
    opt = FusedAdamW(ps)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    ps[1].grad = None
    opt.step()
    assert opt.counts.tolist() == [2, 1]
    saved = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in opt.state_dict().items()}
    other = FusedAdamW([p.clone() for p in ps])
    other.load_state_dict(saved)
    assert other.counts.tolist() == [2, 1] and int(other.steps) == 2
    del saved['counts']  # one from before they were counted
    other.load_state_dict(saved)
    assert other.counts.tolist() == [2, 2]
    for bad in (opt.counts[:1], opt.counts.int(), opt.counts.cpu(), torch.zeros(2, 2, dtype=torch.int64, device=cuda)[:, 0]):
        with pytest.raises(ValueError, match='counts'):
            adamw_step(ps, [p.clone() for p in ps], opt.exp_avg, opt.exp_avg_sq, opt.steps, counts=bad)
    assert int(opt.steps) == 2


def test_second_moment_in_8_bits_does_not_drift(cuda):
    """The 8-bit sqrt(v) under a constant gradient, within what its rounding's variance allows. While u <= 0.7, u only grows: a
    step from a code q to u' = q + D, D <= 0.001 (w - q^2) / 2 q with w = 0.49, is rounded to q or to the next code d <= q / 8
    above, with a variance of at most D d <= 0.001 (w - q^2) / 16. v's mean gains just that variance a step, so it grows as if
    1 - b2 were 17 / 16 of itself at most (1 / 256 more in the first step, whose d^2 / 4 is the bound), and as fast as in 32 bits
    at least. The variances add up to 0.3 w / 16 at most, so that v's deviation is below 2 0.7 sqrt(0.0092) = 0.134, a mean's of
    2^16 elements below 0.41 % of 0.127; five of those are 2 %."""
    from siren_amd.optim import FusedAdamW
    n, steps, w = 1 << 16, 300, 0.49
    p = torch.zeros(n, device=cuda, requires_grad=True)
    opt = FusedAdamW([p], lr=0., weight_decay=0., state_bits=8, seed=3)
    p.grad = torch.full((n,), 0.7, device=cuda)
    for _ in range(steps):
        opt.step()
    v = (opt.exp_avg_sq.float() * torch.exp2(opt.scales[1].float() - 127).repeat_interleave(128)).double().square()
    assert bool((v <= w).all())  # and so in every step before
    exact = w * (1 - 0.999 ** steps)
    most = w * (1 - (1 - 0.001 * 17 / 16) ** steps) * (1 + 1 / 256)
    assert 0.98 * exact <= float(v.mean()) <= 1.02 * most, (float(v.mean()) / exact, most / exact)


@pytest.mark.parametrize('bits', [32, 8])
def test_parameters_without_a_gradient_stay(cuda, bits):
    """Of many tensors of mixed types those without a gradient keep their starting values, byte for byte, and so do their
    moments; clipping or not."""
    from siren_amd.optim import FusedAdamW
    types = [torch.float32, torch.bfloat16, torch.float16]
    for max_norm in (None, 0.5):
        ps = [t.to(types[i % 3]).to(cuda).requires_grad_(True) for i, t in enumerate(make(list(range(1, 331)), torch.float32, 8, 0.1))]
        for i, p in enumerate(ps):
            p.grad = None if i % 7 == 3 else torch.ones_like(p)
        start = [p.detach().clone() for p in ps]
        opt = FusedAdamW(ps, lr=1e-2, state_bits=bits, max_norm=max_norm)
        opt.step(), opt.step()
        off = 0
        for i, (p, s) in enumerate(zip(ps, start)):
            span = slice(off, off + (p.numel() + 127) // 128 * 128)
            off = span.stop
            assert torch.equal(p, s) == (i % 7 == 3), i
            assert bool(opt.exp_avg[span].float().any()) != (i % 7 == 3) and bool(opt.exp_avg_sq[span].float().any()) != (i % 7 == 3)


def test_states_that_overlap_are_refused(cuda):
    """Two states in the same memory, a state inside a parameter, counts that are the step: each would be written by one thread
    and read by another."""
    from siren_amd.optim import FusedAdamW, adamw_step
    p = [torch.ones(128, device=cuda)]
    g = [torch.ones(128, device=cuda)]
    a, b = FusedAdamW(p), FusedAdamW(p, state_bits=8)
    one = dict(params=p, grads=g, exp_avg=a.exp_avg, exp_avg_sq=a.exp_avg_sq, step=a.steps, counts=a.counts)
    eight = dict(params=p, grads=g, exp_avg=b.exp_avg, exp_avg_sq=b.exp_avg_sq, step=b.steps, scales=b.scales)
    shared = torch.zeros(192, device=cuda)
    for ok, change in ((one, dict(exp_avg_sq=a.exp_avg)), (one, dict(counts=a.steps)), (one, dict(exp_avg=p[0])),
                       (one, dict(exp_avg=shared[:128], exp_avg_sq=shared[64:])), (one, dict(step=a.exp_avg[:2].view(torch.int64))),
                       (eight, dict(scales=(b.scales[0],) * 2)), (eight, dict(exp_avg=b.exp_avg_sq)),
                       (eight, dict(scales=(b.scales[0], b.exp_avg[:1].view(torch.uint8))))):
        with pytest.raises(ValueError, match='overlap'):
            adamw_step(**{**ok, **change})
    assert bool((p[0] == 1).all()) and int(a.steps) == 0 and int(b.steps) == 0
    adamw_step(**one), adamw_step(**eight)


def test_elements_past_2_to_the_31(cuda):
    """A tensor of 2^31 elements and more, and one behind it: their last elements and moments are those of a short list, the
    zeros before them stay zeros."""
    from siren_amd.optim import FusedAdamW
    n, tail = (1 << 31) + 777, 5000
    for bits in (32, 8):
        big = [torch.zeros(n, dtype=torch.bfloat16, device=cuda), torch.zeros(300, dtype=torch.bfloat16, device=cuda)]
        for p in big:
            p.grad = torch.zeros_like(p)
        g = make([tail, 300], torch.bfloat16, 3)
        start = make([tail, 300], torch.bfloat16, 4)
        short = [s.to(cuda) for s in start]
        for p, q, s, x in zip(big, short, start, g):
            p[-s.numel():], p.grad[-s.numel():] = s.to(cuda), x.to(cuda)
            q.grad = x.to(cuda)
        a, b = (FusedAdamW(ps, lr=1e-2, weight_decay=0.1, max_norm=1., state_bits=bits) for ps in (big, short))
        a.step(), b.step()
        assert torch.equal(a.grad_norm(), b.grad_norm())
        assert all(torch.equal(p[-q.numel():], q) for p, q in zip(big, short))
        assert not big[0][:-tail].any()
        if bits == 32:
            for s, t in ((a.exp_avg, b.exp_avg), (a.exp_avg_sq, b.exp_avg_sq)):
                assert torch.equal(s[n - tail:n], t[:tail]) and torch.equal(s[-384:], t[-384:]) and not s[:n - tail].any()
        else:
            u = lambda o, k: (o.exp_avg_sq[k].float().view(-1, 128) * torch.exp2(o.scales[1].float()[:, None] - 127)[k.start // 128:k.stop // 128])
            x, y = u(a, slice(a.exp_avg.numel() - 384, a.exp_avg.numel())), u(b, slice(b.exp_avg.numel() - 384, b.exp_avg.numel()))
            assert ((x - y).abs() <= torch.maximum(x, y) / 8 + torch.exp2(b.scales[1][-3:].float() - 127)[:, None] * 2. ** -9).all()  # by other random bits
            assert not a.exp_avg[:n - tail - 128].view(torch.uint8).any()
