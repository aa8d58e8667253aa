"""8-bit training as the framework's modules use it: FCBlock, SingleBVPNet and HyperNetwork with precision='fp8', stepped by
FusedAdamW, alone and through training.train. Needs an MI355X."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def grads_of(model):
    return [p.grad for p in model.parameters()]


@pytest.mark.parametrize('hidden', [64, 130, 256, 1024])
def test_sine_network_is_its_layers(cuda, hidden):
    """SingleBVPNet(precision='fp8') is its layers' operators in a row, value and gradients, at widths that the fp32 kernels
    take and that they do not."""
    from siren_amd import fp8
    from siren_amd.modules import SingleBVPNet
    torch.manual_seed(1)
    model = SingleBVPNet(in_features=3, out_features=3, hidden_features=hidden, num_hidden_layers=2, precision='fp8',
                         verbose=False).to(cuda)
    x = torch.rand(1, 300, 3, device=cuda) * 2 - 1
    gt = torch.rand(1, 300, 3, device=cuda)
    out = model({'coords': x})
    (out['model_out'] - gt).square().mean().backward()
    got = grads_of(model)
    layers = [(l[0].weight.detach().requires_grad_(True), l[0].bias.detach().requires_grad_(True)) for l in model.net.net]
    a = torch.sin(30 * torch.nn.functional.linear(x, *layers[0])).bfloat16()
    for w, b in layers[1:-1]:
        a = fp8.linear(a, w, b, 'sine')
    y = torch.nn.functional.linear(a.float(), *layers[-1])
    assert torch.equal(y, out['model_out'])
    (y - gt).square().mean().backward()
    for g, t in zip(got, [t for pair in layers for t in pair]):
        assert torch.equal(g, t.grad)


def test_sine_network_is_near_fp32(cuda):
    """One hidden layer in 8 bits: the output is off by what rounding its operands can do. An operand is off by 2^-4 of
    itself or 2^-10 of its block's scale (2 amax / 448), the bf16 input by 2^-8, the sine is 1-Lipschitz, its bf16 value
    off by 2^-8, and the last layer sums it."""
    from siren_amd.modules import SingleBVPNet
    nets = []
    for precision in ('fp32', 'fp8'):
        torch.manual_seed(3)
        nets.append(SingleBVPNet(num_hidden_layers=1, precision=precision, verbose=False).to(cuda))
    x = torch.rand(1, 500, 2, device=cuda) * 2 - 1
    with torch.no_grad():
        ref, got = (n({'coords': x})['model_out'] for n in nets)
        w0, b0, w1, b1, w2, b2 = (p.double() for p in nets[0].parameters())
        a = torch.sin(30 * (x.double() @ w0.t() + b0))
        ea = 2. ** -8 * a.abs() + (2. ** -4 * (1 + 2. ** -8) * a.abs() + 2. ** -10 / 224 * 1.01)
        ew = 2. ** -4 * w1.abs() + 2. ** -10 / 224 * w1.abs().max()
        dz = ea @ w1.abs().t() + a.abs() @ ew.t() + ea @ ew.t()
        bound = ((30 * dz).clamp(max=2.) + 2. ** -8) @ w2.abs().t() + 1e-5
    assert ((ref - got).abs() <= bound).all()
    assert (ref - got).abs().max() > 0


def test_gradients_of_gradients_are_refused(cuda):
    from siren_amd import diff_operators
    from siren_amd.modules import SingleBVPNet
    model = SingleBVPNet(precision='fp8', verbose=False).to(cuda)
    out = model({'coords': torch.rand(1, 50, 2, device=cuda)})
    g = diff_operators.gradient(out['model_out'], out['model_in'])
    assert g.shape == (1, 50, 2) and torch.isfinite(g).all()
    with pytest.raises(RuntimeError, match='not differentiable again'):
        g.square().mean().backward()
    from siren_amd._lib import SirenUnsupported
    batched = {k: v[None] for k, v in model.named_parameters()}
    with pytest.raises(SirenUnsupported):
        model({'coords': torch.rand(1, 50, 2, device=cuda)}, params=batched)


def test_relu_block_and_batchlinear(cuda):
    from siren_amd import fp8
    from siren_amd.modules import FCBlock
    torch.manual_seed(0)
    net = FCBlock(96, 200, 1, 128, outermost_linear=True, nonlinearity='relu', precision='fp8').to(cuda)
    assert [l[0].precision for l in net.net] == ['fp8'] * 3
    x = torch.randn(7, 5, 96, device=cuda)
    a = x
    for i, l in enumerate(net.net):
        a = fp8.linear(a, l[0].weight, l[0].bias)
        a = a.relu() if i < 2 else a
    assert torch.equal(net(x), a)
    small = FCBlock(8, 1, 1, 128, outermost_linear=True, nonlinearity='relu', precision='fp8')
    assert [l[0].precision for l in small.net] == ['fp32', 'fp8', 'fp32']


@pytest.mark.parametrize('bits', [32, 8])
def test_hypernetwork_trains(cuda, bits):
    """A hypernetwork with 8-bit products predicts a SIREN's weights, the batched kernels evaluate it, FusedAdamW steps:
    the whole step again from its parts is the same step."""
    from siren_amd import optim
    from siren_amd.meta_modules import HyperNetwork
    from siren_amd.modules import SingleBVPNet

    def build():
        torch.manual_seed(5)
        hypo = SingleBVPNet(out_features=1, in_features=2, hidden_features=256, num_hidden_layers=1, verbose=False).to(cuda)
        return hypo, HyperNetwork(64, 1, 64, hypo, precision='fp8').to(cuda)

    g = torch.Generator(device=cuda).manual_seed(0)
    z, x = torch.randn(4, 64, generator=g, device=cuda), torch.rand(4, 200, 2, generator=g, device=cuda) * 2 - 1
    gt = torch.rand(4, 200, 1, generator=g, device=cuda)

    def loss(hypo, hyper):
        return (hypo({'coords': x}, params=hyper(z))['model_out'] - gt).square().mean()

    hypo, hyper = build()
    opt = optim.FusedAdamW(hyper.parameters(), lr=1e-4, max_norm=1., state_bits=bits, seed=2)
    start = [p.detach().clone() for p in hyper.parameters()]
    for _ in range(3):
        opt.zero_grad()
        loss(hypo, hyper).backward()
        opt.step()
    assert torch.isfinite(opt.grad_norm()) and opt.grad_norm() > 0
    assert all(not torch.equal(p, s) for p, s in zip(hyper.parameters(), start))

    hypo2, hyper2 = build()
    params = list(hyper2.parameters())
    size = sum((p.numel() + 127) // 128 * 128 for p in params)
    states = [torch.zeros(size, device=cuda).to(torch.float32 if bits == 32 else torch.float8_e4m3fn) for _ in range(2)]
    scales = None if bits == 32 else [torch.ones(size // 128, dtype=torch.uint8, device=cuda) for _ in range(2)]
    steps = torch.zeros(1, dtype=torch.int64, device=cuda)
    for _ in range(3):
        grads = torch.autograd.grad(loss(hypo2, hyper2), params)
        optim.adamw_step(params, grads, *states, steps, lr=1e-4, max_norm=1., seed=2, scales=scales)
    assert all(torch.equal(p, q) for p, q in zip(hyper.parameters(), params))
    assert torch.equal(opt.exp_avg.view(torch.uint8), states[0].view(torch.uint8))


@pytest.mark.parametrize('clip', [False, 0.5])
def test_train_loop(cuda, tmp_path, clip):
    """training.train with an 8-bit network and optim.FusedAdamW is the same loop written out; a torch optimiser is clipped
    by the loop."""
    from siren_amd import loss_functions as LF, optim, training
    from siren_amd.dataio import get_mgrid, synthetic_image
    from siren_amd.modules import SingleBVPNet
    x = get_mgrid(32).to(cuda)[None]
    gt = {'img': synthetic_image(x)}

    def build(kind):
        torch.manual_seed(0)
        m = SingleBVPNet(precision='fp8', hidden_features=128, verbose=False).to(cuda)
        if kind == 'torch':
            return m, torch.optim.AdamW(m.parameters(), lr=1e-3)
        return m, optim.FusedAdamW(m.parameters(), lr=1e-3, state_bits=8, seed=1)

    args = dict(train_dataloader=[({'coords': x}, gt)], epochs=4, lr=1., steps_til_summary=100, epochs_til_checkpoint=100,
                loss_fn=lambda out, gt: LF.image_mse(None, out, gt), clip_grad=clip, log=lambda *a: None)
    m, opt = build('own')
    losses = training.train(m, model_dir=str(tmp_path / 'a'), optimizer=opt, **args)
    m2, opt2 = build('own')
    opt2.max_norm = clip or None
    want = []
    for _ in range(4):
        loss = LF.image_mse(None, m2({'coords': x}), gt)['img_loss'].mean()
        opt2.zero_grad()
        loss.backward()
        opt2.step()
        want.append(float(loss.detach()))
    assert losses == want
    assert all(torch.equal(p, q) for p, q in zip(m.parameters(), m2.parameters()))
    m3, opt3 = build('torch')
    training.train(m3, model_dir=str(tmp_path / 'b'), optimizer=opt3, **args)
    if clip:
        norm = torch.stack([p.grad.norm() for p in m3.parameters()]).norm()
        assert float(norm) <= clip * (1 + 1e-5)
    with pytest.raises(ValueError):
        training.train(m3, model_dir=str(tmp_path / 'c'), optimizer=opt3, fused_adam=True, **args)


def test_captured_training_step_of_a_network(cuda):
    """A whole step (forward, backward, AdamW on 8-bit states) captured and replayed is the eager step."""
    from siren_amd import optim
    from siren_amd.modules import SingleBVPNet

    def build():
        torch.manual_seed(7)
        m = SingleBVPNet(precision='fp8', hidden_features=128, num_hidden_layers=1, verbose=False).to(cuda)
        return m, optim.FusedAdamW(m.parameters(), lr=1e-3, max_norm=1., state_bits=8)

    x, gt = torch.rand(1, 300, 2, device=cuda), torch.rand(1, 300, 1, device=cuda)

    def step(m, opt):
        grads = torch.autograd.grad((m({'coords': x})['model_out'] - gt).square().mean(), list(m.parameters()))
        for p, g in zip(m.parameters(), grads):
            p.grad = g
        opt.step()

    eager, captured = build(), build()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # libraries that torch's own layers use set themselves up outside the graph
        warm = build()
        step(*warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*captured)
    for _ in range(3):
        step(*eager)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(eager[0].parameters(), captured[0].parameters()):
            assert torch.equal(p, q)
        torch.randn(1000, device=cuda).sum().item()


@pytest.mark.parametrize('kind', ['sine', 'relu'])
@pytest.mark.parametrize('outer', [True, False])
@pytest.mark.parametrize('rows,out', [(9, 3), (300, 3), (300, 70)])
def test_activations_are_the_networks_own(cuda, kind, outer, rows, out):
    """forward_with_activations shows the network that forward runs: the same last value, the sine of each phase, and (past
    the 32 rows of the few-rows kernel, whose sums run in another order) the same gradients."""
    from siren_amd.modules import FCBlock
    torch.manual_seed(4)
    made = dict(in_features=2, out_features=out, num_hidden_layers=2, hidden_features=128, outermost_linear=outer, nonlinearity=kind)
    net = FCBlock(precision='fp8', **made).to(cuda)
    x = torch.rand(1, rows, 2, device=cuda) * 2 - 1
    acts = net.forward_with_activations(x, retain_grad=True)
    values = list(acts.values())
    assert list(acts) == list(FCBlock(**made).to(cuda).forward_with_activations(x))
    leaf = x.clone().requires_grad_(True)
    y = net(leaf)
    assert torch.equal(values[-1], y)
    if kind == 'sine':
        for z, a in zip(values[1::2], values[2::2]):
            assert ((a - torch.sin(30 * z)).abs() <= 2. ** -8 * a.abs() + 1e-5).all()  # held in bf16
    dy = torch.randn_like(y)
    values[-1].backward(dy)
    got = [values[0].grad] + [p.grad for p in net.parameters()]
    assert all(v.grad is not None and torch.isfinite(v.grad).all() for v in values)
    if rows > 32:
        want = torch.autograd.grad(y, [leaf] + list(net.parameters()), dy)
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_activations_of_an_8_bit_network_refuse_what_it_refuses(cuda):
    from siren_amd._lib import SirenUnsupported
    from siren_amd.modules import FCBlock
    net = FCBlock(2, 3, 1, 64, outermost_linear=True, nonlinearity='sine', precision='fp8').to(cuda)
    with pytest.raises(SirenUnsupported):
        net.forward_with_activations(torch.zeros(1, 4, 2, device=cuda), params={k: v[None] for k, v in net.named_parameters()})
    with pytest.raises(RuntimeError, match='ROCm'):
        net.cpu().forward_with_activations(torch.zeros(1, 4, 2))


def test_relu_block_trains_on_3d_inputs(cuda):
    """Its relu works in place on what the layer returned, a view of its rows where the input has three dimensions: value and
    gradients are those of the layers with a relu that copies."""
    from siren_amd import fp8
    from siren_amd.modules import FCBlock
    torch.manual_seed(0)
    net = FCBlock(96, 70, 2, 128, outermost_linear=False, nonlinearity='relu', precision='fp8').to(cuda)
    x = torch.randn(7, 50, 96, device=cuda)
    dy = torch.randn(7, 50, 70, device=cuda)
    for shape in ((7, 50), (350,)):
        leaf = x.view(*shape, 96).clone().requires_grad_(True)
        got = torch.autograd.grad(net(leaf), [leaf] + list(net.parameters()), dy.view(*shape, 70))
        a = leaf
        for l in net.net:
            a = torch.relu(fp8.linear(a, l[0].weight, l[0].bias))
        want = torch.autograd.grad(a, [leaf] + list(net.parameters()), dy.view(*shape, 70))
        assert all(torch.equal(g, v) for g, v in zip(got, want))


def test_function_transforms_are_refused(cuda):
    """torch.func's wrappers have no memory of their own: an error, not a wrong result."""
    from siren_amd import fp8
    w, x = torch.randn(64, 96, device=cuda), torch.randn(4, 5, 96, device=cuda)
    w8 = fp8.quantize(w, 'tile')
    for call in (lambda: torch.vmap(lambda r: fp8.linear(r, w))(x), lambda: torch.vmap(lambda r: fp8.linear(r, w8))(x),
                 lambda: torch.func.grad(lambda r: fp8.linear(r, w).sum())(x[0]), lambda: torch.vmap(lambda r: fp8.quantize(r).data)(x)):
        with pytest.raises(RuntimeError):
            call()
