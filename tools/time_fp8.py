"""The 8-bit training path as a network uses it, on one MI355X: a layer's training step and forward with and without the sine,
AdamW over 35 million parameters of each type, whole networks against the fp32 and bf16x6 engines, the error of an 8-bit
network's activations and the fit of an image.
usage: python tools/time_fp8.py"""
import math
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from siren_amd import dataio, fp8, optim  # noqa: E402
from siren_amd.modules import SingleBVPNet  # noqa: E402

D = 'cuda'


def time_us(f, warmup=40, n=20):
    """Of passes among others; the first twenty or so of a large product after an idle card are slower by up to a fifth."""
    for _ in range(warmup):
        f()
    out = []
    for _ in range(3):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(n):
            f()
        b.record()
        torch.cuda.synchronize()
        out.append(a.elapsed_time(b) / n * 1e3)
    return sorted(out)[1]


def layers():
    for m, k, n, dt in ((262144, 1024, 1024, torch.float32), (262144, 1024, 1024, torch.bfloat16),
                        (16384, 1024, 1024, torch.bfloat16), (262144, 256, 256, torch.bfloat16)):
        for act in (None, 'sine'):
            x = torch.sin(torch.randn(m, k, device=D)).to(dt).requires_grad_(True)
            w = ((torch.rand(n, k, device=D) * 2 - 1) * math.sqrt(6 / k) / 30).requires_grad_(True)
            b = ((torch.rand(n, device=D) * 2 - 1) / math.sqrt(k)).requires_grad_(True)
            dy = (torch.randn(m, n, device=D) / m).to(dt)

            def forward():
                with torch.no_grad():
                    fp8.linear(x, w, b, act)

            def plain():
                z = F.linear(x.float(), w, b)
                torch.autograd.grad((torch.sin(30 * z) if act else z).to(dt), (x, w, b), dy)

            step = time_us(lambda: torch.autograd.grad(fp8.linear(x, w, b, act), (x, w, b), dy))
            print('layer %d x %d -> %d %s %s: training step %.0f us, forward %.0f; torch fp32 step %.0f'
                  % (m, k, n, str(dt)[6:], act or 'linear', step, time_us(forward), time_us(plain, 10, 5)), flush=True)


def adamw():
    w = 256
    sizes = [s for numel in [w * 2, w] + 2 * [w * w, w] + [w, 1] for s in (w * w, w, w * w, w, numel * w, numel)]
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        for bits in (32, 8):
            for max_norm in (None, 1.):
                ps = [torch.randn(s, device=D).to(dt) for s in sizes]
                opt = optim.FusedAdamW(ps, lr=1e-4, state_bits=bits, max_norm=max_norm)
                for p in ps:
                    p.grad = torch.randn_like(p) * 1e-3
                us = time_us(opt.step)
                size = ps[0].element_size()
                bytes_ = sum(sizes) * (3 * size + (16 if bits == 32 else 4 + 4 / 128) + (size if max_norm else 0))
                print('AdamW %d parameters %s, %d-bit moments%s: %.0f us, %.1f TB/s'
                      % (sum(sizes), str(dt)[6:], bits, ', clipping' if max_norm else '', us, bytes_ / us / 1e6), flush=True)


def networks():
    for hidden, d_in, d_out, precisions in ((1024, 3, 3, ('fp32', 'fp8')), (256, 2, 1, ('fp32', 'bf16x6', 'fp8'))):
        for n in (262144, 16384):
            for precision in precisions:
                torch.manual_seed(0)
                net = SingleBVPNet(in_features=d_in, out_features=d_out, hidden_features=hidden, num_hidden_layers=3,
                                   precision=precision, verbose=False).to(D)
                opt = optim.FusedAdamW(net.parameters(), lr=1e-4)
                x, gt = torch.rand(1, n, d_in, device=D) * 2 - 1, torch.rand(1, n, d_out, device=D)

                def step():
                    opt.zero_grad()
                    (net({'coords': x})['model_out'] - gt).square().mean().backward()
                    opt.step()

                def forward():
                    with torch.no_grad():
                        net({'coords': x})
                print('network 5 x %d, %d coordinates, %s: training step %.0f us, forward %.0f'
                      % (hidden, n, precision, time_us(step, 25, 10), time_us(forward, 25, 10)), flush=True)


def accuracy():
    x = torch.rand(1, 20000, 2, generator=torch.Generator(device=D).manual_seed(0), device=D) * 2 - 1
    for hidden in (256, 1024):
        torch.manual_seed(3)
        net = SingleBVPNet(num_hidden_layers=3, hidden_features=hidden, precision='fp8', verbose=False).to(D)
        got, h, errors = list(net.net.forward_with_activations(x).values()), x, []
        with torch.no_grad():
            for i, layer in enumerate(net.net.net[:-1]):
                h = torch.sin(30 * F.linear(h, layer[0].weight, layer[0].bias))
                errors.append('%.1e' % ((got[2 * i + 2] - h).square().mean().sqrt() / h.square().mean().sqrt()))
        print('5 x %d at its initialisation: rms error of each sine layer\'s output over its rms (the first is fp32): %s'
              % (hidden, ', '.join(errors)), flush=True)
    x = dataio.get_mgrid(256).to(D)[None]
    gt = dataio.synthetic_image(x)
    for hidden in (256, 1024):
        for precision in ('fp32', 'fp8'):
            out = []
            for seed in range(3):
                torch.manual_seed(seed)
                net = SingleBVPNet(precision=precision, hidden_features=hidden, verbose=False).to(D)
                opt = optim.FusedAdamW(net.parameters(), lr=1e-4, weight_decay=0.)
                for t in range(501):
                    loss = (net({'coords': x})['model_out'] - gt).square().mean()
                    if t in (100, 300, 500):
                        out.append(10 * math.log10(4 / loss.item()))
                    opt.zero_grad()
                    loss.backward()
                    opt.step()
            print('fit of a 256 x 256 image, 5 x %d, %s: PSNR after 100, 300, 500 steps, three seeds: %s dB'
                  % (hidden, precision, '; '.join(', '.join('%.1f' % v for v in out[i:i + 3]) for i in range(0, 9, 3))), flush=True)


if __name__ == '__main__':
    layers()
    adamw()
    networks()
    accuracy()
