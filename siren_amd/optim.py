"""FusedAdam: clip_grad_norm_ + torch.optim.Adam.step (training.py:17, 98-104) as two HIP launches over ONE flat
parameter bucket (siren_adam_step, step_kernels.hpp), with the global gradient norm kept on the device.

The parameters are re-seated as views of a flat fp32 buffer (state-dict order), and their .grad as views of a
flat gradient buffer that zero_grad() clears in place, so autograd accumulates straight into the bucket and the
step reads it without a gather. Semantics: torch.optim.Adam (amsgrad off, weight_decay 0, maximize off) after
torch.nn.utils.clip_grad_norm_(params, max_norm) when max_norm is set.

adamw_step / FusedAdamW: clip_grad_norm_ + torch.optim.AdamW.step over a list of tensors where they lie (siren_adamw_step,
tu_adamw.hip), with the moments in 32 bits or in 8 with a scale for each block of 128.
"""
import ctypes
import math

import torch

from . import _lib


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


class FusedAdam:
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, max_norm=None):
        self.params = [p for p in params]
        if not self.params:
            raise ValueError('FusedAdam got an empty parameter list')
        dev = self.params[0].device
        if dev.type != 'cuda' or any(p.device != dev or p.dtype != torch.float32 for p in self.params):
            raise RuntimeError('FusedAdam needs fp32 parameters on one ROCm device')
        self.lib = _lib.load()
        self.lr, self.betas, self.eps, self.max_norm = float(lr), tuple(betas), float(eps), max_norm
        n = sum(p.numel() for p in self.params)
        self.flat = torch.empty(n, device=dev)
        # the gradient bucket + one slot for the coordinate count of a count-weighted all-reduce (allreduce_grad)
        self.bucket = torch.zeros(n + 1, device=dev)
        self.grad = self.bucket[:n]
        self.exp_avg = torch.zeros(n, device=dev)
        self.exp_avg_sq = torch.zeros(n, device=dev)
        cnt = ctypes.c_int64()
        _lib.check(self.lib.siren_adam_scratch_floats(ctypes.byref(cnt)), 'siren_adam_scratch_floats')
        self.scratch = torch.zeros(cnt.value, device=dev)
        off = 0
        with torch.no_grad():
            for p in self.params:
                k = p.numel()
                self.flat[off:off + k].copy_(p.reshape(-1))
                p.data = self.flat[off:off + k].view_as(p)
                off += k
        self._bind_grads()
        self.step_count = 0

    def _bind_grads(self):
        off = 0
        for p in self.params:
            k = p.numel()
            p.grad = self.grad[off:off + k].view_as(p)
            off += k

    def zero_grad(self, set_to_none=False):
        self.grad.zero_()
        self._bind_grads()

    def _gather_grads(self):
        """Copy any .grad that autograd replaced (e.g. after set_to_none) back into the bucket."""
        off = 0
        for p in self.params:
            k = p.numel()
            g = p.grad
            view = self.grad[off:off + k]
            if g is None:
                view.zero_()
            elif g.data_ptr() != view.data_ptr():
                view.copy_(g.reshape(-1))
            off += k
        self._bind_grads()

    @torch.no_grad()
    def allreduce_grad(self, world, count=None):
        """Data parallel: reduce the flat gradient bucket over ranks with ONE all-reduce (RCCL over xGMI), in place.
        count=None averages (equal shards); count = this rank's coordinate count weights the ranks' mean-loss
        gradients by their shares (sum_r n_r g_r / sum_r n_r, distributed.allreduce_gradients), the count riding
        in the bucket's last slot so it stays one collective and no host sync."""
        import torch.distributed as dist
        self._gather_grads()
        if count is None:
            dist.all_reduce(self.grad, op=dist.ReduceOp.SUM)
            self.grad.div_(world)
            return
        self.grad.mul_(float(count))
        self.bucket[-1] = float(count)
        dist.all_reduce(self.bucket, op=dist.ReduceOp.SUM)
        self.grad.div_(self.bucket[-1:].clamp_min(1.))

    @torch.no_grad()
    def step(self):
        self._gather_grads()
        self.step_count += 1
        mx = float(self.max_norm) if self.max_norm else 0.
        st = ctypes.c_void_p(torch.cuda.current_stream(self.flat.device).cuda_stream)
        _lib.check(self.lib.siren_adam_step(_ptr(self.flat), _ptr(self.grad), _ptr(self.exp_avg),
                                            _ptr(self.exp_avg_sq), self.flat.numel(), self.lr, self.betas[0],
                                            self.betas[1], self.eps, self.step_count, mx, _ptr(self.scratch), st),
                   'siren_adam_step')

    def grad_norm(self):
        """The pre-clip global gradient norm of the last clipped step (device tensor; no host sync)."""
        return self.scratch[1024]


_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _state_size(params):
    return sum((p.numel() + 127) // 128 * 128 for p in params)


def adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               max_norm=None, seed=0, scales=None, counts=None):
    """One AdamW step (torch.optim.AdamW: decoupled weight decay, amsgrad and maximize off) over all tensors at once,
    after torch.nn.utils.clip_grad_norm_(max_norm) when max_norm is set. Everything is updated in place; nothing
    synchronises with the host, and a captured step advances by itself on every replay (lr and the rest are captured).

    params, grads: lists of tensors, fp32, bf16 or fp16, each gradient of its parameter's type and shape; a gradient may
    be None (the tensor and its state stay as they are). Parameters are contiguous; they, the gradients and the states do
    not overlap.
    exp_avg, exp_avg_sq: flat states, each tensor's padded to a multiple of 128: fp32, or with scales (two uint8 tensors,
    one byte per 128 elements) torch.float8_e4m3fn: exp_avg holds m, exp_avg_sq holds sqrt(v), value * 2^(byte - 127). The
    8-bit states are rounded up or down at random, from (seed, step, element): the same call gives the same result.
    step: int64, one element, on the device: the steps done so far; 1 is added.
    counts: int64, one element a parameter, on the device: the steps that each has taken; 1 is added where there is a gradient,
    and the bias corrections go by it, as torch's do. Without counts they go by step, for a list whose gradients are all there
    in every step.

    Returns the gradients' norm before clipping (a device tensor), or None without max_norm."""
    if not (0. <= betas[0] < 1. and 0. <= betas[1] < 1. and eps >= 0. and math.isfinite(lr) and math.isfinite(weight_decay)):
        raise ValueError('need 0 <= betas < 1, eps >= 0 and finite lr and weight_decay')
    sm, sv = (None, None) if scales is None else scales
    return _lib.native().adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr, betas[0], betas[1], eps, weight_decay,
                                    max_norm, seed & 0xFFFFFFFFFFFFFFFF, sm, sv, counts)


class FusedAdamW:
    """AdamW over parameters where they lie (any mix of fp32, bf16, fp16; .grad may be replaced freely, and be missing: the
    parameter and its moments then stay, and its bias corrections count its own steps), two launches a step. state_bits 8 keeps the moments in 8 bits (2 bytes a parameter instead of 8), rounded at random from seed. One
    set of hyperparameters (attributes: opt.lr = ... between steps) for all parameters; no torch.optim.Optimizer."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None, state_bits=32,
                 seed=0):
        self.params = [p for p in params]
        if not self.params:
            raise ValueError('FusedAdamW got an empty parameter list')
        dev = self.params[0].device
        if dev.type != 'cuda' or any(p.device != dev or p.dtype not in _DTYPES for p in self.params):
            raise RuntimeError('FusedAdamW needs fp32, bf16 or fp16 parameters on one ROCm device')
        if state_bits not in (8, 32):
            raise ValueError('state_bits must be 8 or 32; got %r' % (state_bits,))
        _lib.load()
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), tuple(betas), float(eps), float(weight_decay)
        self.max_norm, self.state_bits, self.seed = max_norm, state_bits, int(seed)
        n = _state_size(self.params)
        dtype = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        self.exp_avg = torch.zeros(n, device=dev).to(dtype)
        self.exp_avg_sq = torch.zeros(n, device=dev).to(dtype)
        # byte 1 is the scale of a block of zeros
        self.scales = None if state_bits == 32 else tuple(torch.ones(n // 128, dtype=torch.uint8, device=dev)
                                                          for _ in range(2))
        self.steps = torch.zeros(1, dtype=torch.int64, device=dev)  # calls, and each parameter's own
        self.counts = torch.zeros(len(self.params), dtype=torch.int64, device=dev)
        self._norm = None

    def zero_grad(self, set_to_none=True):
        for p in self.params:
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                # as torch's optimisers: a gradient that is a view (of a bucket) cannot be detached in place, and need not be
                if p.grad.grad_fn is not None:
                    p.grad.detach_()
                else:
                    p.grad.requires_grad_(False)
                p.grad.zero_()

    @torch.no_grad()
    def step(self):
        self._norm = adamw_step(self.params, [p.grad for p in self.params], self.exp_avg, self.exp_avg_sq, self.steps,
                                lr=self.lr, betas=self.betas, eps=self.eps, weight_decay=self.weight_decay,
                                max_norm=self.max_norm or None, seed=self.seed, scales=self.scales,
                                counts=self.counts)

    def grad_norm(self):
        """The pre-clip global gradient norm of the last clipped step (device tensor; no host sync)."""
        return self._norm

    def state_dict(self):
        """The state's own tensors (8-bit ones as they are held): clone what must outlive the next step."""
        out = {'state_bits': self.state_bits, 'seed': self.seed, 'steps': self.steps, 'counts': self.counts,
               'exp_avg': self.exp_avg, 'exp_avg_sq': self.exp_avg_sq}
        if self.scales is not None:
            out['exp_avg_scale'], out['exp_avg_sq_scale'] = self.scales
        return out

    def load_state_dict(self, state):
        if state['state_bits'] != self.state_bits or state['exp_avg'].numel() != self.exp_avg.numel():
            raise ValueError('a state of %d bits and %d values does not fit this optimiser\'s %d bits and %d values'
                             % (state['state_bits'], state['exp_avg'].numel(), self.state_bits, self.exp_avg.numel()))
        mine = {k: t for k, t in self.state_dict().items() if isinstance(t, torch.Tensor)}
        # a state of before each parameter's steps were counted: they were the calls
        theirs = {k: state['steps'].expand_as(t) if k == 'counts' and k not in state else state[k] for k, t in mine.items()}
        seed = int(state['seed'])
        for k, t in mine.items():  # all of it fits, or nothing is taken
            if theirs[k].shape != t.shape or theirs[k].dtype != t.dtype:
                raise ValueError('%s of the state is %s %s, this optimiser\'s %s %s'
                                 % (k, tuple(theirs[k].shape), theirs[k].dtype, tuple(t.shape), t.dtype))
        self.seed = seed
        for k, t in mine.items():
            t.copy_(theirs[k])
