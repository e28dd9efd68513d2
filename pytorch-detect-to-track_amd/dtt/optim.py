"""Optimizer operators over all tensors of a model at once (csrc/optim.hip): clipping by the global gradient norm, the AdamW
step with 32-bit moments and the AdamW step with moments in 8 bits, and the optimizer class that keeps their state.

    norm = clip_grad_norm_(model.parameters(), 10.0)                 # any optimizer
    opt = GroupedAdamW(groups, lr=1e-4, max_norm=10.0)               # clipping inside the step: the gradients are not rewritten
    opt = GroupedAdamW(groups, lr=1e-4, state_bits=8)                # 2.02 bytes of moments per element instead of 8

The reference trains with torch.optim's SGD or Adam, one parameter group per parameter (trainval_net.py:280-294).

Nothing here waits for the GPU: norms, step counters and the decision to skip a step stay in device memory, so a call can be
captured into a graph and counts on with every replay.  A captured call keeps the addresses of the tensors it was given and a
learning rate given as a number; a schedule under a graph passes the rate as a float32 tensor and writes to it.
"""
import ctypes
import math

import torch

from . import _lib
from ._lib import check, ptr, stream_ptr

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
BLOCK = 256                      # elements, in memory order, that share a base of the 8-bit moments
_NAN_FLAG = 0x4000


# ------------------------------------------------------------------------------------------------ argument checks
def _dense(t):
    """Whether t fills one run of memory, in whatever order of its dimensions."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, sz) for sz, st in zip(t.shape, t.stride()) if sz != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _same_order(a, b):
    """Whether a and b (same shape, a dense) hold the same element at the same place of their memory."""
    return (a.is_contiguous() and b.is_contiguous()) or all(sz == 1 or x == y for sz, x, y in zip(a.shape, a.stride(), b.stride()))


def _device_of(what, tensors):
    """The one device of all tensors, as an index."""
    dev = None
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s: expected tensors (got %s)" % (what, type(t).__name__))
        d = t.get_device()
        if d < 0:
            raise RuntimeError("dtt ops run on the GPU only (%s got a %s tensor); there is no CPU fallback" % (what, t.device))
        if dev is None:
            dev = d
        elif d != dev:
            raise ValueError("%s: all tensors must be on one device (got cuda:%d and cuda:%d)" % (what, dev, d))
    return dev


def _check_gradients(what, grads):
    grads = list(grads)
    for g in grads:
        if isinstance(g, torch.Tensor) and (g.layout != torch.strided or g.dtype not in _DTYPES):
            raise TypeError("%s: gradients must be dense float32, bfloat16 or float16 tensors (got %s, %s)" % (what, g.dtype, g.layout))
    return grads, _device_of(what, grads)


def _limit(what, max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("%s: max_norm must not be negative (got %r)" % (what, max_norm))
    return max_norm


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _longs(values):
    return (ctypes.c_long * len(values))(*values)


def _written(tensors):
    """The kernels write behind autograd's back: tell it, as torch's own in-place operations do."""
    torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


# ------------------------------------------------------------------------------------------------ gradient norm
def _norm_and_factor(grads, max_norm, dev):
    """(2,) float32: the norm of all gradients and the factor min(1, max_norm / (norm + 1e-6))."""
    n = len(grads)
    out = torch.empty(2, dtype=torch.float32, device=grads[0].device)
    numel = _longs([g.numel() for g in grads])
    L = _lib.lib()
    with torch.cuda.device(dev):
        nbytes = L.dtt_grad_norm_workspace_bytes(n, numel)
        ws = torch.empty(nbytes // 8, dtype=torch.float64, device=out.device)
        check(L.dtt_grad_norm(n, _pointers(grads), numel, (ctypes.c_int * n)(*[_DTYPES[g.dtype] for g in grads]), max_norm, ptr(out), ptr(ws),
                              nbytes, stream_ptr(dev)), "grad_norm")
    return out


def _any_order(what, grads):
    for i, g in enumerate(grads):
        if not _dense(g):
            raise ValueError("%s: gradient %d is not dense (shape %s, strides %s)" % (what, i, tuple(g.shape), g.stride()))


@torch.no_grad()
def grad_norm(grads):
    """The 2-norm of all gradients as if they were one vector: a float32 scalar on their device.  Sums in 64 bits."""
    grads, dev = _check_gradients("grad_norm", grads)
    if not grads:
        return torch.zeros(())
    _any_order("grad_norm", grads)
    return _norm_and_factor(grads, math.inf, dev)[0]


@torch.no_grad()
def clip_grads_(grads, max_norm):
    """Scale all gradients in place by min(1, max_norm / (norm + 1e-6)) and return their norm before that (float32 scalar on their
    device).  Gradients within the limit are not written.  Mixed float32 / bfloat16 / float16 tensors are one vector."""
    max_norm = _limit("clip_grads_", max_norm)
    grads, dev = _check_gradients("clip_grads_", grads)
    if not grads:
        return torch.zeros(())
    _any_order("clip_grads_", grads)
    out = _norm_and_factor(grads, max_norm, dev)
    n = len(grads)
    with torch.cuda.device(dev):
        check(_lib.lib().dtt_grad_scale(n, _pointers(grads), _longs([g.numel() for g in grads]),
                                        (ctypes.c_int * n)(*[_DTYPES[g.dtype] for g in grads]), ptr(out[1:]), stream_ptr(dev)), "grad_scale")
    _written(grads)
    return out[0]


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm):
    """torch.nn.utils.clip_grad_norm_ (2-norm) in three launches: clip_grads_ over the gradients of `parameters` (a tensor or an
    iterable; those without a gradient are left out, a gradient that is an expanded view is made dense first)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = []
    for p in parameters:
        g = p.grad
        if g is None:
            continue
        if g.layout == torch.strided and not _dense(g):
            g = p.grad = g.contiguous()
        grads.append(g)
    return clip_grads_(grads, max_norm)


# ------------------------------------------------------------------------------------------------ AdamW
def _per_tensor(what, name, value, n):
    if isinstance(value, (list, tuple)):
        if len(value) != n:
            raise ValueError("%s: %d values of %s for %d tensors" % (what, len(value), name, n))
        return list(value)
    return [value] * n


class _Step:
    """The arguments of one step, checked; `launch` sends the tensors of each element type."""

    def __init__(self, what, params, grads, moments, steps, lr, betas, eps, weight_decay, max_norm, skip_nonfinite, clip):
        self.what = what
        params, grads, steps = list(params), list(grads), list(steps)
        moments = [list(x) for x in moments]
        n = len(params)
        if any(len(x) != n for x in [grads, steps] + moments):
            raise ValueError("%s: the lists differ in length (%s)" % (what, ", ".join(str(len(x)) for x in [params, grads, steps] + moments)))
        self.beta1, self.beta2 = (float(b) for b in betas)
        self.eps = float(eps)
        if not (0.0 <= self.beta1 < 1.0 and 0.0 <= self.beta2 < 1.0):
            raise ValueError("%s: betas must lie in [0, 1) (got %r)" % (what, betas))
        if not self.eps >= 0.0:
            raise ValueError("%s: eps must not be negative (got %r)" % (what, eps))
        self.max_norm = None if max_norm is None else _limit(what, max_norm)
        self.skip_nonfinite = bool(skip_nonfinite)
        if clip is not None and (max_norm is not None or clip.dtype != torch.float32 or tuple(clip.shape) != (2,) or not clip.is_contiguous()):
            raise ValueError("%s: clip is norm and factor, two float32, and stands in place of max_norm" % what)
        self.lr, self.lr_device = [], []
        for x in _per_tensor(what, "lr", lr, n):
            if isinstance(x, torch.Tensor):
                if x.numel() != 1 or x.dtype != torch.float32:
                    raise TypeError("%s: a learning rate in device memory is one float32 (got %s, %s)" % (what, tuple(x.shape), x.dtype))
                self.lr.append(0.0)
                self.lr_device.append(x)
            else:
                if not x >= 0.0:
                    raise ValueError("%s: lr must not be negative (got %r)" % (what, x))
                self.lr.append(float(x))
                self.lr_device.append(None)
        self.decay = [float(x) for x in _per_tensor(what, "weight_decay", weight_decay, n)]
        if not all(x >= 0.0 for x in self.decay):
            raise ValueError("%s: weight_decay must not be negative" % what)
        for p, g, s in zip(params, grads, steps):
            if not all(isinstance(t, torch.Tensor) for t in (p, g, s)):
                raise TypeError("%s: expected tensors" % what)
            if p.dtype not in _DTYPES or p.layout != torch.strided:
                raise TypeError("%s: parameters must be dense float32, bfloat16 or float16 tensors (got %s, %s)" % (what, p.dtype, p.layout))
            if g.dtype != p.dtype or g.layout != torch.strided:
                raise TypeError("%s: a gradient has its parameter's type (got %s, %s for %s)" % (what, g.dtype, g.layout, p.dtype))
            if g.shape != p.shape:
                raise ValueError("%s: a gradient has its parameter's shape (got %s for %s)" % (what, tuple(g.shape), tuple(p.shape)))
            if not _dense(p):
                raise ValueError("%s: parameters must be dense (got shape %s, strides %s)" % (what, tuple(p.shape), p.stride()))
            if s.dtype != torch.float32 or s.numel() != 1:
                raise TypeError("%s: a step counter is one float32 (got %s, %s)" % (what, tuple(s.shape), s.dtype))
        self.dev = _device_of(what, params + grads + steps + [x for x in self.lr_device + [clip] if x is not None] + [t for x in moments for t in x])
        # a gradient in another order of its dimensions (or an expanded one) is brought into the parameter's
        grads = [g if _same_order(p, g) else torch.empty_like(p).copy_(g) for p, g in zip(params, grads)]
        self.params, self.grads, self.moments, self.steps, self.clip = params, grads, moments, steps, clip
        if self.clip is None and params and (self.max_norm is not None or self.skip_nonfinite):
            self.clip = _norm_and_factor(grads, math.inf if self.max_norm is None else self.max_norm, self.dev)

    def check_moments(self, dtype, lists):
        for x in lists:
            for p, t in zip(self.params, x):
                if t.dtype != dtype:
                    raise TypeError("%s: moments must be %s (got %s)" % (self.what, dtype, t.dtype))
                if t.shape != p.shape or not _same_order(p, t):
                    raise ValueError("%s: moments have their parameter's shape and memory order (got %s, strides %s for %s, strides %s)" %
                                     (self.what, tuple(t.shape), t.stride(), tuple(p.shape), p.stride()))

    def launch(self, call):
        """call(index list, common arguments) once per element type among the parameters."""
        by_type = {}
        for i, p in enumerate(self.params):
            by_type.setdefault(p.dtype, []).append(i)
        L = _lib.lib()
        with torch.cuda.device(self.dev):
            for dtype, at in by_type.items():
                n = len(at)
                pick = (lambda x: x) if n == len(self.params) else (lambda x: [x[i] for i in at])
                nbytes = L.dtt_adamw_workspace_bytes(n)
                ws = torch.empty(nbytes, dtype=torch.uint8, device=self.params[at[0]].device)
                rates = pick(self.lr_device)
                rates = None if all(x is None for x in rates) else (ctypes.c_void_p * n)(*[None if x is None else x.data_ptr() for x in rates])
                call(L, n, at, pick, _DTYPES[dtype], _longs([p.numel() for p in pick(self.params)]), _pointers(pick(self.steps)),
                     (ctypes.c_double * n)(*pick(self.lr)), rates, (ctypes.c_double * n)(*pick(self.decay)),
                     (ptr(self.clip), int(self.skip_nonfinite), ptr(ws), nbytes, stream_ptr(self.dev)))
        _written(self.params)
        return None if self.clip is None else self.clip[0]


@torch.no_grad()
def adamw_(params, grads, exp_avgs, exp_avg_sqs, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None,
           skip_nonfinite=False, clip=None):
    """One AdamW step of all tensors, in place.  Per tensor t <- t + 1 in its step counter (one float32), then
        g <- c g,  m <- beta1 m + (1 - beta1) g,  v <- beta2 v + (1 - beta2) g^2,
        p <- p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps).
    params / grads: float32, bfloat16 or float16 (each gradient in its parameter's type); exp_avgs / exp_avg_sqs: float32, in the
    parameters' memory order.  A parameter is rounded to its type once, to nearest: a bfloat16 parameter does not see steps below
    2^-9 of its value.  lr and weight_decay: numbers, or a list with one for each tensor; lr also float32 tensors (read on the device).
    max_norm: c = min(1, max_norm / (norm + 1e-6)) of the norm over all gradients (which stay as they are), else c = 1.
    skip_nonfinite: where that norm is infinite or NaN, nothing changes, the counters neither.  clip: norm and factor computed before
    (float32, 2 entries), in place of max_norm.  Returns the norm (float32 scalar on the device), or None without any of the three."""
    s = _Step("adamw_", params, grads, (exp_avgs, exp_avg_sqs), steps, lr, betas, eps, weight_decay, max_norm, skip_nonfinite, clip)
    if not s.params:
        return None
    s.check_moments(torch.float32, s.moments)

    def call(L, n, at, pick, dtype, numel, counters, rates, rates_device, decay, tail):
        check(L.dtt_adamw_step(n, dtype, _pointers(pick(s.params)), _pointers(pick(s.grads)), _pointers(pick(s.moments[0])),
                               _pointers(pick(s.moments[1])), numel, counters, rates, rates_device, decay, s.beta1, s.beta2, s.eps, *tail),
              "adamw_")
    norm = s.launch(call)
    _written([t for x in s.moments for t in x] + s.steps)
    return norm


def blocks_of(numel):
    """Blocks (pairs of bases) of the 8-bit moments of a tensor."""
    return (numel + BLOCK - 1) // BLOCK


@torch.no_grad()
def adamw8_(params, grads, exp_avgs, exp_avg_sqs, bases, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None,
            skip_nonfinite=False, clip=None, seed=0, ids=None):
    """adamw_ with the moments in 8 bits: exp_avgs / exp_avg_sqs are uint8 codes in the parameters' shape and memory order, bases int16
    (blocks_of(numel), 2); all zero = moments of zero.  A value has three bits of mantissa; codes span 15.7 (m) and 31.7 (v) powers of
    two below the largest of their block of 256, what lies lower is 0 (m) or the smallest step (v): an element whose gradients stay
    2^-15.7 below its block's largest is not moved.  The rounding of a moment is dithered, right on average, by a hash of seed, ids
    (default: the position in the list), step counter and element; the same inputs give the same codes.  Infinite and NaN moments stay
    in their element, as NaN."""
    s = _Step("adamw8_", params, grads, (exp_avgs, exp_avg_sqs, bases), steps, lr, betas, eps, weight_decay, max_norm, skip_nonfinite, clip)
    ids = list(range(len(s.params))) if ids is None else [int(i) for i in ids]
    if len(ids) != len(s.params):
        raise ValueError("adamw8_: %d ids for %d tensors" % (len(ids), len(s.params)))
    if not s.params:
        return None
    s.check_moments(torch.uint8, s.moments[:2])
    _check_bases("adamw8_", s.params, s.moments[2])

    def call(L, n, at, pick, dtype, numel, counters, rates, rates_device, decay, tail):
        check(L.dtt_adamw8_step(n, dtype, _pointers(pick(s.params)), _pointers(pick(s.grads)), _pointers(pick(s.moments[0])),
                                _pointers(pick(s.moments[1])), _pointers(pick(s.moments[2])), numel, counters, rates, rates_device, decay,
                                (ctypes.c_uint * n)(*[i & 0xFFFFFFFF for i in pick(ids)]), int(seed) & 0xFFFFFFFF, s.beta1, s.beta2, s.eps,
                                *tail), "adamw8_")
    norm = s.launch(call)
    _written([t for x in s.moments for t in x] + s.steps)
    return norm


def _check_bases(what, like, bases):
    for t, b in zip(like, bases):
        if b.dtype != torch.int16 or tuple(b.shape) != (blocks_of(t.numel()), 2) or not b.is_contiguous():
            raise ValueError("%s: bases are int16, contiguous, two for each %d elements (got %s, %s for %d elements)" %
                             (what, BLOCK, b.dtype, tuple(b.shape), t.numel()))


@torch.no_grad()
def unpack_moments_(exp_avgs, exp_avg_sqs, bases, out_avgs, out_avg_sqs):
    """Write the values that 8-bit moments stand for into out_avgs / out_avg_sqs (all float32 or all bfloat16, which holds them exactly;
    in the codes' shape and memory order)."""
    lists = [list(x) for x in (exp_avgs, exp_avg_sqs, bases, out_avgs, out_avg_sqs)]
    n = len(lists[0])
    if any(len(x) != n for x in lists):
        raise ValueError("unpack_moments_: the lists differ in length (%s)" % ", ".join(str(len(x)) for x in lists))
    if n == 0:
        return
    dev = _device_of("unpack_moments_", [t for x in lists for t in x])
    dtype = lists[3][0].dtype
    if dtype not in (torch.float32, torch.bfloat16) or any(t.dtype != dtype for t in lists[3] + lists[4]):
        raise TypeError("unpack_moments_: the values come as float32 or as bfloat16")
    for a, b, x, y in zip(lists[0], lists[1], lists[3], lists[4]):
        if a.dtype != torch.uint8 or b.dtype != torch.uint8:
            raise TypeError("unpack_moments_: codes are uint8 (got %s, %s)" % (a.dtype, b.dtype))
        if not _dense(a) or not all(t.shape == a.shape and _same_order(a, t) for t in (b, x, y)):
            raise ValueError("unpack_moments_: codes and values have one shape and memory order")
    _check_bases("unpack_moments_", lists[0], lists[2])
    with torch.cuda.device(dev):
        check(_lib.lib().dtt_adamw8_unpack(n, _pointers(lists[0]), _pointers(lists[1]), _pointers(lists[2]), _longs([t.numel() for t in lists[0]]),
                                           _DTYPES[dtype], _pointers(lists[3]), _pointers(lists[4]), stream_ptr(dev)), "unpack_moments_")
    _written(lists[3] + lists[4])


@torch.no_grad()
def pack_moments(exp_avg, exp_avg_sq):
    """8-bit moments of float32 ones: (codes, codes, bases), rounded to the nearest level.  For state that comes from elsewhere (a
    checkpoint with 32-bit moments); torch operations, on any device.  Values that 8-bit moments stand for come back unchanged."""
    out, bases = [], []
    for x, top, signed in ((exp_avg, 126, True), (exp_avg_sq, 254, False)):
        if x.dtype != torch.float32 or not _dense(x):
            raise ValueError("pack_moments: dense float32 moments (got %s, strides %s)" % (x.dtype, x.stride()))
        flat = torch.as_strided(x, (x.numel(),), (1,))
        bits = flat.abs().view(torch.int32)
        level = (bits + (1 << 19)) >> 20
        level = torch.where(bits >= 0x7F800000, 0x7F8, level)       # (a NaN's bits may carry into the sign)
        odd = level >= 0x7F8
        pad = blocks_of(x.numel()) * BLOCK - x.numel()
        finite = torch.nn.functional.pad(torch.where(odd, 0, level), (0, pad)).view(-1, BLOCK)
        base = (finite.amax(1) - top).clamp_(min=0) if finite.numel() else finite.new_zeros(0)
        code = (level - base.repeat_interleave(BLOCK)[:x.numel()]).clamp_(min=0)
        if not signed:
            code = torch.maximum(code, (flat > 0).int())
        code = torch.where(odd, top + 1, code)
        if signed:
            code = code | ((flat < 0).int() << 7)
        out.append(torch.empty_like(x, dtype=torch.uint8))
        torch.as_strided(out[-1], (x.numel(),), (1,)).copy_(code)
        bases.append(base)
        if len(bases) == 1:
            odd_any = torch.nn.functional.pad(odd, (0, pad)).view(-1, BLOCK).any(1)
        else:
            odd_any |= torch.nn.functional.pad(odd, (0, pad)).view(-1, BLOCK).any(1)
    flag = odd_any.int() * _NAN_FLAG
    return out[0], out[1], torch.stack([b | flag for b in bases], 1).to(torch.int16)


class GroupedAdamW(torch.optim.Optimizer):
    """AdamW with torch.optim.AdamW's update, parameter groups and -- with 32-bit moments -- state layout: checkpoints go either way
    (`step`, `exp_avg`, `exp_avg_sq`).  All parameters of an element type and (betas, eps) go in the same launches, whatever their
    groups' learning rates and weight decays: the reference's one-group-per-parameter layout costs nothing (trainval_net.py:280-294).

    state_bits: 32, or 8 for uint8 moments (`exp_avg_code`, `exp_avg_sq_code`, `block_base`; see adamw8_); a checkpoint of either
    kind loads into the other.  max_norm: limit on the norm of all gradients, applied inside the step; the norm of the last step is
    `grad_norm` (float32 scalar on the device).  skip_nonfinite: a step whose gradients hold infinities or NaN changes nothing.
    seed: of the rounding of 8-bit moments.  The moments of bfloat16 / float16 parameters are float32 too.

    Before a step is captured into a graph it has to run once (the state is made at its first run), and the gradients have to keep
    their addresses.  amsgrad, maximize and the like are not offered."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_norm=None, skip_nonfinite=False,
                 seed=0):
        if state_bits not in (8, 32):
            raise ValueError("GroupedAdamW: state_bits is 8 or 32 (got %r)" % (state_bits,))
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError("GroupedAdamW: lr must not be negative (got %r)" % (lr,))
        if not all(0.0 <= b < 1.0 for b in betas) or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("GroupedAdamW: betas in [0, 1), eps and weight_decay not negative (got %r, %r, %r)" % (betas, eps, weight_decay))
        self.state_bits, self.skip_nonfinite, self.seed = state_bits, bool(skip_nonfinite), int(seed)
        self.max_norm = None if max_norm is None else _limit("GroupedAdamW", max_norm)
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        return dict(super().__getstate__(), state_bits=self.state_bits, skip_nonfinite=self.skip_nonfinite, seed=self.seed,
                    max_norm=self.max_norm, grad_norm=None)

    # ------------------------------------------------------------------ state
    def _make_state(self, fresh):
        """Zero moments for parameters that take their first step."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("GroupedAdamW: run a step before capturing one (its state would be made anew by every replay)")
        by_device = {}
        for p in fresh:
            if not _dense(p):
                raise ValueError("GroupedAdamW: parameters must be dense (got shape %s, strides %s)" % (tuple(p.shape), p.stride()))
            by_device.setdefault(p.device, []).append(p)
        for dev, ps in by_device.items():
            counters = torch.zeros(len(ps), dtype=torch.float32, device=dev).unbind()
            for p, t in zip(ps, counters):
                st = self.state[p]
                st["step"] = t
                if self.state_bits == 32:
                    st["exp_avg"], st["exp_avg_sq"] = (torch.zeros_like(p, dtype=torch.float32) for _ in range(2))
                else:
                    st["exp_avg_code"], st["exp_avg_sq_code"] = (torch.zeros_like(p, dtype=torch.uint8) for _ in range(2))
                    st["block_base"] = torch.zeros(blocks_of(p.numel()), 2, dtype=torch.int16, device=dev)

    def _moments(self, p, st):
        """float32 moments of a parameter, in the memory order that its state has."""
        if "exp_avg" in st:
            return st["exp_avg"], st["exp_avg_sq"]
        out = [torch.empty_like(st["exp_avg_code"], dtype=torch.float32) for _ in range(2)]
        unpack_moments_([st["exp_avg_code"]], [st["exp_avg_sq_code"]], [st["block_base"]], out[:1], out[1:])
        return out

    @torch.no_grad()
    def moments(self, p):
        """(exp_avg, exp_avg_sq) of a parameter as float32, whatever its state holds them in; None before its first step."""
        st = self.state.get(p)
        return tuple(t.clone() for t in self._moments(p, st)) if st else None

    def _keep_moments(self, p, st, m, v):
        """The state entries for float32 moments, in the parameter's memory order and this optimizer's form."""
        m, v = (torch.empty_like(p, dtype=torch.float32).copy_(x) for x in (m, v))
        for k in ("exp_avg", "exp_avg_sq", "exp_avg_code", "exp_avg_sq_code", "block_base"):
            st.pop(k, None)
        if self.state_bits == 32:
            st["exp_avg"], st["exp_avg_sq"] = m, v
        else:
            st["exp_avg_code"], st["exp_avg_sq_code"], st["block_base"] = pack_moments(m, v)

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Of this class (32 or 8 bits) or of torch.optim.AdamW / Adam.  The moments keep float32 (or their codes) whatever the
        parameters' type is, and are re-packed where the other form was saved."""
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("GroupedAdamW: a checkpoint with amsgrad or maximize does not load")
        saved = dict(state_dict["state"])
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        names = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(names, [p for g in self.param_groups for p in g["params"]]):
            if i not in saved:
                continue
            src = saved[i]
            st = self.state[p]
            t = src["step"]
            st["step"] = torch.as_tensor(t).detach().clone().to(device=p.device, dtype=torch.float32).reshape(())
            for k, dt in (("exp_avg", torch.float32), ("exp_avg_sq", torch.float32), ("exp_avg_code", torch.uint8),
                          ("exp_avg_sq_code", torch.uint8), ("block_base", torch.int16)):
                if k in src:
                    st[k] = src[k].detach().to(device=p.device, dtype=dt, copy=True)
            if ("exp_avg" in st) != (self.state_bits == 32):
                self._keep_moments(p, st, *self._moments(p, st))

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, fresh, grads = {}, [], []
        place = -1
        for g in self.param_groups:
            for p in g["params"]:
                place += 1
                grad = p.grad
                if grad is None:
                    continue
                if grad.layout != torch.strided:
                    raise TypeError("GroupedAdamW: gradients must be dense tensors (got %s)" % grad.layout)
                if p not in self.state or not self.state[p]:
                    fresh.append(p)
                grads.append(grad)
                work.setdefault((tuple(g["betas"]), g["eps"]), []).append((p, grad, g["lr"], g["weight_decay"], place))
        if not grads:
            return loss
        _device_of("GroupedAdamW", grads)
        if fresh:
            self._make_state(fresh)
        clip = None
        if self.max_norm is not None or self.skip_nonfinite:
            dense = [g if _dense(g) else g.contiguous() for g in grads]
            checked, dev = _check_gradients("GroupedAdamW", dense)
            clip = _norm_and_factor(checked, math.inf if self.max_norm is None else self.max_norm, dev)
            self.grad_norm = clip[0]
        for (betas, eps), rows in work.items():
            states = []
            for p, _, _, _, _ in rows:
                st = self.state[p]
                first = st["exp_avg"] if self.state_bits == 32 else st["exp_avg_code"]
                if not _same_order(p, first):   # the parameter took another memory order since (channels-last filters)
                    self._keep_moments(p, st, *self._moments(p, st))
                states.append(st)
            common = dict(lr=[r[2] for r in rows], betas=betas, eps=eps, weight_decay=[r[3] for r in rows], skip_nonfinite=self.skip_nonfinite,
                          clip=clip)
            params, gs, counters = [r[0] for r in rows], [r[1] for r in rows], [st["step"] for st in states]
            if self.state_bits == 32:
                adamw_(params, gs, [st["exp_avg"] for st in states], [st["exp_avg_sq"] for st in states], counters, **common)
            else:
                adamw8_(params, gs, [st["exp_avg_code"] for st in states], [st["exp_avg_sq_code"] for st in states],
                        [st["block_base"] for st in states], counters, seed=self.seed, ids=[r[4] for r in rows], **common)
        return loss
