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
import contextlib
import math
from array import array

import torch

from . import _lib
from ._lib import check

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_UINT8 = 3
BLOCK = 256                      # elements, in memory order, that share a base of the 8-bit moments
_NAN_FLAG = 0x4000
_ONE = (1).to_bytes(8, "little")
_MOMENTS32 = ("exp_avg", "exp_avg_sq")                               # entries of the optimizer's state
_MOMENTS8 = ("exp_avg_code", "exp_avg_sq_code", "block_base")

_host = None


def _tensorlist():
    """The compiled module that reads lists of tensors (csrc/tensorlist.cpp)."""
    global _host
    if _host is None:
        try:
            from . import _tensorlist as module
        except ImportError as e:
            raise _lib.DttLibraryError("dtt/_tensorlist.so is missing or does not load (%s) -- build it with `make -C %s` (or "
                                       "__graft_entry__.build())" % (e, _lib.CSRC))
        _host = module
    return _host


# ------------------------------------------------------------------------------------------------ lists of tensors
class _List:
    """Addresses, element counts and types (as the arrays that the library takes) of a list of tensors."""
    __slots__ = ("tensors", "ptrs", "counts", "types", "device", "type", "odd")

    def __init__(self, what, tensors):
        self.tensors = tensors
        try:
            self.ptrs, self.counts, self.types, self.device, self.type, self.odd = _tensorlist().describe(tensors)
        except TypeError as e:
            raise TypeError("%s: %s" % (what, e)) from None

    def __len__(self):
        return len(self.tensors)

    def floats(self, what, name):
        """All strided float32, bfloat16 or float16."""
        if not 0 <= self.type <= 2:
            for t in self.tensors:
                if t.layout != torch.strided or t.dtype not in _DTYPES or t.is_neg():
                    raise TypeError("%s: %s must be dense float32, bfloat16 or float16 tensors (got %s, %s)" % (what, name, _kind(t), t.layout))
        return self

    def dense(self, what, name):
        if self.odd >= 0:
            t = self.tensors[self.odd]
            raise ValueError("%s: %s must be dense (entry %d: shape %s, strides %s)" % (what, name, self.odd, tuple(t.shape), t.stride()))
        return self


def _kind(t):
    """A tensor's type, and what keeps its memory from being its values."""
    return "%s%s" % (t.dtype, ", a negated view: resolve_neg() first" if t.is_neg() else "")


def _device_of(what, lists):
    """The one device of all tensors, as an index."""
    dev = lists[0].device
    for x in lists:
        if x.device == -1 or (x.device == -2 and not all(t.is_cuda for t in x.tensors)):
            raise RuntimeError("dtt ops run on the GPU only (%s got a %s tensor); there is no CPU fallback" %
                               (what, next(t.device for t in x.tensors if not t.is_cuda)))
    if dev == -2 or any(x.device != dev for x in lists):
        raise ValueError("%s: all tensors must be on one device (got %s)" % (what, sorted({str(t.device) for x in lists for t in x.tensors})))
    return dev


def _dense(t):
    """Whether t fills one run of memory, in whatever order of its dimensions."""
    return t.is_contiguous() or _tensorlist().describe([t])[5] < 0


def _same_order(a, b):
    """Whether a and b (same shape, a dense) hold the same element at the same place of their memory."""
    return (a.is_contiguous() and b.is_contiguous()) or all(sz == 1 or x == y for sz, x, y in zip(a.shape, a.stride(), b.stride()))


def _limit(what, max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("%s: max_norm must not be negative (got %r)" % (what, max_norm))
    return max_norm


def _written(*lists):
    """The kernels write behind autograd's back: tell it of these tensors, as torch's own in-place operations do."""
    _tensorlist().bump(*lists)


_HERE = contextlib.nullcontext()


def _on(dev):
    """The device of a call's tensors as the current one (a step of a few small tensors takes 13 us: no guard where none is needed)."""
    return _HERE if torch.cuda.current_device() == dev else torch.cuda.device(dev)


def _stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev)


# ------------------------------------------------------------------------------------------------ gradient norm
def _norm_and_factor(grads, max_norm, scale=False):
    """(2,) float32: the norm of all gradients (a _List on one GPU) and the factor min(1, max_norm / (norm + 1e-6)); scale: the
    gradients are multiplied by it."""
    n = len(grads)
    device = grads.tensors[0].device
    out = torch.empty(2, dtype=torch.float32, device=device)
    L = _lib.lib()
    nbytes = L.dtt_grad_norm_workspace_bytes(n, grads.counts)
    ws = torch.empty(nbytes // 8, dtype=torch.float64, device=device)
    with _on(grads.device):
        check((L.dtt_grad_clip if scale else L.dtt_grad_norm)(n, grads.ptrs, grads.counts, grads.types, max_norm, out.data_ptr(), ws.data_ptr(),
                                                              nbytes, _stream(grads.device)), "grad_clip" if scale else "grad_norm")
    return out


def _gradients(what, grads):
    grads = _List(what, list(grads)).floats(what, "gradients")
    if len(grads):
        _device_of(what, [grads])
    return grads.dense(what, "gradients")


def grad_norm(grads):
    """The 2-norm of all gradients as if they were one vector: a float32 scalar on their device.  Sums in 64 bits."""
    grads = _gradients("grad_norm", grads)
    return _norm_and_factor(grads, math.inf)[0] if len(grads) else torch.zeros(())


def clip_grads_(grads, max_norm):
    """Scale all gradients in place by min(1, max_norm / (norm + 1e-6)) and return their norm before that (float32 scalar on their
    device).  Gradients within the limit are not written.  Mixed float32 / bfloat16 / float16 tensors are one vector.  An infinite norm
    gives the factor 0 and NaN gives NaN, as the formula has it; an infinite limit asks for the norm alone and leaves the gradients as they
    are, whatever it is.  No tensor may appear twice."""
    max_norm = _limit("clip_grads_", max_norm)
    grads = _gradients("clip_grads_", grads)
    if not len(grads):
        return torch.zeros(())
    out = _norm_and_factor(grads, max_norm, scale=True)
    _written(grads.tensors)
    return out[0]


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm):
    """torch.nn.utils.clip_grad_norm_ (2-norm) in a few launches: clip_grads_ over the gradients of `parameters` (a tensor or an
    iterable; those without a gradient are left out, a gradient that is an expanded or negated view is made dense first)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = []
    for p in parameters:
        g = p.grad
        if g is None:
            continue
        if g.layout == torch.strided and (g.is_neg() or not _dense(g)):
            g = p.grad = g.detach().resolve_neg().contiguous()
        grads.append(g)
    return clip_grads_(grads, max_norm)


# ------------------------------------------------------------------------------------------------ AdamW
def _numbers(what, name, value, n):
    """One number, or a list of n, as the array of doubles that the library takes."""
    if isinstance(value, (list, tuple)):
        if len(value) != n:
            raise ValueError("%s: %d values of %s for %d tensors" % (what, len(value), name, n))
        values = array("d", value)
        if n and not min(values) >= 0.0:
            raise ValueError("%s: %s must not be negative (got %r)" % (what, name, min(values)))
        return values
    if not value >= 0.0:
        raise ValueError("%s: %s must not be negative (got %r)" % (what, name, value))
    return array("d", [value]) * n


def _rates(what, lr, n):
    """(numbers, addresses of those in device memory or None, the tensors among them)"""
    if isinstance(lr, torch.Tensor):
        lr = [lr] * n
    if not isinstance(lr, (list, tuple)) or not any(isinstance(x, torch.Tensor) for x in lr):
        return _numbers(what, "lr", lr, n), None, []
    tensors = [x for x in lr if isinstance(x, torch.Tensor)]
    for x in tensors:
        if x.numel() != 1 or x.dtype != torch.float32 or x.is_neg():
            raise TypeError("%s: a learning rate in device memory is one float32 (got %s, %s)" % (what, tuple(x.shape), _kind(x)))
    return (_numbers(what, "lr", [0.0 if isinstance(x, torch.Tensor) else x for x in lr], n),
            array("Q", [x.data_ptr() if isinstance(x, torch.Tensor) else 0 for x in lr]), tensors)


def _mend(what, lists, moment_type):
    """Why the lists of a step are not plain: raises what is wrong with them, or returns them with gradients in their parameters' order."""
    params, grads, steps = lists[:3]
    p, g, s = (_List(what, x) for x in lists[:3])
    if g.types != p.types:
        grads = [y.resolve_neg() if y.layout == torch.strided else y for y in grads]
        g = _List(what, grads)
    p.floats(what, "parameters").dense(what, "parameters")
    if g.types != p.types:
        raise TypeError("%s: a gradient has its parameter's type (got %s for %s)" % ((what,) + next(
            (y.dtype if y.layout == torch.strided else y.layout, x.dtype) for x, y in zip(params, grads) if x.dtype != y.dtype or y.layout != torch.strided)))
    for x, y in zip(params, grads):
        if x.shape != y.shape:
            raise ValueError("%s: a gradient has its parameter's shape (got %s for %s)" % (what, tuple(y.shape), tuple(x.shape)))
    if s.type != 0 or s.counts != _ONE * len(steps):
        bad = next(t for t in steps if t.dtype != torch.float32 or t.numel() != 1 or t.layout != torch.strided or t.is_neg())
        raise TypeError("%s: a step counter is one float32 (got %s, %s)" % (what, tuple(bad.shape), _kind(bad)))
    _device_of(what, [p, g, s] + [_List(what, x) for x in lists[3:]])
    for x in lists[3:5]:
        m = _List(what, x)
        if m.type != moment_type:
            raise TypeError("%s: moments must be %s (got %s)" % (what, "float32" if moment_type == 0 else "uint8", sorted({_kind(t) for t in x})))
        at = _tensorlist().differ(params, x)
        if at >= 0:
            t, q = x[at >> 1], params[at >> 1]
            raise ValueError("%s: moments have their parameter's shape and memory order (got %s, strides %s for %s, strides %s)" %
                             (what, tuple(t.shape), t.stride(), tuple(q.shape), q.stride()))
    if len(lists) == 6:
        _check_bases(what, params, lists[5])
    # a gradient in another order of its dimensions (or an expanded one) is brought into the parameter's
    with torch.no_grad():
        grads = [y if _same_order(x, y) else torch.empty_like(x).copy_(y) for x, y in zip(params, grads)]
    return [params, grads] + lists[2:]


def _calls(what, lists, moment_type, lr, betas, eps, weight_decay, ids):
    """(calls, gradients in the parameters' order) of the lists [params, grads, steps, m, v] (32-bit moments) or [..., bases] (8-bit).  A
    call of the library takes tensors of one element type: (lists, (type, device, addresses of each list, counts), rates, addresses of those
    in device memory, the tensors among them, decay, (beta1, beta2, eps), ids)."""
    lists = [x if type(x) is list else list(x) for x in lists]
    n = len(lists[0])
    if any(len(x) != n for x in lists) or (ids is not None and len(ids) != n):
        raise ValueError("%s: the lists differ in length (%s)" % (what, ", ".join(str(len(x)) for x in lists + ([] if ids is None else [ids]))))
    beta1, beta2 = betas
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError("%s: betas must lie in [0, 1) (got %r)" % (what, betas))
    if not eps >= 0.0:
        raise ValueError("%s: eps must not be negative (got %r)" % (what, eps))
    rates, device_rates, tensors = _rates(what, lr, n)
    decay = _numbers(what, "weight_decay", weight_decay, n)
    if n == 0:
        return [], []
    coefficients = (beta1, beta2, eps)
    T = _tensorlist()
    plain = T.step_lists(lists, moment_type, BLOCK)
    if plain is not None:
        return [(lists, plain, rates, device_rates, tensors, decay, coefficients, ids)], lists[1]
    lists = _mend(what, lists, moment_type)
    by_type = {}
    for i, p in enumerate(lists[0]):
        by_type.setdefault(p.dtype, []).append(i)
    calls = []
    for at in by_type.values():
        part = [[x[i] for i in at] for x in lists]
        plain = T.step_lists(part, moment_type, BLOCK)
        if plain is None:
            raise RuntimeError("%s: the lists changed while they were read" % what)
        some = None if device_rates is None else array("Q", [device_rates[i] for i in at])
        calls.append((part, plain, array("d", [rates[i] for i in at]), some, tensors, array("d", [decay[i] for i in at]), coefficients,
                      at if ids is None else [ids[i] for i in at]))
    return calls, lists[1]


def _check_together(what, calls, moment_type, clip):
    """Several calls are one step: all that one of them would refuse is refused before the first."""
    join = lambda parts: b"".join(parts)
    lists, plain, rates, device_rates, _, decay, _, _ = zip(*calls)
    sizes = [len(x[0]) for x in lists]
    types, _, ptrs, counts = zip(*plain)
    p, g, s, m, v = (join(x[k] for x in ptrs) for k in range(5))
    on_device = None
    if any(x is not None for x in device_rates):
        on_device = join(bytes(8 * n) if x is None else x.tobytes() for n, x in zip(sizes, device_rates))
    check(_lib.lib().dtt_adamw_check(sum(sizes), join(array("i", [t]).tobytes() * n for n, t in zip(sizes, types)), p, g, m, v,
                                     None if moment_type == 0 else join(x[5] for x in ptrs), join(counts), s, join(x.tobytes() for x in rates),
                                     on_device, join(x.tobytes() for x in decay), None if clip is None else clip.data_ptr()), what)


def _step(what, jobs, moment_type, max_norm, skip_nonfinite, clip, seed=0):
    """One step of all jobs, each (lists, lr, betas, eps, weight_decay, ids) as _calls takes them, under one norm: done or refused as a
    whole.  Returns the norm or None."""
    if max_norm is not None:
        max_norm = _limit(what, max_norm)
    if clip is not None and (max_norm is not None or clip.dtype != torch.float32 or tuple(clip.shape) != (2,) or not clip.is_contiguous() or clip.is_neg()):
        raise ValueError("%s: clip is norm and factor, two float32, and stands in place of max_norm" % what)
    calls, grads = [], []
    for job in jobs:
        more, own = _calls(what, job[0], moment_type, *job[1:])
        calls = calls + more if calls else more
        grads = grads + own if grads else own
    if not calls:
        return None
    for _, plain, _, _, tensors, _, _, _ in calls:
        if tensors or clip is not None:
            for x in tensors if clip is None else tensors + [clip]:
                if x.get_device() != plain[1]:
                    raise ValueError("%s: all tensors must be on one device (got cuda:%d and %s)" % (what, plain[1], x.device))
    limit = -1.0
    if clip is None and (max_norm is not None or skip_nonfinite):
        limit = math.inf if max_norm is None else max_norm
    if len(calls) > 1:
        _check_together(what, calls, moment_type, clip)
        if limit >= 0.0:                 # one norm over all of them
            grads = _List(what, grads)
            _device_of(what, [grads])
            clip, limit = _norm_and_factor(grads, limit), -1.0
    L, T = _lib.lib(), _tensorlist()
    for lists, (dtype, dev, ptrs, counts), rates, device_rates, _, decay, (beta1, beta2, eps), ids in calls:
        n, device = len(lists[0]), lists[0][0].device
        if limit >= 0.0:                 # the library computes the norm on its way
            clip = torch.empty(2, dtype=torch.float32, device=device)
        nbytes = L.dtt_adamw_workspace_bytes(n, counts)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        rates, decay = rates.tobytes(), decay.tobytes()
        device_rates = None if device_rates is None else device_rates.tobytes()
        tail = (beta1, beta2, eps, limit, None if clip is None else clip.data_ptr(), 1 if skip_nonfinite else 0, ws.data_ptr(), nbytes, _stream(dev))
        with _on(dev):
            if moment_type == 0:
                p, g, s, m, v = ptrs
                check(L.dtt_adamw_step(n, dtype, p, g, m, v, counts, s, rates, device_rates, decay, *tail), what)
            else:
                p, g, s, m, v, b = ptrs
                ids = None if ids is None else array("I", [int(i) & 0xFFFFFFFF for i in ids]).tobytes()
                check(L.dtt_adamw8_step(n, dtype, p, g, m, v, b, counts, s, rates, device_rates, decay, ids, int(seed) & 0xFFFFFFFF, *tail), what)
        T.bump(lists[0])     # (the state is the optimizer's own: its versions would cost 18 us of a 75 us step of 301 tensors)
    return None if clip is None else clip[0]


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
    (float32, 2 entries), in place of max_norm.  Returns the norm (float32 scalar on the device), or None without any of the three.
    Tensors of several types are one step: a call that is refused has changed nothing.  Autograd is told that the parameters changed;
    moments and counters do not count a version."""
    return _step("adamw_", [([params, grads, steps, exp_avgs, exp_avg_sqs], lr, betas, eps, weight_decay, None)], 0, max_norm, skip_nonfinite, clip)


def blocks_of(numel):
    """Blocks (pairs of bases) of the 8-bit moments of a tensor."""
    return (numel + BLOCK - 1) // BLOCK


def adamw8_(params, grads, exp_avgs, exp_avg_sqs, bases, steps, *, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None,
            skip_nonfinite=False, clip=None, seed=0, ids=None):
    """adamw_ with the moments in 8 bits: exp_avgs / exp_avg_sqs are uint8 codes in the parameters' shape and memory order, bases int16
    (blocks_of(numel), 2); all zero = moments of zero.  A value has three bits of mantissa; codes span 15.7 (m) and 31.7 (v) powers of
    two below the largest of their block of 256, what lies lower is 0 (m) or the smallest step (v): an element whose gradients stay
    2^-15.7 below its block's largest is not moved.  The rounding of a moment is dithered, right on average, by a hash of seed, ids
    (default: the position in the list), step counter and element; the same inputs give the same codes.  Infinite and NaN moments, and
    those that round beyond the largest float32, stay in their element, as NaN."""
    return _step("adamw8_", [([params, grads, steps, exp_avgs, exp_avg_sqs, bases], lr, betas, eps, weight_decay, ids)], _UINT8, max_norm,
                 skip_nonfinite, clip, seed)


def _check_bases(what, like, bases):
    at = _tensorlist().rows_of(like, bases, BLOCK)
    if at >= 0:
        b = bases[at]
        raise ValueError("%s: bases are int16, contiguous, (blocks_of(numel), 2): two for each %d elements (got %s, %s, strides %s for %d elements)" %
                         (what, BLOCK, b.dtype, tuple(b.shape), b.stride(), like[at].numel()))


def unpack_moments_(exp_avgs, exp_avg_sqs, bases, out_avgs, out_avg_sqs):
    """Write the values that 8-bit moments stand for into out_avgs / out_avg_sqs (all float32 or all bfloat16, which holds them exactly;
    in the codes' shape and memory order)."""
    what = "unpack_moments_"
    lists = [list(x) for x in (exp_avgs, exp_avg_sqs, bases, out_avgs, out_avg_sqs)]
    n = len(lists[0])
    if any(len(x) != n for x in lists):
        raise ValueError("%s: the lists differ in length (%s)" % (what, ", ".join(str(len(x)) for x in lists)))
    if n == 0:
        return
    m, v, b, x, y = (_List(what, t) for t in lists)
    if x.type not in (0, 1) or y.type != x.type:
        raise TypeError("%s: the values come as float32 or as bfloat16" % what)
    if m.type != _UINT8 or v.type != _UINT8:
        raise TypeError("%s: codes are uint8" % what)
    m.dense(what, "codes")
    if any(_tensorlist().differ(lists[0], t) >= 0 for t in (lists[1], lists[3], lists[4])):
        raise ValueError("%s: codes and values have one shape and memory order" % what)
    dev = _device_of(what, [m, v, b, x, y])
    _check_bases(what, lists[0], lists[2])
    with _on(dev):
        check(_lib.lib().dtt_adamw8_unpack(n, m.ptrs, v.ptrs, b.ptrs, m.counts, x.type, x.ptrs, y.ptrs, _stream(dev)), what)
    _written(lists[3], lists[4])


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
    seed: of the rounding of 8-bit moments.  The moments of bfloat16 / float16 parameters are float32 too.  A step that is refused
    has changed nothing, whatever its groups are.

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
        if m.shape != p.shape or v.shape != p.shape:
            raise ValueError("GroupedAdamW: the state of a parameter of shape %s has shapes %s and %s" % (tuple(p.shape), tuple(m.shape), tuple(v.shape)))
        m, v = (torch.empty_like(p, dtype=torch.float32).copy_(x) for x in (m, v))
        for k in _MOMENTS32 + _MOMENTS8:
            st.pop(k, None)
        if self.state_bits == 32:
            st["exp_avg"], st["exp_avg_sq"] = m, v
        else:
            st["exp_avg_code"], st["exp_avg_sq_code"], st["block_base"] = pack_moments(m, v)

    def _saved(self, src, p):
        """The names of a parameter's moments in a checkpoint; raises where the entry is not a state of this parameter."""
        if "step" not in src or not any(all(k in src for k in names) for names in (_MOMENTS32, _MOMENTS8)):
            raise ValueError("GroupedAdamW: not a state of AdamW or Adam (it holds %s)" % sorted(src))
        step = torch.as_tensor(src["step"])
        if step.numel() != 1:
            raise ValueError("GroupedAdamW: step is one number (the checkpoint has shape %s)" % (tuple(step.shape),))
        names = _MOMENTS32 if all(k in src for k in _MOMENTS32) else _MOMENTS8
        m, v = (src[k] for k in names[:2])
        if m.shape != p.shape or v.shape != p.shape:
            raise ValueError("GroupedAdamW: moments have their parameter's shape (the checkpoint has %s and %s for %s)" %
                             (tuple(m.shape), tuple(v.shape), tuple(p.shape)))
        if names is _MOMENTS8:
            if m.dtype != torch.uint8 or v.dtype != torch.uint8 or not _dense(m) or not _same_order(m, v):
                raise ValueError("GroupedAdamW: codes are uint8, dense, both in one memory order (the checkpoint has %s, strides %s and %s, strides %s)" %
                                 (m.dtype, m.stride(), v.dtype, v.stride()))
            _check_bases("GroupedAdamW", [m], [src[names[2]]])
        if names is _MOMENTS8 and self.state_bits == 32 and not p.is_cuda:
            raise RuntimeError("dtt ops run on the GPU only (8-bit moments of a parameter on %s); there is no CPU fallback" % p.device)
        return names

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Of this class (32 or 8 bits) or of torch.optim.AdamW / Adam.  The moments keep float32 (or their codes) whatever the
        parameters' type is, and are re-packed where the other form was saved.  A checkpoint that is refused changes nothing."""
        for g in state_dict["param_groups"]:
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("GroupedAdamW: a checkpoint with amsgrad or maximize does not load")
        names = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        saved = [(p, state_dict["state"][i]) for i, p in zip(names, params) if i in state_dict["state"]]
        saved = [(p, src, self._saved(src, p)) for p, src in saved]
        for g in state_dict["param_groups"]:
            missing = [k for k in ("lr", "betas", "eps", "weight_decay") if k not in g]
            if missing:
                raise ValueError("GroupedAdamW: not a checkpoint of AdamW or Adam (a group without %s)" % ", ".join(missing))
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})   # (refuses groups of other sizes first)
        moved = {}          # a rate that groups share stays one tensor
        for g in self.param_groups:
            if isinstance(g["lr"], torch.Tensor) and g["params"]:   # (a checkpoint read into host memory)
                lr, dev = g["lr"], g["params"][0].device
                if (id(lr), dev) not in moved:
                    moved[id(lr), dev] = lr, lr.to(device=dev, dtype=torch.float32)
                g["lr"] = moved[id(lr), dev][1]
        for p, src, moments in saved:
            st = self.state[p]
            st["step"] = torch.as_tensor(src["step"]).detach().clone().to(device=p.device, dtype=torch.float32).reshape(())
            for k, dt in zip(moments, (torch.float32, torch.float32) if moments is _MOMENTS32 else (torch.uint8, torch.uint8, torch.int16)):
                st[k] = src[k].detach().to(device=p.device, dtype=dt, copy=True)
            if (moments is _MOMENTS32) != (self.state_bits == 32) or not _same_order(st[moments[0]], st[moments[1]]):
                self._keep_moments(p, st, *self._moments(p, st))

    # ------------------------------------------------------------------ step
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, fresh = {}, []
        state, place = self.state, -1
        names = _MOMENTS32 if self.state_bits == 32 else _MOMENTS8
        for g in self.param_groups:
            key = (g["betas"], g["eps"])
            key = key if type(key[0]) is tuple else (tuple(key[0]), key[1])
            rows = work.get(key)
            if rows is None:
                rows = work[key] = ([], [], [], [], [])
            lr, decay = g["lr"], g["weight_decay"]
            for p in g["params"]:
                place += 1
                grad = p.grad
                if grad is None:
                    continue
                if not state.get(p):
                    fresh.append(p)
                rows[0].append(p)
                rows[1].append(grad)
                rows[2].append(lr)
                rows[3].append(decay)
                rows[4].append(place)
        work = {k: rows for k, rows in work.items() if rows[0]}
        if not work:
            self.grad_norm = None
            return loss
        what = "GroupedAdamW"
        if fresh:
            for rows in work.values():
                _device_of(what, [_List(what, rows[0]).floats(what, "parameters").dense(what, "parameters"), _List(what, rows[1])])
        try:
            if fresh:
                self._make_state(fresh)
            jobs = []
            for (betas, eps), (params, grads, lr, decay, places) in work.items():
                states = [state[p] for p in params]
                m = [st[names[0]] for st in states]
                at = _tensorlist().differ(params, m)
                while at >= 0:      # the parameter took another memory order since (channels-last filters)
                    i = at >> 1
                    if at & 1 == 0:
                        raise ValueError("GroupedAdamW: the state of a parameter of shape %s has shape %s" % (tuple(params[i].shape), tuple(m[i].shape)))
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("GroupedAdamW: run a step before capturing one (the state follows a parameter's new memory order)")
                    self._keep_moments(params[i], states[i], *self._moments(params[i], states[i]))
                    m[i] = states[i][names[0]]
                    at = _tensorlist().differ(params, m)
                lists = [params, grads, [st["step"] for st in states], m, [st[names[1]] for st in states]]
                if self.state_bits == 8:
                    lists.append([st["block_base"] for st in states])
                jobs.append((lists, lr, betas, eps, decay, places))
            self.grad_norm = _step(what, jobs, 0 if self.state_bits == 32 else _UINT8, self.max_norm, self.skip_nonfinite, None, self.seed)
        except Exception:
            for p in fresh:         # a refused step leaves no state behind
                state.pop(p, None)
            raise
        return loss
