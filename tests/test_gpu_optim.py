"""The optimizer operators (dtt/optim.py, csrc/optim.hip) on the GPU against 64-bit formulas (oracle/optim_oracle.py).

Tolerances are the oracle's counted rounding errors (each rounding half a step of its type: fp32 2^-24, bf16 2^-8, fp16 2^-11
of the value), not measured ones; codes of the 8-bit moments are compared for equality."""
import copy
import math

import numpy as np
import pytest
import torch

from oracle import optim_oracle as oo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
SIZES = [1, 2, 3, 255, 256, 257, 1023, 4096, 4097, 0, 16384, 16385, 70001]


def f64(t):
    return t.detach().double().cpu().numpy()


def place(sizes, dtype, packed, seed, scale=1.0):
    """One buffer and its views: neighbours without a gap (packed: no view is aligned), or 64 elements of guard behind each."""
    gap = 0 if packed else 64
    total = sum(sizes) + gap * len(sizes) + 1
    g = torch.Generator().manual_seed(seed)
    flat = (torch.randn(total, generator=g) * scale).to(dtype).to(DEV)
    at, views = 1 if packed else 0, []
    for n in sizes:
        views.append(flat[at:at + n])
        at += n + gap
    return flat, views


def spread(n, seed, lo=-12.0, hi=2.0):
    """Values over decades, both signs, some zero."""
    rs = np.random.RandomState(seed)
    return (np.exp(rs.uniform(lo, hi, n)) * np.sign(rs.randn(n)) * (rs.rand(n) > 0.1)).astype(np.float32)


# ------------------------------------------------------------------------------------------------ norm, clipping
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", list(HALF), ids=str)
def test_clip_scales_to_the_limit(dtype, packed):
    from dtt.optim import clip_grads_, grad_norm
    flat, grads = place(SIZES, dtype, packed, 1)
    before = f64(flat)
    host = [f64(g) for g in grads]
    for limit in (math.inf, 1e9, 3.0, 0.0):
        flat.copy_(torch.from_numpy(before))
        norm, c = oo.norm_and_factor(host, limit)
        c = 1.0 if math.isinf(limit) else c
        assert abs(float(grad_norm(grads)) - norm) <= norm * 2.0 ** -23    # (the sums' own error, 2^-53 a term, is far below)
        assert abs(float(clip_grads_(grads, limit)) - norm) <= norm * 2.0 ** -23
        want = before.copy()
        at = 1 if packed else 0
        for n in SIZES:
            want[at:at + n] *= c
            at += n + (0 if packed else 64)
        got = f64(flat)
        # the factor and the product are rounded (2 * 2^-24), then the type
        tol = np.abs(want) * (2 * oo.U + HALF[dtype]) + SMALLEST[dtype] if c != 1.0 else 0.0
        assert (np.abs(got - want) <= tol).all(), (limit, np.abs(got - want).max())


def test_norm_of_mixed_types_many_tensors_and_extreme_values():
    from dtt.optim import clip_grads_, grad_norm
    rs = np.random.RandomState(3)
    types = list(HALF)
    grads = [torch.from_numpy(rs.randn(int(rs.randint(0, 3000))).astype(np.float32)).to(DEV).to(types[i % 3]) for i in range(401)]
    norm, _ = oo.norm_and_factor([f64(g) for g in grads], 1.0)
    first = grad_norm(grads)
    assert abs(float(first) - norm) <= norm * 2.0 ** -23
    assert all(torch.equal(grad_norm(grads), first) for _ in range(5))                # fixed order: the same bits
    # channels-last, transposed, scalar tensors: any dense order
    odd = [torch.randn(3, 5, 7, 2, device=DEV).contiguous(memory_format=torch.channels_last), torch.randn(17, 9, device=DEV).t(),
           torch.randn((), device=DEV), torch.randn(4, 1, 6, device=DEV).permute(2, 1, 0)]
    norm, c = oo.norm_and_factor([f64(g) for g in odd], 0.5)
    want = [f64(g) * c for g in odd]
    assert abs(float(clip_grads_(odd, 0.5)) - norm) <= norm * 2.0 ** -23
    assert all((np.abs(f64(g) - w) <= np.abs(w) * 3 * oo.U).all() for g, w in zip(odd, want))
    # squares beyond fp32, values whose squares vanish in fp32, infinities, NaN
    big = [torch.full((1000,), 1e30, device=DEV), torch.full((7,), -3e38, device=DEV)]
    norm = oo.norm_and_factor([f64(g) for g in big], 1.0)[0]
    assert math.isinf(np.float32(norm)) == math.isinf(float(grad_norm(big)))
    small = [torch.full((1000,), 1e-30, device=DEV)]
    assert abs(float(grad_norm(small)) - math.sqrt(1000) * 1e-30) <= math.sqrt(1000) * 1e-30 * 2.0 ** -22   # (1e-30 itself is rounded)
    large = [torch.full((100,), 1e30, device=DEV)]
    assert abs(float(grad_norm(large)) - 1e31) <= 1e31 * 2.0 ** -22
    bad = torch.ones(5000, device=DEV)
    bad[4321] = math.inf
    assert math.isinf(float(grad_norm([bad])))
    bad[17] = math.nan
    assert math.isnan(float(grad_norm([bad, torch.ones(3, device=DEV)])))
    assert float(grad_norm([torch.empty(0, device=DEV)])) == 0.0


def test_clip_of_many_tensors_of_mixed_types():
    """More tensors than a launch holds, empty ones among them, one norm over three types; within the limit nothing is written."""
    from dtt.optim import clip_grads_
    rs = np.random.RandomState(4)
    types = list(HALF)
    grads = [torch.from_numpy(rs.randn(int(rs.randint(0, 2000)) if i % 9 else 0).astype(np.float32)).to(DEV).to(types[i % 3]) for i in range(401)]
    old = [f64(g) for g in grads]
    norm, c = oo.norm_and_factor(old, 10.0)
    assert c < 1
    first = [g.clone() for g in grads]
    assert abs(float(clip_grads_(grads, 1e6)) - norm) <= norm * 2.0 ** -23 and all(torch.equal(a, b) for a, b in zip(grads, first))
    assert abs(float(clip_grads_(grads, 10.0)) - norm) <= norm * 2.0 ** -23
    for g, o in zip(grads, old):
        assert (np.abs(f64(g) - o * c) <= np.abs(o * c) * (2 * oo.U + HALF[g.dtype]) + SMALLEST[g.dtype]).all()
    empty = [torch.empty(0, device=DEV), torch.empty(0, 3, device=DEV, dtype=torch.bfloat16)]
    assert float(clip_grads_(empty, 1.0)) == 0.0


def test_clip_grad_norm_over_parameters():
    from dtt.optim import clip_grad_norm_
    torch.manual_seed(0)
    a, b, c, d = (torch.nn.Parameter(torch.randn(*s, device=DEV)) for s in ((30, 4), (7,), (5, 5), (64, 3)))
    (a.square().sum() + b.sum() + (d * 0.1).mean()).backward()         # c has no gradient, b's is an expanded view
    ref = [x.grad.clone() for x in (a, b, d)]
    norm = float(torch.sqrt(sum(x.double().square().sum() for x in ref)))
    version = a.grad._version
    assert abs(float(clip_grad_norm_([a, b, c, d], 0.25)) - norm) <= norm * 2.0 ** -23
    assert c.grad is None and a.grad._version > version
    f = 0.25 / (norm + 1e-6)
    for x, r in zip((a, b, d), ref):
        assert ((x.grad.double() - r.double() * f).abs() <= r.double().abs() * f * 3 * oo.U).all()
    assert abs(float(clip_grad_norm_(a, 1e9)) - float(a.grad.double().norm())) <= 1e-6


def test_a_gradient_given_twice_is_refused():
    from dtt.optim import clip_grads_
    g = torch.ones(100, device=DEV)
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grads_([g, g], 1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grads_([g[:60], g[50:]], 1.0)
    with pytest.raises(ValueError, match="dense"):
        clip_grads_([g[::2]], 1.0)
    assert float(g.sum()) == 100.0


# ------------------------------------------------------------------------------------------------ AdamW, 32-bit moments
def state_of(sizes, dtype, packed, seed):
    fp, p = place(sizes, dtype, packed, seed, 0.05)
    fg, g = place(sizes, dtype, packed, seed + 1)
    fm, m = place(sizes, torch.float32, packed, seed + 2)
    fv, v = place(sizes, torch.float32, packed, seed + 3)
    for i, n in enumerate(sizes):
        g[i].copy_(torch.from_numpy(spread(n, seed + 10 + i)))
        m[i].copy_(torch.from_numpy(spread(n, seed + 50 + i)))
        v[i].copy_(torch.from_numpy(np.square(spread(n, seed + 90 + i))))
        m[i][v[i] == 0] = 0          # (what has no second moment has never moved)
    return (fp, fg, fm, fv), p, g, m, v


def check_step(p0, g0, m0, v0, t, p, m, v, dtype, **k):
    wp, wm, wv, ep, em, ev = oo.adamw(p0, g0, m0, v0, t, **k)
    gm, gv, gp = f64(m), f64(v), f64(p)
    assert (np.abs(gm - wm) <= em).all(), ("m", np.abs(gm - wm).max())
    assert (np.abs(gv - wv) <= ev).all(), ("v", np.abs(gv - wv).max())
    ep = ep + (0 if dtype == torch.float32 else HALF[dtype] * (np.abs(wp) + ep) + SMALLEST[dtype])
    assert (np.abs(gp - wp) <= ep).all(), ("p", float((np.abs(gp - wp) / ep).max()))


@pytest.mark.parametrize("clipped", [False, True])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", list(HALF), ids=str)
def test_adamw_steps_match_64_bits(dtype, packed, clipped):
    from dtt.optim import adamw_
    flats, p, g, m, v = state_of(SIZES, dtype, packed, 5)
    outside = [f64(x) for x in flats]
    steps = [torch.zeros((), device=DEV) for _ in SIZES]
    lr = [1e-3 * (1 + i % 3) for i in range(len(SIZES))]
    decay = [0.0 if i % 2 else 0.1 for i in range(len(SIZES))]
    limit = 2.0 if clipped else None
    for t in (1, 2, 3):
        old = [[f64(x) for x in row] for row in zip(p, g, m, v)]
        norm = adamw_(p, g, m, v, steps, lr=lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=decay, max_norm=limit)
        c = 1.0
        if clipped:
            n64, c = oo.norm_and_factor([o[1] for o in old], limit)
            assert abs(float(norm) - n64) <= n64 * 2.0 ** -23
        else:
            assert norm is None
        for i, o in enumerate(old):
            check_step(*o, t, p[i], m[i], v[i], dtype, lr=lr[i], beta1=0.9, beta2=0.999, eps=1e-8, decay=decay[i], c=c)
            assert np.array_equal(f64(g[i]), o[1]) and float(steps[i]) == t
    at = 1 if packed else 0                                                            # what lies between the tensors
    keep = np.ones(flats[0].numel(), dtype=bool)
    for n in SIZES:
        keep[at:at + n] = False
        at += n + (0 if packed else 64)
    assert all(np.array_equal(f64(x)[keep], o[keep]) for x, o in zip(flats, outside))


def test_adamw_many_tensors_of_mixed_types_and_orders():
    """More tensors than a launch holds, three types, channels-last filters, gradients in another order than their parameter's,
    expanded gradients, counters that differ."""
    from dtt.optim import adamw_
    torch.manual_seed(2)
    rs = np.random.RandomState(2)
    types = list(HALF)
    params = [torch.randn(int(rs.randint(1, 900)), device=DEV).to(types[i % 3]) for i in range(260)]
    params += [torch.randn(8, 4, 3, 3, device=DEV).contiguous(memory_format=torch.channels_last), torch.randn(9, 7, device=DEV).t(),
               torch.randn(6, 5, device=DEV), torch.randn((), device=DEV), torch.randn(4, 8, 1, 1, device=DEV)]
    grads = [torch.randn_like(p) for p in params]
    grads[-5] = grads[-5].contiguous()                                   # row-major for a channels-last parameter
    grads[-3] = torch.full((1, 1), 0.5, device=DEV).expand(6, 5)         # broadcast
    grads[-1] = grads[-1].as_strided((4, 8, 1, 1), (8, 1, 8, 8))         # the same memory under another name
    ms = [torch.randn_like(p, dtype=torch.float32) for p in params]
    vs = [torch.randn_like(p, dtype=torch.float32).square() for p in params]
    steps = [torch.full((), float(i % 7), device=DEV) for i in range(len(params))]
    old = [[f64(x) for x in row] for row in zip(params, grads, ms, vs)]
    adamw_(params, grads, ms, vs, steps, lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.01)
    for i, o in enumerate(old):
        check_step(*o, i % 7 + 1, params[i], ms[i], vs[i], params[i].dtype, lr=1e-2, beta1=0.8, beta2=0.95, eps=1e-6, decay=0.01)


@pytest.mark.parametrize("beta1,beta2,eps", [(0.0, 0.0, 1e-8), (0.9, 0.999, 1.0), (0.0, 0.999, 1e-8), (0.95, 0.9999, 1e-12)])
def test_adamw_corner_coefficients(beta1, beta2, eps):
    from dtt.optim import adamw_
    for t0 in (0, 9, 100000):
        _, p, g, m, v = state_of([1000], torch.float32, True, 33)
        if t0 == 0:
            m[0].zero_(), v[0].zero_()
        s = torch.full((), float(t0), device=DEV)
        old = [f64(x[0]) for x in (p, g, m, v)]
        adamw_(p, g, m, v, [s], lr=0.1, betas=(beta1, beta2), eps=eps, weight_decay=0.5)
        check_step(*old, t0 + 1, p[0], m[0], v[0], torch.float32, lr=0.1, beta1=beta1, beta2=beta2, eps=eps, decay=0.5)


def test_adamw_zero_gradients_infinities_and_skipping():
    from dtt.optim import adamw8_, adamw_
    n = 700
    one = torch.ones(n, device=DEV)
    # nothing has ever moved: 0 / (0 + eps) = 0, only the decay acts
    p, m, v, s = one.clone(), one * 0, one * 0, torch.zeros((), device=DEV)
    adamw_([p], [one * 0], [m], [v], [s], lr=0.1, weight_decay=0.5)
    assert torch.equal(p, one * np.float32(1 - 0.1 * 0.5)) and not m.any() and not v.any()
    # a NaN and an infinity stay in their element
    for bits in (32, 8):
        p = one.clone()
        g = one.clone()
        g[300], g[301] = math.nan, math.inf
        s = torch.zeros((), device=DEV)
        if bits == 32:
            m, v = one * 0, one * 0
            call = lambda **k: adamw_([p], [g], [m], [v], [s], lr=0.1, weight_decay=0.0, **k)
            state = lambda: [m, v]
        else:
            cm, cv, b = (torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV),
                         torch.zeros(3, 2, dtype=torch.int16, device=DEV))
            call = lambda **k: adamw8_([p], [g], [cm], [cv], [b], [s], lr=0.1, weight_decay=0.0, **k)
            state = lambda: [cm, cv, b]
        before = [x.clone() for x in state()]
        norm = call(skip_nonfinite=True)                               # skipped: nothing moves, the counter neither
        assert math.isnan(float(norm)) and torch.equal(p, one) and float(s) == 0.0
        assert all(torch.equal(x, y) for x, y in zip(state(), before))
        g[300] = 1.0
        assert math.isinf(float(call(skip_nonfinite=True, max_norm=1.0))) and torch.equal(p, one) and float(s) == 0.0
        g[300] = math.nan
        call()
        ok = torch.ones(n, dtype=torch.bool, device=DEV)
        ok[300:302] = False
        assert float(s) == 1.0 and torch.isnan(p[300]) and not torch.isfinite(p[301])
        assert torch.equal(p[ok], torch.full((n - 2,), float(p[0]), device=DEV)) and abs(float(p[0]) - 0.9) < 1e-6
        g[300:302] = 1.0
        call()                                                         # and the neighbours go on
        assert torch.isfinite(p[ok]).all() and torch.isnan(p[300])
        g2 = one * 2
        q, norm2 = p.clone(), None
        norm2 = adamw_([q], [g2], [one * 0], [one * 0], [torch.zeros((), device=DEV)], lr=0.1, skip_nonfinite=True)
        assert abs(float(norm2) - 2 * math.sqrt(n)) < 1e-4             # finite: not skipped
        assert not torch.equal(q[ok], p[ok])


def test_adamw_refuses_overlaps_and_wrong_moments():
    from dtt.optim import adamw8_, adamw_
    x = [torch.zeros(100, device=DEV) for _ in range(8)]
    s = [torch.zeros((), device=DEV) for _ in range(2)]
    with pytest.raises(RuntimeError, match="share memory"):
        adamw_([x[0], x[0]], x[1:3], x[3:5], x[5:7], s, lr=1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        adamw_([x[0]], [x[1]], [x[2]], [x[2]], s[:1], lr=1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        adamw_(x[:2], x[2:4], x[4:6], x[6:8], [s[0], s[0]], lr=1.0)
    with pytest.raises(ValueError, match="memory order"):
        adamw_([x[0].view(10, 10)], [x[1].view(10, 10)], [x[2].view(10, 10).t()], [x[3].view(10, 10)], s[:1], lr=1.0)
    with pytest.raises(TypeError, match="moments must be"):
        adamw_([x[0]], [x[1]], [x[2].half()], [x[3]], s[:1], lr=1.0)
    codes = [torch.zeros(100, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for bases in (torch.zeros(2, 2, dtype=torch.int16, device=DEV), torch.zeros(1, 2, device=DEV), torch.zeros(1, 4, dtype=torch.int16, device=DEV)[:, ::2]):
        with pytest.raises(ValueError, match="bases"):
            adamw8_([x[0]], [x[1]], codes[:1], codes[1:], [bases], s[:1], lr=1.0)
    with pytest.raises(RuntimeError, match="GPU only"):
        adamw_([x[0]], [x[1]], [x[2]], [x[3].cpu()], s[:1], lr=1.0)
    assert all(not t.any() for t in x) and float(s[0]) == 0.0


# ------------------------------------------------------------------------------------------------ 8-bit moments
def state8_of(sizes, dtype, packed, seed):
    from dtt.optim import blocks_of
    flats, p, g, _, _ = state_of(sizes, dtype, packed, seed)
    fcm, cm = place(sizes, torch.float32, packed, 0, 0.0)
    fcm, fcv = fcm.to(torch.uint8), fcm.to(torch.uint8)
    at, cm, cv, bases = 1 if packed else 0, [], [], []
    for i, n in enumerate(sizes):
        v = np.square(spread(n, seed + 90 + i))
        a, b, c = oo.encode(spread(n, seed + 50 + i) * (v > 0), v, 1 << 19, 1 << 19)
        cm.append(fcm[at:at + n].copy_(torch.from_numpy(a)))
        cv.append(fcv[at:at + n].copy_(torch.from_numpy(b)))
        bases.append(torch.from_numpy(c.reshape(blocks_of(n), 2)).to(DEV))
        at += n + (0 if packed else 64)
    return (flats[0], fcm, fcv), p, g, cm, cv, bases


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", list(HALF), ids=str)
def test_adamw8_codes_are_those_of_the_definition(dtype, packed):
    from dtt.optim import adamw8_
    flats, p, g, cm, cv, bases = state8_of(SIZES, dtype, packed, 7)
    outside = [f64(x) for x in flats]
    steps = [torch.full((), 41.0, device=DEV) for _ in SIZES]
    ids = [3 * i + 1 for i in range(len(SIZES))]
    lr = [1e-3 * (1 + i % 3) for i in range(len(SIZES))]
    for t in (42, 43):
        old = [[f64(p[i]), g[i].float().cpu().numpy(), *oo.decode(cm[i].cpu().numpy(), cv[i].cpu().numpy(), bases[i].cpu().numpy())]
               for i in range(len(SIZES))]
        assert adamw8_(p, g, cm, cv, bases, steps, lr=lr, weight_decay=0.1, seed=1234567891011, ids=ids) is None
        for i, (p0, g0, m0, v0) in enumerate(old):
            m1, v1 = oo.moments_f32(g0, m0, v0, 0.9, 0.999)
            em, ev, eb = oo.encode(m1, v1, *oo.dither(SIZES[i], 1234567891011 & 0xFFFFFFFF, ids[i], t))
            assert np.array_equal(bases[i].cpu().numpy(), eb), SIZES[i]
            assert np.array_equal(cv[i].cpu().numpy(), ev), SIZES[i]
            got, same = cm[i].cpu().numpy(), em & 127 != 0               # (a zero's sign does not matter)
            assert np.array_equal(got & 127, em & 127) and np.array_equal(got[same], em[same]), SIZES[i]
            wp, wm, wv, ep, _, _ = oo.adamw(p0, g0, m0, v0, t, lr[i], 0.9, 0.999, 1e-8, 0.1)
            ep = ep + (0 if dtype == torch.float32 else HALF[dtype] * (np.abs(wp) + ep) + SMALLEST[dtype])
            assert (np.abs(f64(p[i]) - wp) <= ep).all()
            # and they are what 64 bits give, to a level (1/8 of a value) or the end of the span
            dm, dv = oo.decode(em, ev, eb)
            if SIZES[i]:
                top = np.array([np.abs(wm[k // 256 * 256:k // 256 * 256 + 256]).max() for k in range(SIZES[i])])
                assert (np.abs(dm - wm) <= np.maximum(np.abs(wm) / 8 * 1.001, top * 2.0 ** -15.5)).all()
                assert ((dv > 0) == (wv > 0)).all()
    at = 1 if packed else 0
    keep = np.ones(flats[0].numel(), dtype=bool)
    for n in SIZES:
        keep[at:at + n] = False
        at += n + (0 if packed else 64)
    assert all(np.array_equal(f64(x)[keep], o[keep]) for x, o in zip(flats, outside))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_unpacked_moments_are_the_codes_values(dtype):
    from dtt.optim import unpack_moments_
    rs = np.random.RandomState(1)
    sizes = [1, 5, 255, 256, 257, 5000, 0, 16385] * 12
    codes = [[torch.from_numpy(rs.randint(0, 256, n).astype(np.uint8)).to(DEV) for n in sizes] for _ in range(2)]
    bases = [rs.randint(0, 1700, ((n + 255) // 256, 2)).astype(np.int16) for n in sizes]
    for b in bases:
        b[::3] |= 0x4000
    dbases = [torch.from_numpy(b).to(DEV) for b in bases]
    om, ov = ([torch.full((n,), 7.0, dtype=dtype, device=DEV) for n in sizes] for _ in range(2))
    unpack_moments_(codes[0], codes[1], dbases, om, ov)
    for i in range(len(sizes)):
        wm, wv = oo.decode(codes[0][i].cpu().numpy(), codes[1][i].cpu().numpy(), bases[i])
        assert np.array_equal(om[i].float().cpu().numpy(), wm, equal_nan=True) and np.array_equal(ov[i].float().cpu().numpy(), wv, equal_nan=True)
    with pytest.raises(TypeError):
        unpack_moments_(codes[0], codes[1], dbases, [x.half() for x in om], [x.half() for x in ov])
    with pytest.raises(RuntimeError, match="share memory"):
        unpack_moments_(codes[0][:1], codes[1][:1], dbases[:1], om[:1], om[:1])


def test_8_bit_moments_follow_32_bit_ones_on_average():
    """Long runs of noise whose size drops by ten: the mean of the 8-bit v over 2^17 elements follows the 32-bit one.  One element's v
    has a standard deviation of sqrt(0.125 / 2) = 0.25 of its value from the rounding and 0.03 from the noise; over 2^17 elements
    0.0007, and the terms' 16 bits leave a drift of at most 2^-17 of a level a step, 1000 steps long: 0.125 * 2^-17 * 1000 = 0.001.
    Five standard deviations and the drift are under 0.005.  (To the nearest level v would keep its first value.)"""
    from dtt.optim import adamw8_, adamw_, blocks_of, unpack_moments_
    n = 1 << 17
    gen = torch.Generator(device=DEV).manual_seed(5)
    p8, p32, m, v = (torch.zeros(n, device=DEV) for _ in range(4))
    cm, cv = (torch.zeros(n, dtype=torch.uint8, device=DEV) for _ in range(2))
    b = torch.zeros(blocks_of(n), 2, dtype=torch.int16, device=DEV)
    s8, s32 = torch.zeros((), device=DEV), torch.zeros((), device=DEV)
    vm, vv = torch.empty(n, device=DEV), torch.empty(n, device=DEV)
    for t in range(3000):
        g = torch.randn(n, device=DEV, generator=gen) * (1.0 if t < 1000 else 0.1) + 0.01
        adamw8_([p8], [g], [cm], [cv], [b], [s8], lr=1e-3, weight_decay=0.0, seed=9)
        adamw_([p32], [g], [m], [v], [s32], lr=1e-3, weight_decay=0.0)
        if t in (500, 999, 2000, 2999):
            unpack_moments_([cm], [cv], [b], [vm], [vv])
            assert abs(float(vv.double().mean() / v.double().mean()) - 1) < 0.005, t
            # m: noise of one element, 0.12 / sqrt(6) * sqrt(1 / 0.19) = 0.11 of a value; its mean over the elements against the noise's size
            assert abs(float((vm.double() - m.double()).mean())) < 5 * 0.11 * float(m.double().abs().mean()) / math.sqrt(n) * 2, t


# ------------------------------------------------------------------------------------------------ streams, graphs, sizes
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on_and_equal_eager_ones(bits):
    """Two graphs of two optimizers, replayed in turn with eager work between, against eager twins; the learning rate is a tensor."""
    from dtt.optim import GroupedAdamW
    torch.manual_seed(4)
    shapes = [(300, 17), (5,), (70, 70), (1,)]

    def build():
        ps = [torch.nn.Parameter(torch.randn(*s, device=DEV)) for s in shapes]
        for p in ps:
            p.grad = torch.zeros_like(p)
        rate = torch.full((), 1e-2, device=DEV)
        return ps, rate, GroupedAdamW([{"params": [p], "weight_decay": 0.1 * (p.dim() > 1)} for p in ps], lr=rate, state_bits=bits, max_norm=1.0,
                                      skip_nonfinite=True)
    pairs = []
    for k in range(2):
        torch.manual_seed(k)
        a = build()
        torch.manual_seed(k)
        pairs.append((a, build()))
    def gradients(ps, seed):
        torch.manual_seed(seed)
        for p in ps:
            p.grad.copy_(torch.randn_like(p))
    graphs = []
    side = torch.cuda.Stream()
    for (ps, rate, opt), (qs, _, ref) in pairs:
        gradients(ps, 1); gradients(qs, 1)
        fresh = GroupedAdamW([torch.nn.Parameter(torch.ones(3, device=DEV))], state_bits=bits)
        fresh.param_groups[0]["params"][0].grad = torch.ones(3, device=DEV)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            opt.step()
        torch.cuda.current_stream().wait_stream(side)
        ref.step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            with pytest.raises(RuntimeError, match="before capturing"):
                fresh.step()
            opt.step()
        graphs.append(g)
    for it in range(4):
        for g, ((ps, rate, opt), (qs, qrate, ref)) in zip(graphs, pairs):
            rate.fill_(1e-2 / (1 + it)); qrate.fill_(1e-2 / (1 + it))
            gradients(ps, 10 + it); gradients(qs, 10 + it)
            if it == 2:
                ps[0].grad[0, 0] = math.inf; qs[0].grad[0, 0] = math.inf        # this one is skipped, on the device
            g.replay()
            ref.step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(ps, qs)), it
            assert float(opt.state[ps[0]]["step"]) == float(ref.state[qs[0]]["step"]) == 2 + it - (it >= 2)
            for p, q in zip(ps, qs):
                assert all(torch.equal(opt.state[p][k], ref.state[q][k]) for k in opt.state[p])


def test_steps_on_another_stream_and_two_at_once():
    from dtt.optim import adamw_, clip_grads_
    sets = []
    for k in range(2):
        _, p, g, m, v = state_of([100000, 33], torch.float32, True, 60 + k)
        sets.append((p, g, m, v, [torch.zeros((), device=DEV) for _ in range(2)]))
    want = []
    for p, g, m, v, s in sets:
        c = [[x.clone() for x in l] for l in (p, g, m, v, s)]
        for _ in range(5):
            clip_grads_(c[1], 0.5)
            adamw_(*c, lr=1e-2, max_norm=0.3)
        want.append(c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                clip_grads_(s[1], 0.5)
                adamw_(*s, lr=1e-2, max_norm=0.3)
    torch.cuda.synchronize()
    for got, w in zip(sets, want):
        assert all(torch.equal(a, b) for x, y in zip(got, w) for a, b in zip(x, y))


def test_more_rates_than_a_launch_holds_and_rates_in_device_memory():
    from dtt.optim import adamw8_, adamw_, blocks_of
    rs = np.random.RandomState(9)
    n = 290
    params = [torch.from_numpy(rs.randn(37).astype(np.float32)).to(DEV) for _ in range(n)]
    grads = [torch.randn(37, device=DEV) for _ in range(n)]
    ms, vs = ([torch.zeros(37, device=DEV) for _ in range(n)] for _ in range(2))
    steps = list(torch.zeros(n, device=DEV).unbind())
    on_device = [torch.full((1,) if i % 2 else (), 1e-2 / (i + 1), device=DEV) for i in range(n)]
    lr = [on_device[i] if i % 3 == 0 else 1e-2 / (i + 1) for i in range(n)]
    decay = [0.1 * (i % 11) for i in range(n)]
    old = [[f64(x) for x in row] for row in zip(params, grads, ms, vs)]
    q = [p.clone() for p in params]
    adamw_(params, grads, ms, vs, steps, lr=lr, weight_decay=decay)
    codes = [[torch.zeros(37, dtype=torch.uint8, device=DEV) for _ in range(n)] for _ in range(2)]
    bases = [torch.zeros(blocks_of(37), 2, dtype=torch.int16, device=DEV) for _ in range(n)]
    adamw8_(q, grads, codes[0], codes[1], bases, list(torch.zeros(n, device=DEV).unbind()), lr=lr, weight_decay=decay)
    for i, o in enumerate(old):
        rate = float(on_device[i]) if i % 3 == 0 else lr[i]
        check_step(*o, 1, params[i], ms[i], vs[i], torch.float32, lr=rate, beta1=0.9, beta2=0.999, eps=1e-8, decay=decay[i])
        wp, _, _, ep, _, _ = oo.adamw(*o, 1, rate, 0.9, 0.999, 1e-8, decay[i])
        assert (np.abs(f64(q[i]) - wp) <= ep).all()
    with pytest.raises(ValueError, match="one device"):
        adamw_(params, grads, ms, vs, steps, lr=torch.zeros(()))


@pytest.mark.parametrize("bits", [32, 8])
def test_tiny_eps_and_subnormal_second_moments(bits):
    """Gradients whose second moments are subnormal in fp32, beside an eps that does not hide them (the 8-bit step's quotient takes
    its exact form there)."""
    from dtt.optim import adamw8_, adamw_, blocks_of
    n = 512
    g = torch.from_numpy((np.random.RandomState(2).uniform(3e-21, 3e-19, n) * np.where(np.arange(n) % 2, 1, -1)).astype(np.float32)).to(DEV)
    for eps in (0.0, 1e-25, 1e-12):
        p, s = torch.ones(n, device=DEV), torch.zeros((), device=DEV)
        if bits == 32:
            adamw_([p], [g], [torch.zeros(n, device=DEV)], [torch.zeros(n, device=DEV)], [s], lr=0.1, betas=(0.5, 0.5), eps=eps, weight_decay=0.0)
        else:
            adamw8_([p], [g], [torch.zeros(n, dtype=torch.uint8, device=DEV)], [torch.zeros(n, dtype=torch.uint8, device=DEV)],
                    [torch.zeros(blocks_of(n), 2, dtype=torch.int16, device=DEV)], [s], lr=0.1, betas=(0.5, 0.5), eps=eps, weight_decay=0.0)
        x = g.double().cpu().numpy()
        v = 0.5 * x * x
        den = np.sqrt(v) / np.sqrt(0.5) + eps
        # v is rounded to multiples of 2^-149: relative error 2^-149 / v (square and sum), half of it in the root
        want, rel = 1 - 0.1 / 0.5 * 0.5 * x / den, np.minimum(1.0, 2 * 2.0 ** -149 / v) + 16 * oo.U
        assert (np.abs(f64(p) - want) <= 0.1 * np.abs(x / den) * rel + 2 * oo.U).all(), (eps, np.abs(f64(p) - want).max())


def test_gradients_in_flat_buckets_give_the_same_step():
    """The data-parallel wrapper hands gradients over as views of flat buckets, none of them aligned: bit for bit the same update."""
    from dtt.dist import DataParallelSnippets
    from dtt.optim import GroupedAdamW
    a, b = _model(6), _model(6)
    runner = DataParallelSnippets(b, 1, bucket_bytes=4096, force_buckets=True)
    oa, ob = (GroupedAdamW(m.parameters(), lr=1e-2, max_norm=0.05) for m in (a, b))
    for t in range(3):
        torch.manual_seed(t)
        x = torch.randn(4, 3, 6, 6, device=DEV)
        oa.zero_grad(set_to_none=True)
        runner.zero_grad(set_to_none=True)
        a(x).square().mean().backward()
        runner(x).square().mean().backward()
        runner.finish_gradients()
        for p, q in zip(a.parameters(), b.parameters()):
            q.grad.copy_(p.grad)             # (the library's convolution gradients need not be the same bits twice)
        oa.step(); ob.step()
        # (sums and elements go by index, not by address)
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))


def test_offsets_beyond_32_bits():
    """A tensor of more than 2^32 elements (bf16, 8-bit moments): its end is what a small tensor with the same values gives."""
    from dtt.optim import adamw8_, blocks_of, grad_norm
    n = (1 << 32) + 1000
    p = torch.full((n,), 0.5, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    cm, cv = (torch.zeros(n, dtype=torch.uint8, device=DEV) for _ in range(2))
    b = torch.zeros(blocks_of(n), 2, dtype=torch.int16, device=DEV)
    tail = torch.from_numpy(spread(1000, 1)).to(DEV).bfloat16()
    g[-1000:] = tail
    assert abs(float(grad_norm([g])) - float(tail.double().norm())) <= float(tail.double().norm()) * 2.0 ** -23
    s = torch.zeros((), device=DEV)
    adamw8_([p], [g], [cm], [cv], [b], [s], lr=0.1, weight_decay=0.0, seed=3)
    h = tail.float().cpu().numpy()
    m1, v1 = oo.moments_f32(h, np.zeros(1000, np.float32), np.zeros(1000, np.float32), 0.9, 0.999)
    em, ev, eb = oo.encode(m1, v1, *oo.dither(1000, 3, 0, 1, first=1 << 32))
    got = cm[-1000:].cpu().numpy()
    assert np.array_equal(got & 127, em & 127) and np.array_equal(cv[-1000:].cpu().numpy(), ev) and np.array_equal(b[-4:].cpu().numpy(), eb)
    wp, _, _, ep, _, _ = oo.adamw(np.full(1000, 0.5), h, np.zeros(1000), np.zeros(1000), 1, 0.1, 0.9, 0.999, 1e-8, 0.0)
    assert (np.abs(f64(p[-1000:]) - wp) <= ep + HALF[torch.bfloat16] * (np.abs(wp) + ep)).all()
    assert not cm[:-1000].any() and bool((p[:1 << 20] == 0.5).all()) and bool((p[-2000:-1000] == 0.5).all())


# ------------------------------------------------------------------------------------------------ the optimizer class
def _model(seed, dtype=torch.float32):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Conv2d(3, 8, 3, padding=1), torch.nn.ReLU(), torch.nn.Conv2d(8, 5, 1), torch.nn.Flatten(),
                               torch.nn.Linear(5 * 36, 7)).to(DEV).to(dtype)


def _train(model, opt, first, count, channels_last=False):
    for t in range(first, first + count):
        torch.manual_seed(100 + t)
        x = torch.randn(4, 3, 6, 6, device=DEV)
        opt.zero_grad(set_to_none=True)
        model(x).square().mean().backward()
        opt.step()


def test_class_matches_torch_adamw_and_exchanges_checkpoints():
    """20 steps beside torch.optim.AdamW on the same gradients: a step's update is off by 16 * 2^-24 of lr-sized updates (|m / sqrt(v)|
    below 1 / sqrt(1 - beta2) = 32 at most), its parameter by 4 roundings, on either side: 20 * 2 * (16 * 32 * lr + 4 |p|) * 2^-24."""
    from dtt.optim import GroupedAdamW
    a, b = _model(0), _model(0)
    groups = lambda m: [{"params": [p], "lr": 1e-3 * (2 if p.dim() == 1 else 1), "weight_decay": 0.0 if p.dim() == 1 else 0.1} for p in m.parameters()]
    oa, ob = torch.optim.AdamW(groups(a)), GroupedAdamW(groups(b))
    def both(first, count, oa, ob):
        for t in range(first, first + count):
            torch.manual_seed(t)
            for p, q in zip(a.parameters(), b.parameters()):
                p.grad = torch.randn_like(p) * 0.1
                q.grad = p.grad.clone()
            oa.step(); ob.step()
        for p, q in zip(a.parameters(), b.parameters()):
            assert ((p - q).abs() <= 40 * (16 * 32 * 2e-3 + 4 * p.abs()) * oo.U).all()
    both(0, 10, oa, ob)
    sa, sb = oa.state_dict(), ob.state_dict()
    assert [g["params"] for g in sa["param_groups"]] == [g["params"] for g in sb["param_groups"]]
    assert set(sa["state"]) == set(sb["state"]) and set(sa["state"][0]) == set(sb["state"][0])
    oa2, ob2 = torch.optim.AdamW(groups(a)), GroupedAdamW(groups(b))
    oa2.load_state_dict(copy.deepcopy(sb))      # either way
    ob2.load_state_dict(copy.deepcopy(sa))
    both(10, 10, oa2, ob2)
    assert float(ob2.state[next(b.parameters())]["step"]) == 20


def test_a_rate_in_device_memory_survives_a_checkpoint(tmp_path):
    from dtt.optim import GroupedAdamW
    w = torch.nn.Parameter(torch.ones(50, device=DEV))
    opt = GroupedAdamW([w], lr=torch.full((), 0.25, device=DEV), weight_decay=0.0)
    w.grad = torch.ones_like(w)
    opt.step()
    torch.save(opt.state_dict(), tmp_path / "o.pth")
    v = torch.nn.Parameter(w.detach().clone())
    again = GroupedAdamW([v], lr=0.5, weight_decay=0.0)
    again.load_state_dict(torch.load(tmp_path / "o.pth", map_location="cpu"))
    v.grad = torch.ones_like(v)
    opt.step(); again.step()
    assert again.param_groups[0]["lr"].device == v.device and torch.equal(v, w)


@pytest.mark.parametrize("bits", [32, 8])
def test_one_norm_over_groups_of_different_betas_and_types(bits):
    """Two (betas, eps) and two element types in one optimizer with a limit: one norm over all gradients; the same update as the
    operators called with that norm."""
    from dtt.optim import GroupedAdamW, adamw8_, adamw_, blocks_of, grad_norm
    torch.manual_seed(8)
    shapes = [((70, 9), torch.float32), ((300,), torch.bfloat16), ((5, 5), torch.float32), ((1000,), torch.bfloat16)]
    ps = [torch.nn.Parameter(torch.randn(*s, device=DEV).to(t)) for s, t in shapes]
    for p in ps:
        p.grad = torch.randn_like(p)
    ps[0].grad = torch.full((1, 1), 0.25, device=DEV).expand(70, 9)          # a broadcast gradient
    betas = [(0.9, 0.999), (0.9, 0.999), (0.8, 0.9), (0.8, 0.9)]
    qs = [p.detach().clone() for p in ps]
    opt = GroupedAdamW([{"params": [p], "betas": b} for p, b in zip(ps, betas)], lr=1e-2, weight_decay=0.1, state_bits=bits, max_norm=0.5,
                       skip_nonfinite=True, seed=11)
    opt.step()
    gs = [p.grad.contiguous() for p in ps]
    norm = grad_norm(gs)
    assert torch.equal(opt.grad_norm, norm) and abs(float(norm) - math.sqrt(sum(float(g.double().square().sum()) for g in gs))) <= float(norm) * 2.0 ** -23
    clip = torch.stack([norm, (0.5 / (norm.double() + 1e-6)).float()])
    for first in (0, 2):
        at = [first, first + 1]
        s = [torch.zeros((), device=DEV) for _ in at]
        common = dict(lr=1e-2, betas=betas[first], weight_decay=0.1, clip=clip, skip_nonfinite=True)
        if bits == 32:
            out = adamw_([qs[i] for i in at], [gs[i] for i in at], *[[torch.zeros_like(qs[i], dtype=torch.float32) for i in at] for _ in range(2)], s, **common)
        else:
            out = adamw8_([qs[i] for i in at], [gs[i] for i in at], *[[torch.zeros_like(qs[i], dtype=torch.uint8) for i in at] for _ in range(2)],
                          [torch.zeros(blocks_of(qs[i].numel()), 2, dtype=torch.int16, device=DEV) for i in at], s, seed=11, ids=at, **common)
        assert torch.equal(out, norm)
    # the factor of the operators' call was rounded from the rounded norm: a last place of the clipped gradient, which the first step of
    # Adam (g / |g|) does not see beyond 32 U of its size, and half a step of the type
    for p, q in zip(ps, qs):
        assert ((p.detach().float() - q.float()).abs() <= 1e-2 * 64 * oo.U + q.float().abs() * (2 * HALF[p.dtype])).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_resumed_run_equals_the_uninterrupted_one(bits, tmp_path):
    from dtt.optim import GroupedAdamW
    make = lambda m: GroupedAdamW(m.parameters(), lr=1e-2, state_bits=bits, max_norm=0.1, seed=4)
    a = _model(1)
    oa = make(a)
    _train(a, oa, 0, 3)
    torch.save({"m": a.state_dict(), "o": oa.state_dict()}, tmp_path / "c.pth")
    _train(a, oa, 3, 3)
    b = _model(2)
    ob = make(b)
    ck = torch.load(tmp_path / "c.pth", map_location="cpu")
    b.load_state_dict(ck["m"])
    ob.load_state_dict(ck["o"])
    _train(b, ob, 3, 3)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    c = copy.deepcopy(ob)
    assert c.state_bits == bits and c.max_norm == 0.1 and c.seed == 4


def test_checkpoints_cross_between_8_and_32_bits_and_16_bit_parameters():
    from dtt.optim import GroupedAdamW
    a = _model(3)
    o8 = GroupedAdamW(a.parameters(), lr=1e-2, state_bits=8)
    _train(a, o8, 0, 4)
    assert set(next(iter(o8.state.values()))) == {"step", "exp_avg_code", "exp_avg_sq_code", "block_base"}
    o32 = GroupedAdamW(a.parameters(), lr=1e-2)
    o32.load_state_dict(o8.state_dict())
    for p in a.parameters():
        m, v = o8.moments(p)
        assert torch.equal(o32.state[p]["exp_avg"], m) and torch.equal(o32.state[p]["exp_avg_sq"], v) and float(v.max()) > 0
    back = GroupedAdamW(a.parameters(), lr=1e-2, state_bits=8)
    back.load_state_dict(o32.state_dict())      # values on the grid come back unchanged
    for p in a.parameters():
        assert all(torch.equal(x, y) for x, y in zip(back.moments(p), o8.moments(p)))
        assert float(back.state[p]["step"]) == 4
    _train(a, back, 4, 1)
    h = _model(4, torch.bfloat16)
    oh = GroupedAdamW(h.parameters(), lr=1e-2)
    for p in h.parameters():
        p.grad = torch.randn_like(p)
    oh.step()
    o2 = GroupedAdamW(h.parameters(), lr=1e-2)
    o2.load_state_dict(oh.state_dict())         # float32 moments of 16-bit parameters stay float32
    assert all(o2.state[p]["exp_avg"].dtype == torch.float32 and torch.equal(o2.state[p]["exp_avg"], oh.state[p]["exp_avg"]) for p in h.parameters())


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_change_their_memory_order(bits):
    """Filters moved to channels-last memory after the state was made (what a resumed run of the trainer does): the moments follow."""
    from dtt.optim import GroupedAdamW
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(16, 8, 3, 3, device=DEV))
    opt = GroupedAdamW([p], lr=1e-2, state_bits=bits, weight_decay=0.0)
    p.grad = torch.randn_like(p)
    opt.step()
    m0, v0 = opt.moments(p)
    p.data = p.data.contiguous(memory_format=torch.channels_last)
    p.grad = torch.zeros_like(p)
    before = p.detach().clone()
    opt.step()
    m1, v1 = opt.moments(p)
    assert m1.stride() == p.stride()
    if bits == 32:
        assert torch.allclose(m1, 0.9 * m0, rtol=1e-6, atol=0) and torch.allclose(v1, 0.999 * v0, rtol=1e-6, atol=0)
    else:   # one relayout (to the nearest, blocks of other elements) and one dithered step, each within a level
        assert ((m1 - 0.9 * m0).abs() <= 0.9 * m0.abs() / 8 + m0.abs().max() * 2.0 ** -15).all()
    step = (p.detach() - before) * -1e2
    assert torch.sign(step)[m1.abs() > 1e-4].eq(torch.sign(m1)[m1.abs() > 1e-4]).all()


def test_version_counters_and_autograd_see_the_update():
    from dtt.optim import GroupedAdamW
    w = torch.nn.Parameter(torch.randn(10, device=DEV))
    x = torch.randn(10, device=DEV)
    opt = GroupedAdamW([w], lr=0.1)
    loss = (w * w * x).sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_trainer_runs_and_resumes_with_the_operators(tmp_path):
    """trainval_net.py --o adamw8 / adamw / sgd with --clip_grad, and a resumed run from the 8-bit checkpoint with 32-bit moments."""
    import os
    import trainval_net
    save = str(tmp_path / "models")
    base = ["--dataset", "synthetic", "--net", "res50", "--bs", "1", "--cag", "--iters_per_epoch", "2", "--disp_interval", "1", "--save_dir", save,
            "--height", "224", "--width", "320", "--lr", "1e-5", "--clip_grad", "5"]
    path = os.path.join(save, "res50", "synthetic", "rfcn_detect_track_1_%d_1.pth")
    trainval_net.main(base + ["--epochs", "2", "--o", "adamw8"])
    ck = torch.load(path % 1, map_location="cpu")
    st = ck["optimizer"]["state"]
    assert all(s["exp_avg_code"].dtype == torch.uint8 and float(s["step"]) == 2 for s in st.values()) and len(st) > 50
    assert all(torch.isfinite(x).all() for x in ck["model"].values() if x.is_floating_point())
    trainval_net.main(base + ["--epochs", "3", "--o", "adamw", "--r", "True", "--checkepoch", "1", "--checkpoint", "1"])
    ck = torch.load(path % 2, map_location="cpu")
    assert all(s["exp_avg"].dtype == torch.float32 and float(s["step"]) == 4 for s in ck["optimizer"]["state"].values())
    trainval_net.main(base + ["--epochs", "2", "--o", "sgd", "--s", "2"])
