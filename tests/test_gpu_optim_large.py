"""The kernel forms of the optimizer operators (dtt/optim.py) that only large tensors take -- four blocks of 8-bit moments to a wave, codes that
pass the caches by, offsets beyond 32 bits -- element by element.

Tolerances are the oracle's counted rounding errors, as in test_gpu_optim.py; codes and bases are compared for equality."""
import math

import numpy as np
import pytest
import torch

from oracle import optim_oracle as oo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def f64(t):
    return t.detach().double().cpu().numpy()


def spread(n, seed, lo=-12.0, hi=2.0):
    rs = np.random.RandomState(seed)
    return (np.exp(rs.uniform(lo, hi, n)) * np.sign(rs.randn(n)) * (rs.rand(n) > 0.1)).astype(np.float32)


# ------------------------------------------------------------------------------------------------ forms of large tensors
@pytest.mark.parametrize("first", [0, 1], ids=["aligned", "odd"])
@pytest.mark.parametrize("dtype", list(HALF), ids=str)
def test_large_8_bit_steps_and_unpacking_match_the_definition(dtype, first):
    """5 M elements: every wave holds four blocks.  Full waves and the end of the tensor, blocks with infinities and NaN among them."""
    from dtt.optim import adamw8_, blocks_of, unpack_moments_
    n = 5_000_777
    assert n > 4 * 256 * 4096
    place = lambda x, dt: torch.zeros(n + 9, dtype=dt, device=DEV)[first:first + n].copy_(torch.from_numpy(x))
    v0 = np.square(spread(n, 3))
    m0 = spread(n, 2) * (v0 > 0)
    odd = [5, 3000, 1_000_003, 4_999_000, n - 2]
    m0[odd[0]], v0[odd[0]], v0[odd[1]], m0[odd[2]] = np.nan, np.nan, np.inf, -np.inf
    cm, cv, b = oo.encode(m0, v0, 1 << 19, 1 << 19)
    p, g = place(spread(n, 4, -5, 0), dtype), place(spread(n, 1), dtype)
    g[odd[3]], g[odd[4]], g[odd[2] + 300] = math.inf, math.nan, -math.inf
    cm, cv, b = place(cm, torch.uint8), place(cv, torch.uint8), torch.from_numpy(b).to(DEV)
    assert b.shape == (blocks_of(n), 2)
    s = torch.full((), 41.0, device=DEV)
    for t in (42, 43):
        p0, g0 = f64(p), g.float().cpu().numpy()
        m0, v0 = oo.decode(cm.cpu().numpy(), cv.cpu().numpy(), b.cpu().numpy())
        adamw8_([p], [g], [cm], [cv], [b], [s], lr=1e-2, weight_decay=0.1, seed=77, ids=[5])
        m1, v1 = oo.moments_f32(g0, m0, v0, 0.9, 0.999)
        em, ev, eb = oo.encode(m1, v1, *oo.dither(n, 77, 5, t))
        got = cm.cpu().numpy()
        assert np.array_equal(b.cpu().numpy(), eb) and np.array_equal(cv.cpu().numpy(), ev) and np.array_equal(got & 127, em & 127)
        signed = (em & 127 != 0) & ~np.isnan(m1)
        assert np.array_equal(got[signed], em[signed])
        with np.errstate(invalid="ignore"):
            wp, _, _, ep, _, _ = oo.adamw(p0, g0, m0, v0, t, 1e-2, 0.9, 0.999, 1e-8, 0.1)
        ep = ep + (0 if dtype == torch.float32 else HALF[dtype] * (np.abs(wp) + ep) + SMALLEST[dtype])
        gp, whole = f64(p), ~np.isnan(wp)
        assert whole.sum() >= n - 6 and np.isnan(gp[~whole]).all() and (np.abs(gp - wp)[whole] <= ep[whole]).all()
    wm, wv = oo.decode(cm.cpu().numpy(), cv.cpu().numpy(), b.cpu().numpy())
    for out in (torch.float32, torch.bfloat16):
        fm, fv = (torch.full((n + 9,), 7.0, dtype=out, device=DEV) for _ in range(2))
        unpack_moments_([cm], [cv], [b], [fm[first:first + n]], [fv[first:first + n]])
        for f, w in ((fm, wm), (fv, wv)):
            assert np.array_equal(f[first:first + n].float().cpu().numpy(), w, equal_nan=True)
            assert bool((f[:first] == 7.0).all()) and bool((f[first + n:] == 7.0).all())


FAR = (1 << 32) + 5000                                              # elements; windows that hold something, at whole blocks
WINDOWS = [(1 << 20, 8192), ((1 << 31) - 4096, 8192), ((1 << 32) - 8192, 8192 + 5000)]


def _outside(t, zero=0):
    """Nothing but `zero` outside the windows."""
    at = 0
    for a, k in WINDOWS:
        if not bool((t[at:a] == zero).all()):
            return False
        at = a + k
    return at == FAR


def test_8_bit_steps_beyond_32_bits_in_full_waves():
    from dtt.optim import adamw8_, blocks_of, unpack_moments_
    p = torch.full((FAR,), 0.5, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(FAR, dtype=torch.bfloat16, device=DEV)
    cm, cv = (torch.zeros(FAR, dtype=torch.uint8, device=DEV) for _ in range(2))
    b = torch.zeros(blocks_of(FAR), 2, dtype=torch.int16, device=DEV)
    start = []
    for i, (a, k) in enumerate(WINDOWS):
        v = np.square(spread(k, 20 + i))
        m = spread(k, 30 + i) * (v > 0)
        g[a:a + k] = torch.from_numpy(spread(k, 40 + i)).to(DEV)
        em, ev, eb = oo.encode(m, v, 1 << 19, 1 << 19)
        cm[a:a + k], cv[a:a + k] = torch.from_numpy(em).to(DEV), torch.from_numpy(ev).to(DEV)
        b[a // 256:a // 256 + len(eb)] = torch.from_numpy(eb).to(DEV)
        start.append((g[a:a + k].float().cpu().numpy(), *oo.decode(em, ev, eb)))
    adamw8_([p], [g], [cm], [cv], [b], [torch.full((), 6.0, device=DEV)], lr=0.1, weight_decay=0.0, seed=3)
    for (a, k), (h, m0, v0) in zip(WINDOWS, start):
        m1, v1 = oo.moments_f32(h, m0, v0, 0.9, 0.999)
        em, ev, eb = oo.encode(m1, v1, *oo.dither(k, 3, 0, 7, first=a))
        got, signed = cm[a:a + k].cpu().numpy(), em & 127 != 0
        assert np.array_equal(got & 127, em & 127) and np.array_equal(got[signed], em[signed]), a
        assert np.array_equal(cv[a:a + k].cpu().numpy(), ev) and np.array_equal(b[a // 256:a // 256 + len(eb)].cpu().numpy(), eb), a
        wp, _, _, ep, _, _ = oo.adamw(np.full(k, 0.5), h, m0, v0, 7, 0.1, 0.9, 0.999, 1e-8, 0.0)
        assert (np.abs(f64(p[a:a + k]) - wp) <= ep + HALF[torch.bfloat16] * (np.abs(wp) + ep)).all(), a
    assert _outside(cm) and _outside(cv) and _outside(p, 0.5)
    del g, p
    om, ov = (torch.full((FAR,), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    unpack_moments_([cm], [cv], [b], [om], [ov])
    for a, k in WINDOWS:
        wm, wv = oo.decode(cm[a:a + k].cpu().numpy(), cv[a:a + k].cpu().numpy(), b[a // 256:(a + k + 255) // 256].cpu().numpy())
        assert np.array_equal(om[a:a + k].float().cpu().numpy(), wm) and np.array_equal(ov[a:a + k].float().cpu().numpy(), wv), a
    assert _outside(om) and _outside(ov)


def test_32_bit_steps_and_scaling_beyond_32_bits():
    from dtt.optim import adamw_, clip_grads_
    p = torch.full((FAR,), 0.5, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(FAR, dtype=torch.bfloat16, device=DEV)
    m, v = (torch.zeros(FAR, device=DEV) for _ in range(2))
    for i, (a, k) in enumerate(WINDOWS):
        x = np.square(spread(k, 20 + i))
        v[a:a + k] = torch.from_numpy(x).to(DEV)
        m[a:a + k] = torch.from_numpy(spread(k, 30 + i) * (x > 0)).to(DEV)
        g[a:a + k] = torch.from_numpy(spread(k, 40 + i)).to(DEV)
    old = [[f64(x[a:a + k]) for x in (p, g, m, v)] for a, k in WINDOWS]
    norm, c = oo.norm_and_factor([o[1] for o in old], 3.0)
    assert c < 1
    got = adamw_([p], [g], [m], [v], [torch.full((), 6.0, device=DEV)], lr=0.1, weight_decay=0.0, max_norm=3.0)
    assert abs(float(got) - norm) <= norm * 2.0 ** -23
    for (a, k), o in zip(WINDOWS, old):
        wp, wm, wv, ep, em, ev = oo.adamw(*o, 7, 0.1, 0.9, 0.999, 1e-8, 0.0, c)
        assert (np.abs(f64(m[a:a + k]) - wm) <= em).all() and (np.abs(f64(v[a:a + k]) - wv) <= ev).all(), a
        assert (np.abs(f64(p[a:a + k]) - wp) <= ep + HALF[torch.bfloat16] * (np.abs(wp) + ep)).all(), a
    assert _outside(m) and _outside(v) and _outside(p, 0.5)
    assert abs(float(clip_grads_([g], 3.0)) - norm) <= norm * 2.0 ** -23
    for (a, k), o in zip(WINDOWS, old):
        want = o[1] * c
        tol = np.abs(want) * (2 * oo.U + HALF[torch.bfloat16]) + SMALLEST[torch.bfloat16]
        assert (np.abs(f64(g[a:a + k]) - want) <= tol).all(), a
    assert _outside(g)
