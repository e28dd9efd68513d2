"""Plain numpy restatement of the optimizer operators (dtt/optim.py): 64-bit formulas with error bounds, and the 8-bit moments
in fp32 arithmetic in the operators' order (test infrastructure only)."""
import numpy as np

U = 2.0 ** -24          # half a step of fp32, relative
BLOCK = 256


def norm_and_factor(grads, max_norm):
    norm = float(np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads)))
    return norm, min(1.0, max_norm / (norm + 1e-6))


def adamw(p, g, m, v, t, lr, beta1, beta2, eps, decay, c=1.0):
    """64-bit step t of one tensor and bounds of the fp32 kernel's error before p's rounding to its type:
    (p, m, v, err_p, err_m, err_v).  Counted in units U: the constants and the factors are rounded once (1 each), a product or a
    sum 1; sqrt 2, reciprocal 2 (one step each way), so the quotient's denominator is off by 4 (half of v's 8) + 2 + 1 + 1 + 1 + 1 = 10
    and the update by 10 + 2 + 1 (times m) + 2 (times size) = 15, rounded up to 16."""
    p, g, m, v = (np.asarray(x, dtype=np.float64) for x in (p, g, m, v))
    g = g * c
    m1 = beta1 * m + (1 - beta1) * g
    err_m = 6 * U * (np.abs(beta1 * m) + np.abs((1 - beta1) * g)) + 2.0 ** -147
    v1 = beta2 * v + (1 - beta2) * g * g
    err_v = 8 * U * v1 + 2.0 ** -147
    size = lr / (1 - beta1 ** t)
    den = np.sqrt(v1) / np.sqrt(1 - beta2 ** t) + eps
    upd = size * m1 / den
    p1 = p * (1 - lr * decay) - upd
    # (a v near the smallest fp32 has an absolute error: it moves the denominator by at most sqrt of it)
    tiny = np.minimum(1.0, np.sqrt(2.0 ** -147) / den)
    err_p = 3 * U * np.abs(p) + (16 * U + tiny) * np.abs(upd) + size / den * err_m + U * np.abs(p1)
    return p1, m1, v1, err_p, err_m, err_v


# ------------------------------------------------------------------------------------------------ 8-bit moments
def mix32(x):
    x = np.asarray(x, dtype=np.uint64) & np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x9E3779B9)) & np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x6A09E667)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def dither(n, seed, ident, t, first=0):
    """The rounding terms of elements first .. first + n - 1 of tensor `ident` at step t, for m and v, in [0, 2^20)."""
    key = mix32((seed + 0x9E3779B9 * (ident + 1)) & 0xFFFFFFFF)
    key = int(mix32((int(key) + t) & 0xFFFFFFFF))
    e = np.arange(first, first + n, dtype=np.uint64)
    r = (mix32((e >> np.uint64(3)) ^ np.uint64(key)) * (np.uint64(2) * (e & np.uint64(7)) + np.uint64(1))) & np.uint64(0xFFFFFFFF)
    return ((r >> np.uint64(16)) * np.uint64(16) + np.uint64(8)).astype(np.int64), ((r & np.uint64(0xFFFF)) * np.uint64(16) + np.uint64(8)).astype(np.int64)


def encode(m, v, um, uv):
    """fp32 moments of one tensor (flat) -> codes, codes, bases."""
    n = m.size
    nb = (n + BLOCK - 1) // BLOCK
    out, bases, odd_block = [], [], np.zeros(nb, dtype=bool)
    for x, u, top in ((m, um, 126), (v, uv, 254)):
        bits = (x.astype(np.float32).view(np.uint32) & np.uint32(0x7FFFFFFF)).astype(np.int64)
        level = (bits + u) >> 20
        odd = level >= 0x7F8
        base = np.zeros(nb, dtype=np.int64)
        for b in range(nb):
            s = slice(b * BLOCK, min(n, (b + 1) * BLOCK))
            fin = level[s][~odd[s]]
            base[b] = max((int(fin.max()) if fin.size else 0) - top, 0)
            odd_block[b] |= bool(odd[s].any())
        code = np.maximum(level - np.repeat(base, BLOCK)[:n], 0)
        if top == 254:
            code = np.maximum(code, (x > 0).astype(np.int64))
        code = np.where(odd, top + 1, code)
        if top == 126:
            code = code | ((x < 0).astype(np.int64) << 7)
        out.append(code.astype(np.uint8))
        bases.append(base)
    return out[0], out[1], np.stack([b | (odd_block.astype(np.int64) << 14) for b in bases], 1).astype(np.int16)


def decode(cm, cv, bases):
    n = cm.size
    out = []
    for code, k, top in ((cm, 0, 127), (cv, 1, 255)):
        b = np.repeat(bases[:, k].astype(np.int64), BLOCK)[:n]
        level = code.astype(np.int64) & top
        bits = np.where(level > 0, (level + (b & 0x3FFF)) << 20, 0).astype(np.uint32)
        x = bits.view(np.float32).copy()
        x[(level == top) & ((b >> 14) & 1 == 1)] = np.nan
        if top == 127:
            x = np.where(code > 127, -x, x)
        out.append(x)
    return out


def moments_f32(g, m, v, beta1, beta2):
    """New moments in fp32, every operation rounded, in the kernel's order."""
    f = np.float32
    with np.errstate(all="ignore"):
        m1 = m * f(beta1) + g * f(1 - beta1)
        v1 = v * f(beta2) + (g * g) * f(1 - beta2)
    return m1, v1
