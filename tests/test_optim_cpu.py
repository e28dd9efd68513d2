"""The optimizer operators without a GPU: the 8-bit grid, refusals, library-side argument checks."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import optim_oracle as oo


def test_every_level_packs_to_itself_and_decodes_to_four_bits():
    """Values on the grid are unchanged by nearest AND by dithered rounding, whatever the term: encode(decode(c)) = c."""
    from dtt.optim import pack_moments
    for base in (0, 900, 1700):
        lv = np.arange(0, 255, dtype=np.int64)
        v = np.where(lv > 0, (lv + base) << 20, 0).astype(np.uint32).view(np.float32)
        lm = np.concatenate([np.arange(0, 127), np.arange(126, -1, -1), [5]])
        m = np.where(lm > 0, (lm + base) << 20, 0).astype(np.uint32).view(np.float32)
        m[128:] *= -1
        for u in (8, 1 << 19, 16 * 65535 + 8):
            cm, cv, b = oo.encode(m, v, u, u)
            dm, dv = oo.decode(cm, cv, b)
            assert np.array_equal(dm, m) and np.array_equal(dv, v), (base, u)
        cm, cv, b = pack_moments(torch.from_numpy(m), torch.from_numpy(v))
        dm, dv = oo.decode(cm.numpy(), cv.numpy(), b.numpy())
        assert np.array_equal(dm, m) and np.array_equal(dv, v)
        assert torch.equal(torch.from_numpy(dm).bfloat16().float(), torch.from_numpy(dm))   # 16 bits hold a value exactly


def test_pack_moments_rounds_to_the_nearest_level_and_keeps_the_odd_values_apart():
    from dtt.optim import pack_moments
    rs = np.random.RandomState(0)
    for n in (1, 255, 256, 257, 1000):
        m = (rs.randn(n) * np.exp(rs.randn(n) * 2)).astype(np.float32)
        v = (np.exp(rs.randn(n) * 4) * (rs.rand(n) > 0.1)).astype(np.float32)
        if n > 300:
            m[3], m[260], v[5], v[6] = np.nan, np.inf, np.inf, 1e-44
        cm, cv, b = pack_moments(torch.from_numpy(m), torch.from_numpy(v))
        em, ev, eb = oo.encode(m, v, 1 << 19, 1 << 19)
        assert np.array_equal(cm.numpy(), em) and np.array_equal(cv.numpy(), ev) and np.array_equal(b.numpy(), eb)
        dm, dv = oo.decode(em, ev, eb)
        fin_m, fin_v = np.isfinite(m), np.isfinite(v)
        assert np.array_equal(np.isnan(dm), ~fin_m) and np.array_equal(np.isnan(dv), ~fin_v)
        # half a spacing is 1/16 of a value at most (mantissa 1.0), or all of what lies below the span
        floor = np.array([np.abs(m[i // 256 * 256:i // 256 * 256 + 256][fin_m[i // 256 * 256:i // 256 * 256 + 256]]).max() * 2.0 ** -15.6 for i in range(n)])
        assert (np.abs(dm - m)[fin_m] <= np.maximum(np.abs(m) / 16, floor)[fin_m]).all()
        assert (dv[fin_v] > 0).sum() == (v[fin_v] > 0).sum()   # nothing that is not zero became zero
    # another memory order than row-major: codes lie as the moments do
    m = torch.randn(3, 5, 7, 2).contiguous(memory_format=torch.channels_last)
    cm, cv, b = pack_moments(m, m.square())
    assert cm.stride() == m.stride()
    flat = m.permute(0, 2, 3, 1).reshape(-1)
    em, ev, eb = oo.encode(flat.numpy(), flat.square().numpy(), 1 << 19, 1 << 19)
    assert np.array_equal(cm.permute(0, 2, 3, 1).reshape(-1).numpy(), em) and np.array_equal(b.numpy(), eb)


def test_dither_is_uniform_for_every_place_of_a_group():
    """Over steps, each of the eight elements that share a hash sees uniform terms: mean 1/2 and variance 1/12 within five standard
    errors (n = 4096 steps: 5 / sqrt(12 n) = 0.0226, and 5 * sqrt(1/180 / n) = 0.0058)."""
    steps = 4096
    tm = np.empty((steps, 16))
    tv = np.empty((steps, 16))
    for t in range(steps):
        a, b = oo.dither(16, 77, 3, t + 1)
        tm[t], tv[t] = a / 2.0 ** 20, b / 2.0 ** 20
    for x in (tm, tv):
        assert (np.abs(x.mean(0) - 0.5) < 0.0226).all() and (np.abs(x.var(0) - 1 / 12) < 0.0058).all()
        assert x.min() >= 0 and x.max() < 1


def _lists(n=2, dtype=torch.float32, shape=(5, 3)):
    p = [torch.zeros(shape, dtype=dtype) for _ in range(n)]
    return (p, [torch.zeros_like(x) for x in p], [torch.zeros_like(x, dtype=torch.float32) for x in p],
            [torch.zeros_like(x, dtype=torch.float32) for x in p], [torch.zeros(()) for _ in p])


def test_refusals_before_any_gpu_work():
    from dtt import optim as O
    p, g, m, v, s = _lists()
    # everything right but the place: the GPU-only error
    for call in (lambda: O.adamw_(p, g, m, v, s, lr=1e-3), lambda: O.grad_norm(g), lambda: O.clip_grads_(g, 1.0)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(ValueError, match="differ in length"):
        O.adamw_(p, g[:1], m, v, s, lr=1e-3)
    with pytest.raises(ValueError, match="betas"):
        O.adamw_(p, g, m, v, s, lr=1e-3, betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="eps"):
        O.adamw_(p, g, m, v, s, lr=1e-3, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        O.adamw_(p, g, m, v, s, lr=1e-3, eps=float("nan"))
    with pytest.raises(ValueError, match="lr"):
        O.adamw_(p, g, m, v, s, lr=-1e-3)
    with pytest.raises(ValueError, match="values of lr"):
        O.adamw_(p, g, m, v, s, lr=[1e-3])
    with pytest.raises(ValueError, match="weight_decay"):
        O.adamw_(p, g, m, v, s, lr=1e-3, weight_decay=[0.0, -1.0])
    with pytest.raises(TypeError, match="learning rate"):
        O.adamw_(p, g, m, v, s, lr=torch.tensor(1e-3, dtype=torch.float64))
    with pytest.raises(ValueError, match="max_norm"):
        O.adamw_(p, g, m, v, s, lr=1e-3, max_norm=-1.0)
    with pytest.raises(ValueError, match="max_norm"):
        O.clip_grads_(g, float("nan"))
    with pytest.raises(TypeError, match="parameter's type"):
        O.adamw_(p, [x.bfloat16() for x in g], m, v, s, lr=1e-3)
    with pytest.raises(ValueError, match="parameter's shape"):
        O.adamw_(p, [x.t() for x in g], m, v, s, lr=1e-3)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        O.adamw_([x.double() for x in p], [x.double() for x in g], m, v, s, lr=1e-3)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        O.grad_norm([x.double() for x in g])
    with pytest.raises(TypeError, match="step counter"):
        O.adamw_(p, g, m, v, [x.long() for x in s], lr=1e-3)
    with pytest.raises(ValueError, match="dense"):
        O.adamw_([torch.zeros(10, 3)[::2]] * 2, g, m, v, s, lr=1e-3)
    with pytest.raises(TypeError):
        O.adamw_(p, [None, g[1]], m, v, s, lr=1e-3)
    with pytest.raises(ValueError, match="differ in length"):
        O.adamw8_([], [], [], [], [], [], lr=1e-3, ids=[1])
    with pytest.raises(ValueError, match="clip"):
        O.adamw_(p, g, m, v, s, lr=1e-3, clip=torch.zeros(3))
    with pytest.raises(ValueError, match="clip"):
        O.adamw_(p, g, m, v, s, lr=1e-3, max_norm=1.0, clip=torch.zeros(2))
    assert O.adamw_([], [], [], [], [], lr=1e-3, max_norm=1.0) is None
    assert float(O.clip_grads_([], 1.0)) == 0.0 and float(O.grad_norm([])) == 0.0 and float(O.clip_grad_norm_([], 1.0)) == 0.0
    w = torch.nn.Parameter(torch.zeros(3))
    for bad in (dict(state_bits=4), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(max_norm=-1.0)):
        with pytest.raises(ValueError):
            O.GroupedAdamW([w], **bad)
    opt = O.GroupedAdamW([w])
    opt.step()                                  # no gradient: nothing to do, no GPU needed
    w.grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match="GPU only"):
        opt.step()
    assert not opt.state                        # a refused step leaves no half-made state
    with pytest.raises(ValueError, match="amsgrad"):
        ref = torch.optim.AdamW([w], amsgrad=True)
        opt.load_state_dict(ref.state_dict())
    sgd = torch.optim.SGD([w], lr=0.1, momentum=0.9)
    sgd.step()
    with pytest.raises(ValueError, match="not a state of AdamW"):
        opt.load_state_dict(sgd.state_dict())


def test_library_refuses_bad_arguments_without_a_gpu():
    """The C entry points check pointers, counts, alignment, workspace and overlaps on the host: status 0 and an error string."""
    from dtt import _lib
    L = _lib.lib()
    buf = (ctypes.c_double * 4096)()
    base = ctypes.addressof(buf)
    P = lambda *a: (ctypes.c_void_p * len(a))(*a)
    N = lambda *a: (ctypes.c_long * len(a))(*a)
    D = lambda *a: (ctypes.c_double * len(a))(*a)
    I = lambda *a: (ctypes.c_int * len(a))(*a)
    ws = base + 16384
    norm = lambda g=P(base), n=N(8), t=I(0), limit=1.0, out=base + 1024, w=ws, wb=4096: L.dtt_grad_norm(1, g, n, t, limit, out, w, wb, None)
    for kw, why in ((dict(g=P(None)), "null"), (dict(g=P(base + 2)), "unaligned"), (dict(n=N(-1)), "element count"), (dict(t=I(3)), "element type"),
                    (dict(limit=-1.0), "negative"), (dict(limit=float("nan")), "negative"), (dict(wb=1), "workspace"), (dict(out=None), "null"),
                    (dict(n=N((1 << 33) + 1)), "element count"), (dict(g=None), "null")):
        assert norm(**kw) == 0 and why in _lib.last_error(), (kw, _lib.last_error())
    assert L.dtt_grad_clip(2, P(base, base + 16), N(8, 8), I(0, 0), 1.0, base + 1024, ws, 4096, None) == 0 and "share memory" in _lib.last_error()
    assert L.dtt_grad_clip(1, P(base), N(8), I(0), 1.0, None, ws, 4096, None) == 0 and "null" in _lib.last_error()
    assert L.dtt_grad_clip(1, P(base), N(8), I(0), -1.0, base + 1024, ws, 4096, None) == 0 and "negative" in _lib.last_error()
    assert L.dtt_grad_clip(1, P(base), N(8), I(0), 1.0, base + 1024, ws, 0, None) == 0 and "workspace" in _lib.last_error()

    def step(p=(base, base + 64), g=(base + 128, base + 192), m=(base + 256, base + 320), v=(base + 384, base + 448), s=(base + 512, base + 516),
             n=(16, 16), dtype=0, lr=(1e-3, 1e-3), wd=(0.0, 0.0), b1=0.9, b2=0.999, eps=1e-8, limit=-1.0, clip=None, skip=0, w=ws, wb=4096):
        return L.dtt_adamw_step(2, dtype, P(*p), P(*g), P(*m), P(*v), N(*n), P(*s), D(*lr), None, D(*wd), b1, b2, eps, limit, clip, skip, w, wb, None)
    for kw, why in ((dict(p=(base, base)), "share memory"), (dict(m=(base + 256, base + 260)), "share memory"), (dict(g=(base + 4, base + 192)), "share memory"),
                    (dict(s=(base + 512, base + 512)), "share memory"), (dict(s=(base + 512, None)), "step counter"), (dict(p=(base + 1, base + 64)), "unaligned"),
                    (dict(v=(base + 384, None)), "moment"), (dict(dtype=5), "element type"), (dict(b1=1.0), "betas"), (dict(b2=-0.1), "betas"),
                    (dict(b2=float("nan")), "betas"), (dict(eps=-1.0), "eps"), (dict(lr=(1e-3, -1.0)), "learning rate"), (dict(wd=(float("nan"), 0.0)), "weight decay"),
                    (dict(skip=1), "norm and factor"), (dict(limit=1.0), "norm and factor"), (dict(limit=float("nan")), "not a number"), (dict(wb=8), "workspace"), (dict(w=ws + 4), "workspace"), (dict(n=(16, -3)), "element count")):
        assert step(**kw) == 0 and why in _lib.last_error(), (kw, _lib.last_error())

    def step8(m=(base + 256,), v=(base + 320,), b=(base + 512,), n=(16,), p=(base,), g=(base + 128,), s=(base + 600,)):
        return L.dtt_adamw8_step(1, 0, P(*p), P(*g), P(*m), P(*v), P(*b), N(*n), P(*s), D(1e-3), None, D(0.0), None, 0, 0.9, 0.999, 1e-8, -1.0, None, 0, ws,
                                 4096, None)
    for kw, why in ((dict(m=(base + 256,), v=(base + 260,)), "share memory"), (dict(b=(base + 513,)), "unaligned"), (dict(b=(None,)), "null"),
                    (dict(b=(base + 256,)), "share memory"), (dict(m=(None,)), "null")):
        assert step8(**kw) == 0 and why in _lib.last_error(), (kw, _lib.last_error())
    assert L.dtt_adamw8_unpack(1, P(base), P(base + 64), P(base + 128), N(16), 2, P(base + 256), P(base + 512), None) == 0 and "fp16" in _lib.last_error()
    assert L.dtt_adamw8_unpack(1, P(base), P(base + 64), P(base + 128), N(16), 0, P(base + 256), P(base + 300), None) == 0 and "share memory" in _lib.last_error()
    assert L.dtt_adamw_workspace_bytes(2, N(4, 4)) >= 40 and L.dtt_grad_norm_workspace_bytes(0, None) > 0


def test_optimizer_choice_and_groups():
    """make_optimizer: the groups of every choice are the reference's (one per parameter, biases without decay)."""
    from dtt.config import cfg
    from dtt.dist import make_optimizer
    from dtt.optim import GroupedAdamW
    model = torch.nn.Sequential(torch.nn.Conv2d(3, 4, 1), torch.nn.Conv2d(4, 2, 1))
    for name, bits in (("adamw", 32), ("adamw8", 8)):
        opt = make_optimizer(model, cfg, lr=1e-4, optimizer=name, max_norm=5.0)
        assert isinstance(opt, GroupedAdamW) and opt.state_bits == bits and opt.max_norm == 5.0
        assert [len(g["params"]) for g in opt.param_groups] == [1, 1, 1, 1]
        assert [g["weight_decay"] for g in opt.param_groups] == [cfg.TRAIN.WEIGHT_DECAY, 0, cfg.TRAIN.WEIGHT_DECAY, 0]
        assert opt.param_groups[0]["lr"] == 1e-4
    assert isinstance(make_optimizer(model, cfg, optimizer="adam"), torch.optim.Adam)
    assert type(make_optimizer(model, cfg)).__name__ == "GroupedSGD"
