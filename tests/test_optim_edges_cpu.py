"""The optimizer operators where calls meet, without a GPU: what the library refuses about buffers that meet, checkpoints that are refused,
learning rates that groups share."""
import copy
import ctypes

import pytest
import torch


def test_library_refuses_results_rates_and_workspaces_that_meet_a_tensor():
    """Norm and factor, the workspace and learning rates in device memory are buffers of the call like any other (status 0, nothing launched)."""
    from dtt import _lib
    L = _lib.lib()
    buf = (ctypes.c_double * 4096)()
    base = ctypes.addressof(buf)
    P = lambda *a: (ctypes.c_void_p * len(a))(*a)
    N = lambda *a: (ctypes.c_long * len(a))(*a)
    D = lambda *a: (ctypes.c_double * len(a))(*a)
    I = lambda *a: (ctypes.c_int * len(a))(*a)
    ws = base + 16384
    for call in (L.dtt_grad_norm, L.dtt_grad_clip):
        norm = lambda g=base, out=base + 1024, w=ws: call(1, P(g), N(8), I(0), 1.0, out, w, 4096, None)
        for kw, why in ((dict(out=base), "share memory"), (dict(out=base + 28), "share memory"), (dict(w=base + 24), "share memory"),
                        (dict(out=ws), "share memory"), (dict(out=base + 1026), "unaligned")):
            assert norm(**kw) == 0 and why in _lib.last_error(), (kw, _lib.last_error())
    p, g, m, v, b, s = (base + k for k in (0, 128, 256, 384, 512, 600))

    def step(bits, rate=None, clip=None, w=ws, limit=-1.0):
        args = [1, 0, P(p), P(g), P(m), P(v)] + ([P(b)] if bits == 8 else []) + [N(16), P(s), D(1e-3), None if rate is None else P(rate), D(0.0)]
        tail = [0.9, 0.999, 1e-8, limit, clip, 0, w, 4096, None]
        return L.dtt_adamw8_step(*args, None, 0, *tail) if bits == 8 else L.dtt_adamw_step(*args, *tail)
    for bits in (32, 8):
        for kw, why in ((dict(rate=p), "share memory"), (dict(rate=m), "share memory"), (dict(rate=s), "share memory"), (dict(rate=s + 1), "unaligned"),
                        (dict(clip=p + 4), "share memory"), (dict(clip=s), "share memory"), (dict(clip=g, limit=1.0), "share memory"),
                        (dict(clip=base + 1024, rate=base + 1028, limit=1.0), "share memory"), (dict(clip=ws + 8, limit=1.0), "share memory"),
                        (dict(clip=base + 1026, limit=1.0), "unaligned"), (dict(w=m), "share memory"), (dict(w=base - 16), "share memory"),
                        (dict(rate=ws), "share memory")):
            assert step(bits, **kw) == 0 and why in _lib.last_error(), (bits, kw, _lib.last_error())


def test_several_calls_are_checked_as_one_step():
    """dtt_adamw_check: the tensors of all calls of a step, of whatever types, before the first is launched."""
    from dtt import _lib
    L = _lib.lib()
    buf = (ctypes.c_double * 4096)()
    base = ctypes.addressof(buf)
    P = lambda *a: (ctypes.c_void_p * len(a))(*a)
    N = lambda *a: (ctypes.c_long * len(a))(*a)
    D = lambda *a: (ctypes.c_double * len(a))(*a)
    I = lambda *a: (ctypes.c_int * len(a))(*a)

    def together(dtypes=(0, 1), p=(base, base + 64), g=(base + 128, base + 192), m=(base + 256, base + 320), v=(base + 384, base + 448), b=None,
                 n=(16, 16), s=(base + 512, base + 516), lr=(1e-3, 1e-3), rate=None, wd=(0.0, 0.0), clip=None):
        return L.dtt_adamw_check(2, I(*dtypes), P(*p), P(*g), P(*m), P(*v), None if b is None else P(*b), N(*n), P(*s), D(*lr),
                                 None if rate is None else P(*rate), D(*wd), clip)
    bases = (base + 600, base + 604)
    assert together() == 1 and together(b=bases) == 1 and together(n=(0, 16), p=(None, base + 64), clip=base + 1024, rate=(base + 1100, None)) == 1
    assert together(m=(base + 256, base + 280), b=bases) == 1      # 16 codes are 16 bytes; 16 values are 64
    for kw, why in ((dict(s=(base + 512, base + 512)), "share memory"), (dict(m=(base + 256, base + 280)), "share memory"),
                    (dict(p=(base, base + 60)), "share memory"), (dict(g=(base + 128, base + 60)), "share memory"),
                    (dict(b=(base + 600, base + 600)), "share memory"), (dict(b=(base + 600, base + 606)), "unaligned"), (dict(b=(base + 600, None)), "null"),
                    (dict(v=(base + 384, base + 450)), "unaligned"), (dict(p=(base, base + 65)), "unaligned"), (dict(dtypes=(0, 3)), "element type"),
                    (dict(n=(16, -1)), "element count"), (dict(lr=(1e-3, float("nan"))), "learning rate"), (dict(wd=(0.0, -1.0)), "weight decay"),
                    (dict(rate=(None, base + 68)), "share memory"), (dict(clip=base + 512), "share memory"), (dict(s=(base + 512, None)), "step counter")):
        assert together(**kw) == 0 and why in _lib.last_error(), (kw, _lib.last_error())
    assert L.dtt_adamw_check(0, None, *[None] * 11) == 1


def _adamw_state(shape=(4, 3), step=3.0):
    torch.manual_seed(0)
    return {"step": torch.tensor(step), "exp_avg": torch.randn(shape), "exp_avg_sq": torch.rand(shape)}


def _optimizer(bits=32):
    """Two parameters of an optimizer that holds a state (read from a checkpoint: 32-bit moments need no GPU)."""
    from dtt.optim import GroupedAdamW
    ps = [torch.nn.Parameter(torch.ones(4, 3)) for _ in range(2)]
    opt = GroupedAdamW([{"params": [ps[0]], "lr": 0.5}, {"params": [ps[1]], "betas": (0.8, 0.9)}], lr=0.25, state_bits=bits)
    sd = opt.state_dict()
    sd["state"] = {0: _adamw_state(), 1: _adamw_state(step=7.0)}
    opt.load_state_dict(sd)
    return opt, ps


def _refused_load(opt, ps, checkpoint, match):
    groups = copy.deepcopy([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups])
    state = [{k: x.clone() for k, x in opt.state[p].items()} for p in ps]
    with pytest.raises(ValueError, match=match):
        opt.load_state_dict(checkpoint)
    assert [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups] == groups
    assert [g["params"][0] is p for g, p in zip(opt.param_groups, ps)] == [True, True]
    assert len(opt.state) == 2
    for p, st in zip(ps, state):
        assert set(opt.state[p]) == set(st) and all(torch.equal(opt.state[p][k], x) for k, x in st.items())


def test_a_refused_checkpoint_leaves_the_optimizer_as_it_was():
    for bits in (32, 8):
        opt, ps = _optimizer(bits)
        sgd = torch.optim.SGD([{"params": [p]} for p in ps], lr=0.1, momentum=0.9)
        for p in ps:
            p.grad = torch.ones_like(p)
        sgd.step()
        _refused_load(opt, ps, sgd.state_dict(), "not a state of AdamW")
        plain = torch.optim.SGD([{"params": [p]} for p in ps], lr=0.1).state_dict()        # its groups have no betas, and there is no state to tell
        _refused_load(opt, ps, plain, "betas")
        good = lambda: copy.deepcopy(opt.state_dict())
        for change, why in ((lambda d: d["param_groups"][1].update(amsgrad=True), "amsgrad"),
                            (lambda d: d["state"][1].pop("step"), "not a state of AdamW"),
                            (lambda d: d["state"][1].pop("exp_avg_sq" if bits == 32 else "exp_avg_sq_code"), "not a state of AdamW"),
                            (lambda d: d["param_groups"].pop(), "parameter group"),
                            (lambda d: d["param_groups"][1]["params"].append(2), "parameter group"),
                            (lambda d: d["state"][1].update(step=torch.zeros(2)), "step")):
            d = good()
            change(d)
            _refused_load(opt, ps, d, why)
        opt.load_state_dict(good())


def test_moments_of_another_shape_do_not_load():
    """A state of another shape would be broadcast into the parameter's, or refused at the next step only."""
    from dtt.optim import pack_moments
    for bits in (32, 8):
        opt, ps = _optimizer(bits)
        with32 = lambda: {"param_groups": copy.deepcopy(opt.state_dict()["param_groups"]), "state": {0: _adamw_state(), 1: _adamw_state()}}

        def with8():
            d = with32()
            for i in d["state"]:
                st = d["state"][i]
                st["exp_avg_code"], st["exp_avg_sq_code"], st["block_base"] = pack_moments(st.pop("exp_avg"), st.pop("exp_avg_sq"))
            return d
        for shape in ((3,), (1,), (), (4, 1), (3, 4), (12,), (4, 4)):
            for k in ("exp_avg", "exp_avg_sq"):
                d = with32()
                d["state"][1][k] = torch.ones(shape)
                _refused_load(opt, ps, d, "shape")
        if bits == 8:
            for change in (lambda st: st.update(exp_avg_code=st["exp_avg_code"][0]), lambda st: st.update(exp_avg_sq_code=st["exp_avg_sq_code"].view(3, 4)),
                           lambda st: st.update(exp_avg_code=st["exp_avg_code"].t().contiguous().t()),            # the two lie in other orders
                           lambda st: st.update(exp_avg_code=torch.zeros(4, 6, dtype=torch.uint8)[:, ::2], exp_avg_sq_code=torch.zeros(4, 6, dtype=torch.uint8)[:, ::2]),
                           lambda st: st.update(exp_avg_code=st["exp_avg_code"].int()), lambda st: st.update(block_base=torch.zeros(2, 2, dtype=torch.int16)),
                           lambda st: st.update(block_base=torch.zeros(1, 2, dtype=torch.int32))):
                d = with8()
                change(d["state"][1])
                _refused_load(opt, ps, d, "shape|int16|uint8")
            opt.load_state_dict(with8())
        opt.load_state_dict(with32())
    opt, ps = _optimizer()
    d = opt.state_dict()
    d["state"] = {0: _adamw_state(), 1: _adamw_state()}
    d["state"][0]["exp_avg_sq"] = d["state"][0]["exp_avg_sq"].t().contiguous().t()         # the same values in another memory order do
    want = d["state"][0]["exp_avg_sq"].clone()
    opt.load_state_dict(d)
    assert opt.state[ps[0]]["exp_avg_sq"].is_contiguous() and torch.equal(opt.state[ps[0]]["exp_avg_sq"], want)


def test_groups_that_share_a_learning_rate_share_it_after_a_checkpoint():
    """One rate tensor for all groups (what a schedule under a graph writes to) stays one, also where it is converted."""
    from dtt.optim import GroupedAdamW
    for dtype in (torch.float32, torch.float64):
        ps = [torch.nn.Parameter(torch.ones(3)) for _ in range(4)]
        rate, other = torch.tensor(0.25, dtype=dtype), torch.tensor(0.5, dtype=dtype)
        groups = lambda: [{"params": [p], "lr": r} for p, r in zip(ps, (rate, rate, other, rate))]
        saved = torch.optim.AdamW(groups(), lr=0.1, foreach=False, capturable=True).state_dict()
        opt = GroupedAdamW([{"params": [p]} for p in ps], lr=0.125)
        opt.load_state_dict(saved)
        lr = [g["lr"] for g in opt.param_groups]
        assert all(x.dtype == torch.float32 for x in lr) and [float(x) for x in lr] == [0.25, 0.25, 0.5, 0.25]
        assert lr[0] is lr[1] and lr[0] is lr[3] and lr[2] is not lr[0]
        lr[0].fill_(1.0)
        assert [float(g["lr"]) for g in opt.param_groups] == [1.0, 1.0, 0.5, 1.0] and float(rate) == 0.25


def test_a_step_without_gradients_has_no_norm():
    from dtt.optim import GroupedAdamW
    p = torch.nn.Parameter(torch.ones(3))
    opt = GroupedAdamW([p], max_norm=1.0)
    opt.grad_norm = torch.ones(())                  # of the step before
    opt.step()
    assert opt.grad_norm is None


def test_a_negated_view_is_not_its_memory():
    """The imaginary part of a conjugate: float32, strided, and the negative of what lies in memory."""
    from dtt import optim as O
    z = torch.complex(torch.ones(1), torch.full((1,), 2.0)).conj()
    g = z.imag
    assert g.is_neg() and float(g) == -2.0
    p, m, v, s = torch.zeros(1), torch.zeros(1), torch.zeros(1), torch.zeros(())
    for call in (lambda: O.grad_norm([g]), lambda: O.clip_grads_([g], 1.0), lambda: O.adamw_([g], [p], [m], [v], [s], lr=0.1),
                 lambda: O.adamw_([p], [m], [g], [v], [s], lr=0.1), lambda: O.adamw_([p], [m], [v], [s], [g.view(())], lr=0.1),
                 lambda: O.adamw_([p], [m], [v], [torch.zeros(1)], [s], lr=g)):
        with pytest.raises((TypeError, RuntimeError), match="resolve_neg|GPU only"):
            call()
    assert O._tensorlist().describe([g])[4] == -1
    with pytest.raises(TypeError, match="resolve_neg"):
        O.clip_grads_([g], 1.0)
