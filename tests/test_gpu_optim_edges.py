"""The optimizer operators (dtt/optim.py) where calls meet: lists of several types and groups of several betas as one step that is done or
refused as a whole, infinite limits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# ------------------------------------------------------------------------------------------------ refused as a whole
def _mixed(bits, types=(torch.float32, torch.bfloat16, torch.float32), n=300):
    """Lists of a step over several element types: [params, grads, m, v, (bases,) steps]."""
    from dtt.optim import blocks_of
    torch.manual_seed(1)
    p = [torch.randn(n, device=DEV).to(t) for t in types]
    g = [torch.randn_like(x) for x in p]
    steps = [torch.zeros((), device=DEV) for _ in p]
    if bits == 32:
        return [p, g, [torch.zeros_like(x, dtype=torch.float32) for x in p], [torch.zeros_like(x, dtype=torch.float32) for x in p], steps]
    return [p, g, [torch.zeros_like(x, dtype=torch.uint8) for x in p], [torch.zeros_like(x, dtype=torch.uint8) for x in p],
            [torch.zeros(blocks_of(n), 2, dtype=torch.int16, device=DEV) for _ in p], steps]


def _refused(lists, match, error=(ValueError, RuntimeError), **k):
    from dtt.optim import adamw8_, adamw_
    before = [[x.clone() for x in l] for l in lists]
    with pytest.raises(error, match=match):
        (adamw_ if len(lists) == 5 else adamw8_)(*lists, **dict(dict(lr=1e-2), **k))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for a, b in zip(lists, before) for x, y in zip(a, b)), "a refused step changed something"


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_over_several_types_is_refused_as_a_whole(bits):
    lists = _mixed(bits)
    lists[-1][1] = lists[-1][0]                                     # one counter for a float32 and a bfloat16 parameter
    _refused(lists, "share memory")
    lists = _mixed(bits)
    lists[2][1] = lists[2][0]                                       # one moment
    _refused(lists, "share memory")
    lists = _mixed(bits)
    lists[3][1] = lists[2][0]
    _refused(lists, "share memory", max_norm=1.0)
    lists = _mixed(bits, (torch.float16, torch.bfloat16, torch.float16))
    lists[0][1] = lists[0][0].view(torch.bfloat16)                  # one parameter under two types
    _refused(lists, "share memory")
    lists = _mixed(bits)                                            # what only the second type's call would see
    _refused(lists, "one device", lr=[torch.full((), 1e-2, device=DEV), torch.full((), 1e-2), 1e-2])
    _refused(lists, "not be negative", weight_decay=[0.1, float("nan"), 0.1])
    _refused(lists, "not be negative", lr=[0.1, float("nan"), 0.1], skip_nonfinite=True)
    if bits == 8:
        lists[4][1] = torch.zeros(5, dtype=torch.int16, device=DEV)[1:].view(2, 2)        # bases at an odd place
        _refused(lists, "unaligned")


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_of_different_betas_are_refused_as_a_whole(bits):
    from dtt.optim import GroupedAdamW
    torch.manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(50, device=DEV)) for _ in range(3)]
    opt = GroupedAdamW([{"params": [ps[0]]}, {"params": [ps[1]], "betas": (0.8, 0.9)}, {"params": [ps[2]], "eps": 1e-6}], lr=1e-2, state_bits=bits,
                       max_norm=1.0)

    def refused(match, error):
        before = [p.detach().clone() for p in ps]
        state = {i: {k: x.clone() for k, x in opt.state[p].items()} for i, p in enumerate(ps) if p in opt.state}
        with pytest.raises(error, match=match):
            opt.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ps, before))
        assert {i for i, p in enumerate(ps) if opt.state.get(p)} == set(state)            # no state of a step that did not happen
        assert all(torch.equal(x, opt.state[ps[i]][k]) for i, st in state.items() for k, x in st.items())
    for p in ps:
        p.grad = torch.randn_like(p)
    opt.param_groups[1]["lr"] = -1.0
    refused("lr must not be negative", ValueError)
    opt.param_groups[1]["lr"] = 1e-2
    opt.step()
    opt.param_groups[2]["weight_decay"] = -1.0
    refused("weight_decay must not be negative", ValueError)
    opt.param_groups[2]["weight_decay"] = 0.0
    own = opt.state[ps[2]]["step"]
    opt.state[ps[2]]["step"] = opt.state[ps[0]]["step"]             # counted twice a step otherwise
    refused("share memory", RuntimeError)
    opt.state[ps[2]]["step"] = own
    opt.step()
    assert [float(opt.state[p]["step"]) for p in ps] == [2.0] * 3


# ------------------------------------------------------------------------------------------------ limits
def test_an_infinite_limit_leaves_the_gradients_whatever_their_norm():
    from dtt.optim import clip_grads_
    for odd in (math.nan, math.inf):
        g = torch.ones(1000, device=DEV)
        g[7] = odd
        want = g.clone()
        norm = float(clip_grads_([g], math.inf))
        assert math.isnan(norm) if math.isnan(odd) else math.isinf(norm)
        assert torch.equal(g.isnan(), want.isnan()) and torch.equal(g.nan_to_num(), want.nan_to_num())
    g = torch.ones(1000, device=DEV)
    g[7] = math.nan
    clip_grads_([g], 1.0)                                           # a finite limit: the factor is NaN as the norm is
    assert bool(g.isnan().all())


# ------------------------------------------------------------------------------------------------ negated views
def test_negated_views_are_read_as_what_they_are_or_refused():
    from dtt.optim import GroupedAdamW, adamw_, clip_grad_norm_, clip_grads_, grad_norm
    g = torch.randn(100, device=DEV)
    neg = torch._neg_view(g)
    assert neg.is_neg()
    p, q = torch.zeros(100, device=DEV), torch.zeros(100, device=DEV)
    state = lambda: ([torch.zeros(100, device=DEV)], [torch.zeros(100, device=DEV)], [torch.zeros((), device=DEV)])
    adamw_([p], [neg], *state(), lr=0.1)
    adamw_([q], [-g], *state(), lr=0.1)
    assert torch.equal(p, q) and p.any()
    with pytest.raises(TypeError, match="resolve_neg"):
        clip_grads_([neg], 0.1)
    with pytest.raises(TypeError, match="resolve_neg"):
        adamw_([torch._neg_view(p)], [g], *state(), lr=0.1)
    m, v, s = state()
    with pytest.raises(TypeError, match="resolve_neg"):
        adamw_([p], [g], [torch._neg_view(m[0])], v, s, lr=0.1)
    with pytest.raises(TypeError, match="resolve_neg"):
        adamw_([p], [g], m, v, [torch._neg_view(s[0])], lr=0.1)
    with pytest.raises(TypeError, match="resolve_neg"):
        grad_norm([neg])
    w, u = torch.nn.Parameter(torch.zeros(100, device=DEV)), torch.nn.Parameter(torch.zeros(100, device=DEV))
    w.grad, u.grad = torch._neg_view(g.clone()), -g
    a, b = clip_grad_norm_([w], 0.5), clip_grad_norm_([u], 0.5)
    assert torch.equal(a, b) and torch.equal(w.grad, u.grad)
    w.grad, u.grad = torch._neg_view(g.clone()), -g
    for x in (w, u):
        GroupedAdamW([x], lr=0.1, max_norm=1.0).step()
    assert torch.equal(w, u)
    w2, w3 = torch.nn.Parameter(w.detach().clone()), torch.nn.Parameter(w.detach().clone())
    u2, u3 = torch.nn.Parameter(w.detach().clone()), torch.nn.Parameter(w.detach().clone())
    for x, y in ((w2, w3), (u2, u3)):                               # two betas: one norm over both
        x.grad, y.grad = (torch._neg_view(g.clone()), g.clone()) if x is w2 else (-g, g.clone())
        GroupedAdamW([{"params": [x]}, {"params": [y], "betas": (0.8, 0.9)}], lr=0.1, max_norm=1.0).step()
    assert torch.equal(w2, u2) and torch.equal(w3, u3)


# ------------------------------------------------------------------------------------------------ captured
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_over_types_and_betas_equals_eager_ones(bits):
    """Three calls under one norm in one graph, a rate in device memory shared by the groups, one gradient in another memory order."""
    from dtt.optim import GroupedAdamW

    def build():
        torch.manual_seed(3)
        ps = [torch.nn.Parameter(torch.randn(*s, device=DEV).to(t)) for s, t in
              (((40, 30), torch.bfloat16), ((300,), torch.float32), ((17, 5), torch.float32))]
        for p in ps:
            p.grad = torch.zeros_like(p)
        ps[0].grad = torch.zeros(30, 40, dtype=torch.bfloat16, device=DEV).t()
        rate = torch.full((), 1e-2, device=DEV)
        return ps, rate, GroupedAdamW([{"params": ps[:2]}, {"params": ps[2:], "betas": (0.8, 0.9)}], lr=rate, state_bits=bits, max_norm=1.0,
                                      skip_nonfinite=True)
    (ps, rate, opt), (qs, qrate, ref) = build(), build()

    def gradients(seed):
        torch.manual_seed(seed)
        for p, q in zip(ps, qs):
            p.grad.copy_(torch.randn(p.shape, device=DEV))
            q.grad.copy_(p.grad)
    gradients(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    ref.step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        opt.step()
    norm = opt.grad_norm
    for it in range(4):
        rate.fill_(1e-2 / (1 + it)); qrate.fill_(1e-2 / (1 + it))
        gradients(10 + it)
        if it == 2:
            ps[2].grad[3, 3] = math.nan; qs[2].grad[3, 3] = math.nan        # skipped in all three calls
        g.replay()
        ref.step()
        torch.cuda.synchronize()
        assert torch.equal(norm.nan_to_num(-1.0), ref.grad_norm.nan_to_num(-1.0)) and math.isnan(float(norm)) == (it == 2)
        for p, q in zip(ps, qs):
            assert torch.equal(p, q) and all(torch.equal(opt.state[p][k], ref.state[q][k]) for k in opt.state[p]), it
            assert float(opt.state[p]["step"]) == 2 + it - (it >= 2)
