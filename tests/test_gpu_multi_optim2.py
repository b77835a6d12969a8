"""More of the many-tensor optimizer: states loaded into the optimizer they came from, tensors exchanged or laid out anew under it, moments
at the end of fp32's range, param groups' other keys and hooks, mixed types, a model with frozen parameters."""
import copy

import numpy as np
import pytest
import torch

import multi_optim_ref as R
from test_gpu_multi_optim import BF16, DEV, F32, np64, tensors, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def O():
    from vae_amd import _lib, optim
    _lib.load()
    return optim


def stepped(O, sizes, dtype, bits, steps=3, seed=0, **kw):
    """(parameters, optimizer) after some steps"""
    vals, _, _ = tensors(sizes, dtype, 0, 4 + seed, 0.1)
    ps = [torch.nn.Parameter(v.clone()) for v in vals]
    opt = O.MultiAdamW(ps, lr=1e-3, state_bits=bits, **kw)
    for t in range(steps):
        step_once(opt, ps, sizes, dtype, 50 + t)
    return ps, opt


def step_once(opt, ps, sizes, dtype, seed):
    for p, g in zip(ps, tensors(sizes, dtype, 0, seed)[0]):
        p.grad = g
    opt.step(max_norm=1.0)


def everything(opt):
    out = []
    for k, st in enumerate(opt._groups):
        out += [*opt.flat_moments(k), opt.flat_master(k), st.steps]
    return [x.clone() for x in out]


def same(xs, ys):
    return len(xs) == len(ys) and all(torch.equal(x, y) for x, y in zip(xs, ys))


# ------------------------------------------------------------------------------------------------ the optimizer's own state_dict
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_its_own_state_dict_changes_nothing(O, dtype, bits):
    """state_dict gives views of the live state, so loading them reads what is being written"""
    n = [700, 3, 256, 0, 4097, 700]
    ps, opt = stepped(O, n, dtype, bits)
    qs, ref = stepped(O, n, dtype, bits)
    was = everything(opt)
    for lr in (3e-3, 2e-3):
        sd = opt.state_dict()
        sd["param_groups"][0]["lr"] = lr
        opt.load_state_dict(sd)
        assert same(everything(opt), was) and opt.param_groups[0]["lr"] == lr
    ref.param_groups[0]["lr"] = 2e-3
    for o, x in ((opt, ps), (ref, qs)):
        step_once(o, x, n, dtype, 99)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and same(everything(opt), everything(ref))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_parts_of_its_own_state_dict_trade_places(O, dtype, bits):
    """entries of two tensors exchanged and one left out: as the same change of a copy"""
    n = [700, 3, 700, 256]
    _, a = stepped(O, n, dtype, bits)
    _, b = stepped(O, n, dtype, bits)
    for opt, sd in ((a, a.state_dict()), (b, copy.deepcopy(b.state_dict()))):
        e = sd["state"]
        e[0], e[2] = e[2], e[0]
        del e[1]
        opt.load_state_dict(sd)
    assert same(everything(a), everything(b))
    assert [float(a.state_dict()["state"][k]["step"]) for k in range(4)] == [3, 0, 3, 3]
    m, v = a.flat_moments()
    assert not bool(m[768:1024].any()) and not bool(v[768:1024].any()) and bool(m[:700].any()) and bool(m[1024:1724].any())


# ------------------------------------------------------------------------------------------------ tensors exchanged or laid out anew
@pytest.mark.parametrize("bits", [32, 8])
def test_a_model_laid_out_anew_is_refused(O, bits):
    """channels_last when the optimizer was made, contiguous at the step: its moments are in another order"""
    conv = torch.nn.Conv2d(6, 8, 3).to(DEV).to(memory_format=torch.channels_last)
    opt = O.MultiAdamW(conv.parameters(), lr=1e-2, state_bits=bits)
    for p in conv.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    was = everything(opt)
    conv.to(memory_format=torch.contiguous_format)
    assert conv.weight.is_contiguous()
    kept = conv.weight.detach().clone()
    for p in conv.parameters():
        p.grad = torch.randn(p.shape, device=DEV)
    for call in (lambda: opt.step(), lambda: opt.step(max_norm=1.0), opt.flat_master):
        with pytest.raises(RuntimeError, match="make a new optimizer"):
            call()
    assert torch.equal(conv.weight, kept)
    conv.to(memory_format=torch.channels_last)       # and back: it fits again
    assert same(everything(opt), was)
    opt.step()


@pytest.mark.parametrize("change", ["replaced", "exchanged", "other list"])
def test_a_list_that_holds_other_tensors_is_refused(O, change):
    n = [300, 300, 40]
    ps, opt = stepped(O, n, F32, 32)
    was, kept = everything(opt), [p.detach().clone() for p in ps]
    group = opt.param_groups[0]
    new = torch.nn.Parameter(ps[0].detach().clone())
    new.grad = torch.ones_like(new)
    if change == "replaced":
        group["params"][0] = new
    elif change == "exchanged":
        group["params"][0], group["params"][1] = ps[1], ps[0]
    else:
        group["params"] = [*ps[:2], new]
    for max_norm in (None, 1.0):
        with pytest.raises(RuntimeError, match="list of tensors was changed"):
            opt.step(max_norm=max_norm)
    assert same(everything(opt), was) and same([p.detach() for p in ps], kept)
    group["params"] = list(ps)
    opt.step()
    assert not torch.equal(ps[0], kept[0])


# ------------------------------------------------------------------------------------------------ the end of fp32's range
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [6e20, -1e25, 3e38])
def test_a_gradient_whose_square_passes_fp32s_range(O, dtype, value):
    """(1 - beta2) g^2 is infinite from 5.8e20 on: the element's step is 0 from there on, whatever the moments' width, and the decay goes on.
    decay * p of both widths is one product of the same numbers, so the values are equal bit for bit.  The other elements, those of its block
    among them, are as if its gradient had been 0."""
    ps = [torch.nn.Parameter(torch.full((900,), 0.5, dtype=dtype, device=DEV)) for _ in range(3)]
    full, small, other = (O.MultiAdamW([p], lr=1e-2, weight_decay=0.1, state_bits=b) for p, b in zip(ps, (32, 8, 8)))
    for t in range(6):
        g = torch.randn(900, device=DEV, generator=torch.Generator(DEV).manual_seed(t)).to(dtype)
        for k, p in enumerate(ps):
            p.grad = g.clone()
            p.grad[300] = value if k < 2 and t == 1 else 0.0
        for o in (full, small, other):
            o.step()
        assert all(bool(torch.isfinite(p).all()) for p in ps), t
        if t >= 1:
            assert torch.equal(full.flat_master()[300], small.flat_master()[300]), t
        away = torch.ones(900, dtype=torch.bool, device=DEV)
        away[300] = False
        assert torch.equal(ps[1][away], ps[2][away]), t
    assert bool(torch.isinf(full.flat_moments()[1][300]))
    m, v = small.flat_moments()
    assert bool(torch.isfinite(m).all()) and bool(torch.isinf(v[300])) and int(torch.isfinite(v[:900]).sum()) == 899


def test_an_infinite_second_moment_goes_from_one_width_to_the_other(O):
    p, q = (torch.nn.Parameter(torch.full((600,), 0.5, device=DEV)) for _ in range(2))
    a, b = O.MultiAdamW([p], lr=1e-2, state_bits=8), O.MultiAdamW([q], lr=1e-2)
    for x, o in ((p, a), (q, b)):
        x.grad = torch.ones(600, device=DEV)
        x.grad[77], x.grad[300], x.grad[301] = 1e22, float("nan"), float("inf")
        o.step()
    for src, bits in ((a, 32), (b, 8)):
        r = torch.nn.Parameter(torch.full((600,), 0.5, device=DEV))
        c = O.MultiAdamW([r], lr=1e-2, state_bits=bits)
        c.load_state_dict(src.state_dict())
        m, v = c.flat_moments()
        assert bool(torch.isfinite(m[77])) and bool(torch.isinf(v[77]))
        r.grad = torch.ones(600, device=DEV)
        c.step()
        fine = torch.isfinite(r)
        assert bool(fine[77]) and not bool(fine[300]) and not bool(fine[301]) and int(fine.sum()) == 598
        assert float(r.detach()[77]) == float(torch.tensor(0.5) * torch.tensor(1 - 1e-2 * 0.01, dtype=F32))       # the decay alone


def test_a_second_moment_that_is_nan_is_not_taken_for_an_infinite_one(O):
    """a state of another origin: NaN in exp_avg_sq beside a finite exp_avg makes the parameter NaN in both widths, as in torch"""
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.full((600,), 0.5, device=DEV))
        opt = O.MultiAdamW([p], state_bits=bits)
        m, v = torch.ones(600, device=DEV), torch.ones(600, device=DEV)
        v[300] = float("nan")
        opt.load_state_dict({"state": {0: {"step": 3.0, "exp_avg": m, "exp_avg_sq": v}}, "param_groups": [{"params": [0]}]})
        assert not bool(torch.isnan(m).any())       # what was handed over stays as it was
        p.grad = torch.ones(600, device=DEV)
        for _ in range(2):
            opt.step()
            assert bool(torch.isnan(p[300])) and int(torch.isnan(p).sum()) == 1


# ------------------------------------------------------------------------------------------------ state_dicts
@pytest.mark.parametrize("key, other, limit", [("exp_avg_base", "exp_avg_sq_base", 0x7F7 - 127), ("exp_avg_sq_base", "exp_avg_base", 0x7F7 - 254)])
@pytest.mark.parametrize("bits", [32, 8])
def test_bases_end_where_their_largest_code_is_fp32s_last_level(O, key, other, limit, bits):
    n = [700, 300]
    _, src = stepped(O, n, F32, 8)
    sd = copy.deepcopy(src.state_dict())
    _, dst = stepped(O, n, F32, bits, seed=1)
    was = everything(dst)
    for bad in (limit + 1, 0x7F7, -1):
        sd["state"][1][key] = torch.tensor([limit, bad], dtype=torch.int32, device=DEV)
        with pytest.raises(ValueError, match="no levels of finite numbers"):
            dst.load_state_dict(sd)
        assert same(everything(dst), was)
    sd["state"][1][key] = torch.tensor([limit, 0], dtype=torch.int32, device=DEV)
    dst.load_state_dict(sd)
    m, v = dst.flat_moments()
    assert bool(torch.isfinite(m).all()) and bool(torch.isfinite(v).all()) and bool((v >= 0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_dict_taken_before_a_step_fits_together_after_it(O, bits):
    """codes and bases are views of the same live state: an old dict gives the present moments, not new codes with old bases"""
    n = [700, 300]
    ps, opt = stepped(O, n, F32, bits)
    sd = opt.state_dict()
    for t in range(3):       # moments of another magnitude, hence of other bases
        for p, g in zip(ps, tensors(n, F32, 0, 80 + t, 1e4)[0]):
            p.grad = g
        opt.step()
    m, v = opt.flat_moments()
    m, v = m.clone(), v.clone()
    opt.load_state_dict(sd)
    assert same(opt.flat_moments(), (m, v))


def test_other_keys_of_the_groups_are_loaded(O):
    """what a cyclic scheduler and the user keep in a group comes back: the schedule goes on where it was"""
    def make():
        ps = [torch.nn.Parameter(torch.ones(300, device=DEV)) for _ in range(2)]
        return O.MultiAdamW([{"params": ps[:1], "name": "first"}, {"params": ps[1:], "name": "second", "state_bits": 8}], lr=1e-3)
    sched = lambda o, last=-1: torch.optim.lr_scheduler.OneCycleLR(o, max_lr=[0.1, 0.2], total_steps=20, last_epoch=last)  # noqa: E731
    a = make()
    s = sched(a)
    for _ in range(5):
        a.step(), s.step()
    saved = copy.deepcopy(a.state_dict())
    saved["param_groups"][0]["tags"] = ["x"]
    b = make()
    b.param_groups[0]["name"] = b.param_groups[1]["name"] = "?"
    b.param_groups[0]["own"] = 7
    b.load_state_dict(saved)
    assert [g["name"] for g in b.param_groups] == ["first", "second"] and [g["state_bits"] for g in b.param_groups] == [32, 8]
    assert b.param_groups[0]["tags"] == ["x"] and b.param_groups[0]["tags"] is not saved["param_groups"][0]["tags"] and b.param_groups[0]["own"] == 7
    r = sched(b, s.last_epoch)
    s.step()
    for _ in range(5):
        assert [(g["lr"], g["betas"], g["max_lr"], g["min_lr"]) for g in a.param_groups] == [(g["lr"], g["betas"], g["max_lr"], g["min_lr"]) for g in b.param_groups]
        a.step(), b.step(), s.step(), r.step()
    # torch's switches are not this optimizer's, and its moments' width stays
    q = torch.nn.Parameter(torch.ones(300, device=DEV))
    c = O.MultiAdamW([q], state_bits=8)
    c.load_state_dict(torch.optim.AdamW([torch.nn.Parameter(torch.ones(300, device=DEV))], lr=0.5, fused=True).state_dict())
    g = c.param_groups[0]
    assert g["lr"] == 0.5 and g["state_bits"] == 8 and not {"fused", "foreach", "amsgrad", "maximize", "capturable", "differentiable"} & set(g)
    assert g["params"][0] is q


def test_hooks_of_the_state_dict(O):
    n, seen = [300], []
    _, opt = stepped(O, n, F32, 32)
    h = [opt.register_state_dict_pre_hook(lambda o: seen.append(("pre", o is opt))),
         opt.register_state_dict_post_hook(lambda o, sd: {**sd, "extra": 5}),
         opt.register_load_state_dict_pre_hook(lambda o, sd: seen.append(("load", o is opt, sd["extra"]))),
         opt.register_load_state_dict_pre_hook(lambda o, sd: {**sd, "param_groups": [{**sd["param_groups"][0], "lr": 0.25}]}),
         opt.register_load_state_dict_post_hook(lambda o: seen.append(("loaded", o is opt, o.param_groups[0]["lr"])))]
    sd = opt.state_dict()
    assert sd["extra"] == 5 and seen == [("pre", True)]
    was = everything(opt)
    opt.load_state_dict(sd)
    assert seen[1:] == [("load", True, 5), ("loaded", True, 0.25)] and sd["param_groups"][0]["lr"] == 1e-3 and same(everything(opt), was)
    for x in h:
        x.remove()
    opt.load_state_dict(sd)
    assert len(seen) == 3 and "extra" not in opt.state_dict() and opt.param_groups[0]["lr"] == 1e-3


def test_a_hook_that_changes_the_state_dict_changes_a_copy(O):
    _, opt = stepped(O, [300], F32, 8)
    sd = opt.state_dict()
    h = opt.register_load_state_dict_pre_hook(lambda o, d: d.update(state={}))       # nothing returned: the dict it was given counts
    opt.load_state_dict(sd)
    h.remove()
    assert len(sd["state"]) == 1 and not bool(opt.flat_moments()[0].any())


def test_entries_of_another_form_change_nothing(O):
    """codes in two dims, a remainder that is no view of the parameter's shape, a remainder of another type: refused before the first write, or
    taken for what they are"""
    n = [700, 64]
    ps, opt = stepped(O, n, BF16, 8)
    was, lr = everything(opt), opt.param_groups[0]["lr"]
    own = copy.deepcopy(opt.state_dict())

    def change(key, value):
        sd = copy.deepcopy(own)
        sd["param_groups"][0]["lr"] = 7.0
        sd["state"][1][key] = value
        return sd
    e = own["state"][1]
    for key, value, error in (("remainder", e["remainder"].float(), TypeError), ("exp_avg_base", e["exp_avg_base"].float(), TypeError),
                              ("exp_avg_sq_q", e["exp_avg_sq_q"].int(), TypeError), ("remainder", e["remainder"][:63], ValueError)):
        with pytest.raises(error, match=key if "_q" not in key else "codes"):
            opt.load_state_dict(change(key, value))
        assert same(everything(opt), was) and opt.param_groups[0]["lr"] == lr
    for key in ("remainder", "exp_avg_q", "exp_avg_sq_q"):       # the same elements in the same order, in another shape
        wide = torch.stack([e[key].view(8, 8)] * 2, 2)[:, :, 0]
        assert not wide.is_contiguous()
        opt.load_state_dict(change(key, wide))
        assert same(everything(opt), was) and opt.param_groups[0]["lr"] == 7.0


# ------------------------------------------------------------------------------------------------ the loop
def test_a_model_with_frozen_parameters_is_clipped_in_the_step(O):
    """the optimizer holds the trainable parameters only: its norm is that of all gradients there are, so it clips while it steps and leaves the
    gradients alone; where the model has a gradient that the optimizer does not step, the clip runs over the model as before"""
    from vae_amd.train import _clip_and_step
    torch.manual_seed(5)
    net = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 10)).to(DEV)
    net[0].requires_grad_(False)
    opt = O.MultiAdamW([p for p in net.parameters() if p.requires_grad], lr=1e-2)
    x = torch.randn(8, 20, device=DEV)

    def gradients():
        opt.zero_grad()
        for p in net[0].parameters():
            p.grad = None
        (net(x) * 50).square().sum().backward()
        return [p.grad.clone() for p in net[1].parameters()]
    kept = gradients()
    norm = R.norm([np64(g) for g in kept])
    assert norm > 10 and opt.holds(net[1].parameters()) and not opt.holds(net.parameters())
    _clip_and_step(net, opt, 1.0)
    assert abs(float(opt.grad_norm) - norm) <= 1.01 * R.EPS24 * norm
    assert all(torch.equal(p.grad, g) for p, g in zip(net[1].parameters(), kept))
    net[0].requires_grad_(True)       # now the model has gradients that are not stepped
    kept, opt.grad_norm = gradients(), torch.full((1,), -1.0, device=DEV)
    norm = R.norm([np64(p.grad) for p in net.parameters()])
    frozen = [p.detach().clone() for p in net[0].parameters()]
    _clip_and_step(net, opt, 1.0)
    for p, g in zip(net[1].parameters(), kept):       # torch's norm and coefficient in fp32: a sum of 970 squares, off by less than 1e-5
        within(p.grad, np64(g) / norm, 2e-5 * np.abs(np64(g) / norm))
    assert same([p.detach() for p in net[0].parameters()], frozen) and float(opt.grad_norm) == -1.0


@pytest.mark.parametrize("bits", [32, 8])
def test_an_infinite_bf16_parameter_written_from_outside_stays_infinite(O, bits):
    """beside a remainder of either sign: bf16's infinity and a positive remainder would be the bits of a NaN"""
    n = [2048, 9]
    ps, opt = stepped(O, n, BF16, bits)
    r = opt._groups[0].remainder[:2048]
    assert int((r > 0).sum()) > 100 and int((r < 0).sum()) > 100
    with torch.no_grad():
        ps[0][::2], ps[0][1::4], ps[0][3::4] = float("inf"), -float("inf"), float("nan")
    want = ps[0].detach().float()
    w = opt.flat_master()[:2048]
    # a negative remainder makes it the 32-bit number that is rounded to infinity: more than bf16's largest
    assert bool(torch.isnan(w[3::4]).all()) and not bool(torch.isnan(w[::2]).any()) and not bool(torch.isnan(w[1::4]).any())
    fine = ~torch.isnan(want)
    assert torch.equal(w[fine].sign(), want[fine].sign()) and bool((w[fine].abs() > torch.finfo(BF16).max).all())
    ps[0].grad, ps[1].grad = torch.zeros(2048, dtype=BF16, device=DEV), torch.zeros(9, dtype=BF16, device=DEV)
    for _ in range(2):
        ps[0].grad.zero_()
        opt.step()
    assert not bool(torch.isnan(ps[0][fine]).any()) and bool(torch.isnan(ps[0][3::4]).all()) and bool(torch.isfinite(ps[1]).all())
    assert torch.equal(ps[0][fine].float().sign(), want[fine].sign())


# ------------------------------------------------------------------------------------------------ mixed types
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [False, True])
def test_a_group_of_all_pairs_of_types(O, bits, clip, shift):
    """fp32 and bf16 parameters in turn, with gradients of either type, in one group: the same bits as each tensor in an optimizer of its own,
    and the step of the 64-bit restatement"""
    n = [300, 4097, 1, 256, 9000, 255, 64, 5000, 0, 0, 0, 0]
    pd, gd = [(F32, F32, BF16, BF16)[k % 4] for k in range(12)], [(F32, BF16)[k % 2] for k in range(12)]
    vals = [tensors([k], d, shift, 11 + i, 0.05)[0][0] for i, (k, d) in enumerate(zip(n, pd))]
    ps, qs = [torch.nn.Parameter(v.clone()) for v in vals], [torch.nn.Parameter(v.clone()) for v in vals]
    for p, q, d in zip(ps, qs, gd):
        p.grad_dtype = q.grad_dtype = d
    opt = O.MultiAdamW(ps, lr=1e-3, weight_decay=0.1, state_bits=bits)
    each = [O.MultiAdamW([q], lr=1e-3, weight_decay=0.1, state_bits=bits) for q in qs]
    for t in range(1, 5):
        gs = [tensors([k], d, shift, 100 * t + i, 0.3)[0][0] for i, (k, d) in enumerate(zip(n, gd))]
        for p, q, g in zip(ps, qs, gs):
            p.grad, q.grad = g, g
        before, m0, v0 = opt.flat_master().clone(), *(x.float().clone() for x in opt.flat_moments())
        opt.step(max_norm=0.5 if clip else None)
        norm = R.norm([np64(g) for g in gs])
        coef = R.coefficient(norm, 0.5) if clip else 1.0
        if clip:
            assert abs(float(opt.grad_norm) - norm) <= 1.01 * R.EPS24 * norm
        after, (m1, v1), at = opt.flat_master(), opt.flat_moments(), 0
        for k, (p, q, o) in enumerate(zip(ps, qs, each)):
            own = slice(at, at + n[k])
            (want, wm, wv), (dp, dm, dv) = R.adamw(np64(before[own]), np64(gs[k]), np64(m0[own]), np64(v0[own]), t, lr=1e-3, wd=0.1, coef=coef)
            within(after[own], want, dp, ("parameter", k, t))
            if bits == 32:
                within(m1[own], wm, dm, ("exp_avg", k, t))
                within(v1[own], wv, dv, ("exp_avg_sq", k, t))
            if pd[k] is F32:
                assert torch.equal(p.detach(), after[own])
            else:
                half = (p.detach().float() - after[own]).abs()
                assert bool((half <= after[own].abs() * 2.0 ** -8).all())
            o.grad_mul = coef       # rounded to fp32 on the way in, as the clip's coefficient is
            o.step()
            assert torch.equal(p, q), (k, t)
            mk, vk = o.flat_moments()
            assert torch.equal(m1[own], mk[:n[k]]) and torch.equal(v1[own], vk[:n[k]]) and torch.equal(after[own], o.flat_master()[:n[k]])
            end = at + -(-n[k] // 256) * 256
            assert not any(bool(x[at + n[k]:end].float().any()) for x in (m1, v1, after)), "padding was written"
            at = end


@pytest.mark.parametrize("bits", [32, 8])
def test_all_pairs_of_types_past_the_caches(O, bits):
    """a call above 96 MB goes past the caches, those of its tensors alone do not: the same bits, read-outs included"""
    n = [3_400_003, 3_400_000, 3_399_999, 3_400_257]
    pd, gd = (F32, F32, BF16, BF16), (F32, BF16, F32, BF16)
    gen = torch.Generator(DEV).manual_seed(3)
    vals = [(torch.randn(k, device=DEV, generator=gen) * 0.05).to(d) for k, d in zip(n, pd)]
    ps, qs = [torch.nn.Parameter(v.clone()) for v in vals], [torch.nn.Parameter(v.clone()) for v in vals]
    for p, q, d in zip(ps, qs, gd):
        p.grad_dtype = q.grad_dtype = d
    opt, each = O.MultiAdamW(ps, lr=1e-3, state_bits=bits), [O.MultiAdamW([q], lr=1e-3, state_bits=bits) for q in qs]
    for _ in range(2):
        for k, d, p, q in zip(n, gd, ps, qs):
            p.grad = torch.randn(k, device=DEV, generator=gen).to(d)
            q.grad = p.grad
        opt.step()
        for o in each:
            o.step()
    m, v, w = *opt.flat_moments(), opt.flat_master()
    at = 0
    for p, q, o in zip(ps, qs, each):
        end = at + o.flat_master().numel()
        assert torch.equal(p, q) and torch.equal(w[at:end], o.flat_master())
        assert torch.equal(m[at:end], o.flat_moments()[0]) and torch.equal(v[at:end], o.flat_moments()[1])
        at = end
    assert at == w.numel()


# ------------------------------------------------------------------------------------------------ graphs
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_with_and_without_a_norm_of_one_optimizer(O, bits):
    """a small step without a norm counts its workgroups in the state's scratch, one with a norm leaves numbers there: two graphs of one
    optimizer and eager steps in between, in turn, against an optimizer that only steps eagerly"""
    n = [700, 64, 9000, 0]
    vals, _, _ = tensors(n, F32, 0, 4, 0.1)
    ps, qs = [torch.nn.Parameter(v.clone()) for v in vals], [torch.nn.Parameter(v.clone()) for v in vals]
    a, b = O.MultiAdamW(ps, lr=1e-3, state_bits=bits), O.MultiAdamW(qs, lr=1e-3, state_bits=bits)
    static = [torch.zeros_like(v) for v in vals]
    for p, q, g in zip(ps, qs, static):
        p.grad, q.grad = g, g
    plain, clipped = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(plain):
        a.step()
    with torch.cuda.graph(clipped):
        a.step(max_norm=1.0)
    for t, kind in enumerate(["plain", "plain", "clipped", "eager", "plain", "clipped", "clipped", "eager clipped", "plain"]):
        for g, new in zip(static, tensors(n, F32, 0, 70 + t)[0]):
            g.copy_(new)
        norm = 1.0 if "clipped" in kind else None
        if "eager" in kind:
            a.step(max_norm=norm)
        else:
            (clipped if norm else plain).replay()
        b.step(max_norm=norm)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), (t, kind)
    assert same(everything(a), everything(b)) and [int(x) for x in a._groups[0].steps] == [9] * 4


def test_a_tensor_lr_is_filled_by_a_loaded_state(O):
    """a captured step reads that tensor, so it stays the one it is"""
    lr = torch.tensor(1e-3, device=DEV)
    p = torch.nn.Parameter(torch.ones(300, device=DEV))
    opt = O.MultiAdamW([p], lr=lr)
    sd = copy.deepcopy(opt.state_dict())
    sd["param_groups"][0]["lr"] = 0.5
    opt.load_state_dict(sd)
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.5
    opt.load_state_dict(opt.state_dict())
    assert opt.param_groups[0]["lr"] is lr and float(lr) == 0.5


def test_a_state_loaded_on_another_stream_is_recorded_there(O, monkeypatch):
    """the allocator learns of that stream's writes, so that the state of an optimizer that is dropped right away is not handed on before them"""
    seen, stream = [], torch.cuda.Stream()
    monkeypatch.setattr(O._GroupState, "used_on", lambda self, s: seen.append((self, s)))
    _, opt = stepped(O, [300], F32, 8)
    sd = copy.deepcopy(opt.state_dict())
    stream.wait_stream(torch.cuda.current_stream())
    seen.clear()
    with torch.cuda.stream(stream):
        opt.load_state_dict(sd)
    torch.cuda.current_stream().wait_stream(stream)
    assert (opt._groups[0], stream.cuda_stream) in seen
