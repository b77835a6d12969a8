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
