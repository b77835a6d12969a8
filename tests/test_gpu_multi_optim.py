"""Gradient norm, clip and AdamW over many separate tensors against 64-bit restatements (tests/multi_optim_ref.py), the 8-bit
codes bit for bit, and the operators together as a training program uses them."""
import copy
import pickle

import numpy as np
import pytest
import torch

import multi_optim_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16

SIZES = {
    "one": [1],
    "odd": [1, 2, 3, 5, 255, 256, 257, 4095, 4096, 4097, 1023, 7],
    "block": [1728, 64, 64, 64, 36864, 64, 64, 64],              # the GroupNorm double conv
    "empty": [0, 5, 0, 300, 0],
    "many": [(37 * k) % 611 + 1 for k in range(401)],            # three launches
    "large": [2_000_003, 17, 1_048_576],
}


@pytest.fixture(scope="module")
def O():
    from vae_amd import _lib, optim
    _lib.load()
    return optim


def tensors(sizes, dtype=F32, shift=0, seed=0, scale=1.0):
    """views into one guarded arena, each `shift` elements off a 64-byte boundary: (tensors, arena, mask of the elements nobody owns)"""
    g = torch.Generator().manual_seed(seed)
    at, spans = 32, []
    for n in sizes:
        spans.append((at + shift, n))
        at += (n + shift + 31) // 32 * 32 + 32
    arena = torch.full((at + 32,), 7.0, dtype=dtype)
    free = torch.ones(at + 32, dtype=torch.bool)
    for o, n in spans:
        arena[o:o + n] = (torch.randn(n, generator=g) * scale).to(dtype)
        free[o:o + n] = False
    arena = arena.to(DEV)
    return [arena[o:o + n] for o, n in spans], arena, free.to(DEV)


def params_of(values, grads):
    ps = [torch.nn.Parameter(v) for v in values]
    for p, g in zip(ps, grads):
        p.grad = g
    return ps


def np64(t):
    return t.detach().double().cpu().numpy()


def within(got, want, bound, what=""):
    off = np.abs(np64(got).reshape(-1) - np.asarray(want).reshape(-1))
    bound = np.asarray(bound).reshape(-1) + 1e-45
    assert np.all(off <= bound), (what, float(np.max(off - bound)))


# ------------------------------------------------------------------------------------------------ norm and clip
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("dtype, shift", [(F32, 0), (F32, 1), (BF16, 0), (BF16, 3)])
@pytest.mark.parametrize("scale", [3.0, 1e-6])
def test_norm_and_clip(O, sizes, dtype, shift, scale):
    n = SIZES[sizes]
    gs, arena, free = tensors(n, dtype, shift, 1, scale)
    ps = params_of([torch.zeros_like(g) for g in gs], gs)
    ref = [np64(g) for g in gs]
    norm = R.norm(ref)
    # sums in 64 bits (N * 2^-53 is nothing), one rounding to fp32
    assert abs(float(O.grad_norm(ps)) - norm) <= 1.01 * R.EPS24 * norm
    got = O.clip_grad_norm_(ps, 1.0)
    assert got.shape == () and got.dtype == F32 and abs(float(got) - norm) <= 1.01 * R.EPS24 * norm
    coef = R.coefficient(norm, 1.0)
    half = 2.0 ** -8 if dtype is BF16 else R.EPS24
    for g, r in zip(gs, ref):       # coef rounded, product rounded (and, for bf16, rounded once more)
        within(g, r * coef, (2.01 * R.EPS24 + (half if dtype is BF16 else 0)) * np.abs(r * coef))
    assert bool((arena[free] == 7).all()), "an element between the tensors was written"


def test_norm_of_mixed_types_and_no_gradient(O):
    a, _, _ = tensors([300, 5], F32, 1, 2)
    b, _, _ = tensors([70, 4099], BF16, 0, 3)
    ps = params_of([torch.zeros_like(x) for x in a + b], a + b)
    ps.append(torch.nn.Parameter(torch.ones(4, device=DEV)))       # without a gradient
    want = R.norm([np64(x) for x in a + b])
    assert abs(float(O.grad_norm(ps)) - want) <= 1.01 * R.EPS24 * want
    assert abs(float(O.clip_grad_norm_(iter(ps), 1e9)) - want) <= 1.01 * R.EPS24 * want
    assert float(O.grad_norm([ps[-1]])) == 0.0


def test_norm_passes_fp32s_range_inside(O):
    g = torch.full((1000,), 1e30, device=DEV)       # squares are 1e60
    p = params_of([torch.zeros_like(g)], [g])
    want = 1e30 * np.sqrt(1000.0)
    assert abs(float(O.clip_grad_norm_(p, 2.0)) / want - 1) < 2 * R.EPS24 + 4e-8       # 1e30 itself is rounded in fp32
    within(g, np.full(1000, 2.0 / np.sqrt(1000)), 1e-6)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_clip_with_a_norm_that_is_not_finite_is_torchs(O, bad):
    x = torch.randn(600)
    x[77] = bad
    mine, theirs = params_of([torch.zeros(600, device=DEV)], [x.to(DEV)]), params_of([torch.zeros(600)], [x.clone()])
    n = O.clip_grad_norm_(mine, 1.0)
    t = torch.nn.utils.clip_grad_norm_(theirs, 1.0)
    assert str(float(n)) == str(float(t))
    assert torch.equal(torch.nan_to_num(mine[0].grad.cpu(), nan=5.0), torch.nan_to_num(theirs[0].grad, nan=5.0))
    p = params_of([torch.zeros(600, device=DEV)], [x.to(DEV)])
    with pytest.raises(RuntimeError, match="cannot be clipped"):
        O.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert torch.equal(torch.nan_to_num(p[0].grad.cpu(), nan=5.0), torch.nan_to_num(x, nan=5.0))       # left as they were


def test_clip_refuses_what_it_cannot_write_in_place(O):
    p = torch.nn.Parameter(torch.zeros(8, 8, device=DEV))
    p.sum().backward()
    p.grad = torch.zeros(1, 1, device=DEV).expand(8, 8)
    with pytest.raises(ValueError, match="gaps or overlaps"):
        O.clip_grad_norm_([p], 1.0)
    g = torch.randn(8, device=DEV)
    ps = params_of([torch.zeros(8, device=DEV), torch.zeros(8, device=DEV)], [g, g])
    with pytest.raises(ValueError, match="same memory"):
        O.clip_grad_norm_(ps, 1.0)
    q = torch.nn.Parameter(torch.zeros(8, device=DEV, dtype=torch.float16))
    q.grad = torch.zeros_like(q)
    with pytest.raises(TypeError, match="float16"):
        O.clip_grad_norm_([q], 1.0)


def test_norm_is_the_same_on_every_run(O):
    gs, _, _ = tensors(SIZES["many"] + SIZES["large"], F32, 1, 9)
    ps = params_of([torch.zeros_like(g) for g in gs], gs)
    first = O.grad_norm(ps)
    assert all(torch.equal(O.grad_norm(ps), first) for _ in range(4))


# ------------------------------------------------------------------------------------------------ the step
def state_of(opt, i=0):
    return opt.state_dict()["state"][i]


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("pd, gd, shift", [(F32, F32, 0), (F32, F32, 1), (BF16, BF16, 0), (BF16, BF16, 1), (F32, BF16, 3)])
@pytest.mark.parametrize("bits", [32, 8])
def test_three_steps(O, sizes, pd, gd, shift, bits):
    n = SIZES[sizes]
    vals, arena, free = tensors(n, pd, shift, 11, 0.05)
    ps = [torch.nn.Parameter(v) for v in vals]
    if gd is not pd:
        for p in ps:
            p.grad_dtype = gd       # gradients of another type than the parameter's
    opt = O.MultiAdamW(ps, lr=1e-3, weight_decay=0.1, state_bits=bits)
    total = sum(n)
    clip = sizes in ("odd", "many", "large")
    for t in range(1, 4):
        gs, garena, _ = tensors(n, gd, shift, 20 + t, 0.3)
        for p, g in zip(ps, gs):
            p.grad = g
        before, kept = opt.flat_master().clone(), garena.clone()
        sd = opt.state_dict()["state"]
        old = [{k: (x.clone() if torch.is_tensor(x) else x) for k, x in sd[i].items()} for i in range(len(n))]
        opt.step(max_norm=0.5 if clip else None)
        assert torch.equal(garena, kept), "a gradient was written"
        norm = R.norm([np64(g) for g in gs])
        coef = R.coefficient(norm, 0.5) if clip else 1.0
        if clip:
            assert abs(float(opt.grad_norm) - norm) <= 1.01 * R.EPS24 * norm
        after, new, at = opt.flat_master(), opt.state_dict()["state"], 0
        for i, k in enumerate(n):
            w0, w1 = np64(before[at:at + k]), after[at:at + k]
            if bits == 32:
                m0, v0 = np64(old[i]["exp_avg"]), np64(old[i]["exp_avg_sq"])
            else:
                m0 = R.unpack_tensor(old[i]["exp_avg_q"].cpu().numpy(), old[i]["exp_avg_base"].cpu().numpy(), True)
                v0 = R.unpack_tensor(old[i]["exp_avg_sq_q"].cpu().numpy(), old[i]["exp_avg_sq_base"].cpu().numpy(), False)
            (p1, m1, v1), (dp, dm, dv) = R.adamw(w0, np64(gs[i]), m0, v0, t, lr=1e-3, wd=0.1, coef=coef)
            within(w1, p1, dp, ("parameter", i, t))
            if bits == 32:
                within(new[i]["exp_avg"], m1, dm, ("exp_avg", i, t))
                within(new[i]["exp_avg_sq"], v1, dv, ("exp_avg_sq", i, t))
            else:       # codes: the same bits as the definition applied to the same fp32 moments
                gk = gs[i].float().cpu().numpy() * np.float32(min(1.0, 0.5 / (norm + 1e-6)) if clip else 1.0)
                m32, v32 = R.moments32(gk, m0.astype(np.float32), v0.astype(np.float32))
                q, b = R.pack_tensor(m32, t, R.RATE_M, 127, True)
                assert np.array_equal(new[i]["exp_avg_base"].cpu().numpy(), b) and np.array_equal(new[i]["exp_avg_q"].cpu().numpy(), q), (i, t)
                q, b = R.pack_tensor(v32, t, R.RATE_V, 254, False)
                assert np.array_equal(new[i]["exp_avg_sq_base"].cpu().numpy(), b) and np.array_equal(new[i]["exp_avg_sq_q"].cpu().numpy(), q), (i, t)
            if pd is BF16:      # the parameter is its master rounded to nearest
                half = (ps[i].detach().float() - w1).abs()
                assert bool((half <= w1.abs() * 2.0 ** -8).all())
            assert float(new[i]["step"]) == t
            at += -(-k // 256) * 256
        m, v = opt.flat_moments()
        own = torch.zeros(max(at, 256), dtype=torch.bool, device=DEV)
        at = 0
        for k in n:
            own[at:at + k] = True
            at += -(-k // 256) * 256
        for flat in (m, v, after):
            assert not bool(flat[~own].float().abs().any()), "padding was written"
    assert bool((arena[free] == 7).all()), "an element between the tensors was written"
    assert total == sum(p.numel() for p in ps)


@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("bits", [32, 8])
def test_with_and_without_a_norm_the_step_is_the_same(O, sizes, bits):
    """a norm that clips nothing changes no bit: the numbers prepared beside the norm, those worked out by every workgroup of a small step and
    those of a launch of their own agree, and the counts advance alike"""
    n = SIZES[sizes]
    vals, _, _ = tensors(n, F32, 0, 3, 0.05)
    ps, qs = [torch.nn.Parameter(v.clone()) for v in vals], [torch.nn.Parameter(v.clone()) for v in vals]
    a, b = O.MultiAdamW(ps, lr=1e-3, state_bits=bits), O.MultiAdamW(qs, lr=1e-3, state_bits=bits)
    for t in range(5):
        gs, _, _ = tensors(n, F32, 0, 30 + t, 0.3)
        for k, (p, q, g) in enumerate(zip(ps, qs, gs)):
            p.grad = q.grad = None if (k + t) % 3 == 0 and len(n) > 1 else g
        a.step()
        b.step(max_norm=1e30)
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), t
    assert all(torch.equal(x, y) for x, y in zip(a.flat_moments(), b.flat_moments()))
    sa, sb = a.state_dict()["state"], b.state_dict()["state"]
    want = [sum(not ((k + t) % 3 == 0 and len(n) > 1) for t in range(5)) for k in range(len(n))]
    assert [float(sa[k]["step"]) for k in range(len(n))] == want == [float(sb[k]["step"]) for k in range(len(n))]


def test_two_optimizers_at_once(O):
    """two threads, each with its own model, optimizer and stream, against the same steps one after the other"""
    import threading
    n = [5000, 300, 70_000, 1]

    def make(seed):
        vals, _, _ = tensors(n, F32, 0, seed, 0.05)
        ps = [torch.nn.Parameter(v) for v in vals]
        return ps, O.MultiAdamW(ps, lr=1e-3, state_bits=8), [tensors(n, F32, 0, 1000 * seed + t, 0.3)[0] for t in range(20)]

    def run(ps, opt, grads, out):
        with torch.cuda.stream(torch.cuda.Stream()):
            for g in grads:
                for p, x in zip(ps, g):
                    p.grad = x.clone()
                out.append(O.clip_grad_norm_(ps, 1.0))
                opt.step(max_norm=0.5)
        torch.cuda.current_stream().synchronize()
    both, alone = [make(1), make(2)], [make(1), make(2)]
    torch.cuda.synchronize()
    norms = [[] for _ in range(4)]
    threads = [threading.Thread(target=run, args=(*x, norms[k])) for k, x in enumerate(both)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k, x in enumerate(alone):
        run(*x, norms[2 + k])
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(p, q) for p, q in zip(both[k][0], alone[k][0]))
        assert all(torch.equal(x, y) for x, y in zip(norms[k], norms[2 + k])) and len(norms[k]) == 20


def test_bf16_parameters_follow_the_fp32_run_to_the_bit(O):
    """parameter and remainder are 32 bits of master: the run is that of fp32 parameters with the same start and gradients"""
    n = [300, 4097, 1]
    for bits in (32, 8):
        vals, _, _ = tensors(n, BF16, 1, 5, 0.02)
        half, full = [torch.nn.Parameter(v) for v in vals], [torch.nn.Parameter(v.float()) for v in vals]
        a, b = O.MultiAdamW(half, lr=1e-4, state_bits=bits), O.MultiAdamW(full, lr=1e-4, state_bits=bits)
        for t in range(30):
            gs, _, _ = tensors(n, BF16, 0, 100 + t, 1e-3)
            for p, q, g in zip(half, full, gs):
                p.grad, q.grad = g, g.float()
            a.step(max_norm=1.0)
            b.step(max_norm=1.0)
        assert torch.equal(a.flat_master(), b.flat_master())
        assert all(torch.equal(x, y) for x, y in zip(a.flat_moments(), b.flat_moments()))
        moved = torch.cat([(p.detach().float() - v.float()).abs() for p, v in zip(full, tensors(n, BF16, 1, 5, 0.02)[0])])
        assert float(moved.max()) > 0


def test_a_parameter_written_from_outside_keeps_what_was_written(O):
    p = torch.nn.Parameter(torch.randn(2048, device=DEV).to(BF16))
    opt = O.MultiAdamW([p], lr=1e-3)
    for t in range(3):
        p.grad = torch.randn(2048, device=DEV).to(BF16)
        opt.step()
    new = torch.randn(2048, device=DEV).to(BF16)
    new[:6] = torch.tensor([0.0, -0.0, float("nan"), float("inf"), -float("inf"), 1e-40], device=DEV)
    with torch.no_grad():
        p.copy_(new)
    w = opt.flat_master()
    fine = torch.isfinite(new)
    # the remainder left from before is at most half a last place (half a step: 2^-8 relative, of the lower binade twice that)
    assert bool(((w - new.float()).abs() <= new.float().abs() * 2.0 ** -7 + 1e-38)[fine].all())
    assert bool(torch.isnan(w[2])) and bool((torch.signbit(w) == torch.signbit(new.float()))[~torch.isnan(new)].all())
    p.grad = torch.zeros_like(p)
    opt.step()
    assert bool(torch.isfinite(p[fine]).all()) and bool(torch.isnan(p[2]))


def test_groups_missing_gradients_and_step_counts(O):
    vals, _, _ = tensors([600, 77, 256, 1000], F32, 0, 1, 0.1)
    ps = [torch.nn.Parameter(v) for v in vals]
    opt = O.MultiAdamW([{"params": ps[:2], "weight_decay": 0.0, "lr": 1e-2}, {"params": ps[2:], "betas": (0.5, 0.9), "state_bits": 8}], lr=1e-3)
    start = [p.detach().clone() for p in ps]
    for t in range(4):
        for k, p in enumerate(ps):
            p.grad = torch.randn(p.shape, device=DEV, generator=torch.Generator(DEV).manual_seed(t * 10 + k)) if (t + k) % 2 or k == 3 else None
        have = [p.grad is not None for p in ps]
        was = [p.detach().clone() for p in ps]
        opt.step(max_norm=1.0)
        want = R.norm([np64(p.grad) for p in ps if p.grad is not None])       # over both groups
        assert abs(float(opt.grad_norm) - want) <= 1.01 * R.EPS24 * want
        for p, w, h in zip(ps, was, have):
            assert torch.equal(p, w) != h
    assert [float(opt.state_dict()["state"][k]["step"]) for k in range(4)] == [2, 2, 2, 4]
    for p in ps:
        p.grad = None
    opt.step(max_norm=1.0)       # nothing to do
    assert [float(opt.state_dict()["state"][k]["step"]) for k in range(4)] == [2, 2, 2, 4]
    assert all(not torch.equal(p, s) for p, s in zip(ps, start))


def test_a_group_added_later_and_a_scheduler(O):
    a, b = (torch.nn.Parameter(torch.ones(300, device=DEV)) for _ in range(2))
    opt = O.MultiAdamW([a], lr=0.1, weight_decay=0.0)
    sched = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.1)
    ta, tb = (torch.nn.Parameter(torch.ones(300)) for _ in range(2))
    ref = torch.optim.AdamW([ta], lr=0.1, weight_decay=0.0)
    rs = torch.optim.lr_scheduler.StepLR(ref, step_size=1, gamma=0.1)
    for t in range(4):
        if t == 2:
            opt.add_param_group({"params": [b], "lr": 0.5})
            ref.add_param_group({"params": [tb], "lr": 0.5})
        g = torch.randn(300)
        for p, q in ((a, ta), (b, tb)):
            p.grad, q.grad = g.to(DEV), g.clone()
        assert opt.step(lambda: 3.5) == 3.5
        ref.step()
        if t < 2:
            sched.step(), rs.step()
    for p, q in ((a, ta), (b, tb)):
        within(p, np64(q), 3e-6 * np.ones(300))       # both in fp32: a few halves of 2^-24 of 1 and of steps of 0.1 to 0.5
    with pytest.raises(ValueError, match="share memory"):
        opt.add_param_group({"params": [torch.nn.Parameter(a.detach()[5:9])]})
    assert len(opt.param_groups) == 2


def test_hooks_and_a_list_that_was_changed(O):
    p, seen = torch.nn.Parameter(torch.ones(300, device=DEV)), []
    opt = O.MultiAdamW([p], lr=0.1)
    pre = opt.register_step_pre_hook(lambda o, args, kw: seen.append(("pre", o is opt, args[0] is opt, kw["max_norm"])))
    post = opt.register_step_post_hook(lambda o, args, kw: seen.append(("post", o is opt)))
    p.grad = torch.ones_like(p)
    opt.step(max_norm=2.0)
    assert seen == [("pre", True, True, 2.0), ("post", True)]
    pre.remove(), post.remove()
    opt.register_step_pre_hook(lambda o, args, kw: (args, {"max_norm": 0.0}))       # a clip to nothing
    opt.step(max_norm=2.0)
    assert float(opt.grad_norm) > 0 and len(seen) == 2
    opt.param_groups[0]["params"].append(torch.nn.Parameter(torch.ones(5, device=DEV)))
    with pytest.raises(RuntimeError, match="list of tensors was changed"):
        opt.step()


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_bad_gradient_stays_in_its_element(O, what, bits):
    p, q = (torch.nn.Parameter(torch.full((700,), 0.5, device=DEV)) for _ in range(2))
    a, b = O.MultiAdamW([p], state_bits=bits), O.MultiAdamW([q], state_bits=bits)
    for t in range(3):
        g = torch.randn(700, device=DEV, generator=torch.Generator(DEV).manual_seed(t))
        q.grad = g.clone()
        if t == 0:
            g[300] = float(what)
        p.grad = g
        if t == 0:
            q.grad[300] = 0.0       # the neighbours' block: its largest value is another element's
        a.step()
        b.step()
    keep = torch.arange(700, device=DEV) != 300
    assert torch.equal(p[keep], q[keep]) and bool(torch.isnan(p[300]))
    (m, v), (mq, vq) = a.flat_moments(), b.flat_moments()
    assert torch.equal(m[:700][keep], mq[:700][keep]) and torch.equal(v[:700][keep], vq[:700][keep])
    if bits == 8:
        assert bool(torch.isnan(m[300])) and bool(torch.isnan(v[300]))


def test_extreme_values(O):
    """zero, tiny and huge gradients in one block: nothing turns into NaN, nothing that has a second moment loses it"""
    g = torch.zeros(512, device=DEV)
    g[1], g[2], g[3], g[4] = 1e-18, 1e-12, 1e18, -1e-3
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.zeros(512, device=DEV))
        opt = O.MultiAdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits)
        for t in range(5):
            p.grad = g.clone()
            opt.step()
        m, v = opt.flat_moments()
        assert bool(torch.isfinite(p).all()) and not bool(p[5:].any()) and not bool(p[0]) and not bool(v[5:512].any())
        assert bool((v[1:5] > 0).all())
        assert bool((p.abs() <= 5 * 1e-3 * (1 + 1e-5)).all())       # |m| <= sqrt(v): five steps of at most lr with a constant gradient


def test_a_norm_that_is_nan_leaves_the_padding_alone(O):
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(300, device=DEV))
        opt = O.MultiAdamW([p], state_bits=bits)
        p.grad = torch.ones(300, device=DEV)
        p.grad[7] = float("nan")
        opt.step(max_norm=1.0)
        assert bool(torch.isnan(p).all()) and bool(torch.isnan(opt.grad_norm))       # as clip_grad_norm_ and step() of torch
        for flat in (*opt.flat_moments(), opt.flat_master()):
            assert not bool(flat[300:].any())


@pytest.mark.parametrize("pd, bits", [(F32, 8), (BF16, 32)])
def test_offsets_beyond_32_bits(O, pd, bits):
    """one tensor of more than 2^31 elements: its last ones are stepped like the same ones of a small tensor, its first ones too"""
    n, m = (1 << 31) + 4097, 5000
    p = torch.nn.Parameter(torch.full((n,), 0.5, dtype=pd, device=DEV))
    p.grad = torch.zeros(n, dtype=pd, device=DEV)
    g = torch.randn(m, device=DEV).to(pd)
    p.grad[:m], p.grad[-m:] = g, g
    q = torch.nn.Parameter(torch.full((m,), 0.5, dtype=pd, device=DEV))
    q.grad = g.clone()
    a, b = O.MultiAdamW([p], lr=1e-2, state_bits=bits), O.MultiAdamW([q], lr=1e-2, state_bits=bits)
    norm = R.norm([np64(g)]) * np.sqrt(2.0)
    a.step(max_norm=1.0)
    b.grad_mul = R.coefficient(norm, 1.0)
    b.step()
    assert abs(float(a.grad_norm) - norm) <= 1.01 * R.EPS24 * norm
    # coef is the same number rounded to fp32 in both, so the small tensor's bits are the large one's
    assert torch.equal(p[:m], q) and torch.equal(p[-m:], q)
    mid = p[m:m + 100].float()
    assert bool((mid == mid[0]).all())       # no gradient there: the decay alone
    del a, p
    torch.cuda.empty_cache()


def test_a_group_added_after_a_capture_leaves_the_graph_alone(O):
    p, q = (torch.nn.Parameter(torch.ones(5000, device=DEV)) for _ in range(2))
    a, b = O.MultiAdamW([p], lr=1e-2), O.MultiAdamW([q], lr=1e-2)
    p.grad, q.grad = torch.randn(5000, device=DEV), None
    q.grad = p.grad.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(max_norm=1.0)
    a.add_param_group({"params": [torch.nn.Parameter(torch.ones(40_000, device=DEV))]})
    fill = [torch.full((321,), 3.0, dtype=torch.float64, device=DEV) for _ in range(64)]       # what a freed scratch would be given to
    for _ in range(3):
        graph.replay()
        b.step(max_norm=1.0)
        torch.cuda.synchronize()
        assert torch.equal(p, q)
    assert all(bool((x == 3).all()) for x in fill)


def test_state_dicts_that_do_not_fit_change_nothing(O):
    p = torch.nn.Parameter(torch.randn(700, device=DEV))
    opt = O.MultiAdamW([p], state_bits=8)
    p.grad = torch.randn(700, device=DEV)
    opt.step()
    kept, lr = [x.clone() for x in opt.flat_moments()], opt.param_groups[0]["lr"]

    def broken(key, value):
        sd = copy.deepcopy(opt.state_dict())
        sd["param_groups"][0]["lr"] = 7.0
        sd["state"][0][key] = value
        return sd
    for key, value, match in (("step", -1.0, "step count"), ("step", 1.5, "step count"), ("step", float("nan"), "step count"),
                              ("exp_avg_base", torch.full((3,), 3000, dtype=torch.int32), "no levels"),
                              ("exp_avg_sq_base", torch.full((3,), -5, dtype=torch.int32), "no levels"),
                              ("exp_avg_q", torch.zeros(699, dtype=torch.uint8), "exp_avg_q"), ("stride", (2,), "order of strides")):
        with pytest.raises((ValueError, RuntimeError), match=match):
            sd = broken(key, value)
            if "base" in key:       # both on one device
                for k2 in ("exp_avg_base", "exp_avg_sq_base"):
                    sd["state"][0][k2] = sd["state"][0][k2].cpu()
            opt.load_state_dict(sd)
        assert all(torch.equal(x, y) for x, y in zip(opt.flat_moments(), kept)) and opt.param_groups[0]["lr"] == lr
        assert float(state_of(opt)["step"]) == 1


def test_memory_orders_and_expanded_gradients(O):
    a = torch.nn.Parameter(torch.randn(8, 6, 3, 3, device=DEV).to(memory_format=torch.channels_last))
    b = torch.nn.Parameter(a.detach().contiguous().clone())
    c = torch.nn.Parameter(torch.randn(40, 7, device=DEV).t())
    d = torch.nn.Parameter(c.detach().contiguous().clone())
    for bits in (32, 8):
        opts = [O.MultiAdamW([p], lr=1e-2, state_bits=bits) for p in (a, b, c, d)]
        for t in range(3):
            g4, g2 = torch.randn(8, 6, 3, 3, device=DEV), torch.randn(7, 40, device=DEV)
            a.grad, b.grad, c.grad, d.grad = (g4 if t else g4.to(memory_format=torch.channels_last)), g4.clone(), g2, g2.clone()
            if t == 2:
                c.grad = d.grad = torch.ones(1, 1, device=DEV).expand(7, 40)       # what sum().backward() leaves
            for o in opts:
                o.step()
        if bits == 32:
            assert torch.equal(a, b) and torch.equal(c, d)
            for x, y in ((opts[0], opts[1]), (opts[2], opts[3])):
                assert torch.equal(state_of(x)["exp_avg"], state_of(y)["exp_avg"])
    assert a.is_contiguous(memory_format=torch.channels_last) and not c.is_contiguous()


def test_refusals_on_the_device(O):
    p = torch.nn.Parameter(torch.zeros(16, device=DEV))
    with pytest.raises(ValueError, match="gaps or overlaps"):
        O.MultiAdamW([torch.nn.Parameter(torch.zeros(8, 8, device=DEV)[:, :4])])
    with pytest.raises(ValueError, match="share memory"):
        O.MultiAdamW([p, torch.nn.Parameter(p.detach()[4:8])])
    with pytest.raises(TypeError, match="float16"):
        O.MultiAdamW([torch.nn.Parameter(torch.zeros(4, device=DEV, dtype=torch.float16))])
    with pytest.raises(RuntimeError, match="MI355X only"):
        O.MultiAdamW([p, torch.nn.Parameter(torch.zeros(4))])
    opt = O.MultiAdamW([p])
    p.grad = torch.zeros_like(p)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            opt.step(max_norm=bad)
    opt.param_groups[0]["state_bits"] = 8
    with pytest.raises(RuntimeError, match="state_bits"):
        opt.step()
    opt.param_groups[0]["state_bits"] = 32
    opt.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError, match="lr"):
        opt.step()
    opt.param_groups[0]["lr"] = 1e-3
    before = p.detach().clone()
    p.data = torch.zeros(32, device=DEV)
    with pytest.raises(RuntimeError, match="make a new optimizer"):
        opt.step()
    p.data = torch.zeros(16)       # moved to the host after the optimizer was made
    with pytest.raises(RuntimeError, match="make a new optimizer"):
        opt.step()
    p.data = before
    opt.step()
    for f in (copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="state_dict"):
            f(opt)


# ------------------------------------------------------------------------------------------------ state
def test_state_interchanges_with_torch(O):
    shapes = [(5, 3, 3, 3), (300,), (1,)]
    mine = [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in shapes]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    a, b = O.MultiAdamW(mine, lr=1e-3), torch.optim.AdamW(theirs, lr=1e-3)

    def go(pairs, k):
        for t in range(k):
            for ps in pairs:
                for i, p in enumerate(ps[1]):
                    p.grad = torch.randn(p.shape, device=DEV, generator=torch.Generator(DEV).manual_seed(100 * t + i))
                ps[0].step()

    def near(xs, ys):       # two fp32 runs of the same formula: 5 steps of at most 2 lr, each off by some halves, and p's own roundings
        for x, y in zip(xs, ys):
            within(x, np64(y), 10 * R.EPS24 * np.abs(np64(y)) + 5 * 2e-3 * 40 * R.EPS24)

    go([(a, mine), (b, theirs)], 3)
    near(mine, theirs)
    mine2, theirs2 = [torch.nn.Parameter(p.detach().clone()) for p in mine], [torch.nn.Parameter(p.detach().clone()) for p in mine]
    a2, b2 = O.MultiAdamW(mine2, lr=9.0), torch.optim.AdamW(theirs2, lr=9.0)
    a2.load_state_dict(b.state_dict())       # torch's state here, this one's there
    b2.load_state_dict(copy.deepcopy(a.state_dict()))       # torch's loader keeps the tensors it is given, and `a` goes on stepping
    assert a2.param_groups[0]["lr"] == 1e-3 == b2.param_groups[0]["lr"]
    go([(a2, mine2), (b2, theirs2), (a, mine)], 2)
    near(mine2, theirs2)
    near(mine2, mine)
    with pytest.raises(ValueError, match="amsgrad"):
        a2.load_state_dict(torch.optim.AdamW(theirs, lr=1e-3, amsgrad=True).state_dict())
    with pytest.raises(ValueError, match="other lengths"):
        O.MultiAdamW(mine[:2]).load_state_dict(a.state_dict())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_run_goes_on_from_its_saved_state(O, tmp_path, dtype, bits):
    n = [700, 3, 256, 0, 4097]
    vals, _, _ = tensors(n, dtype, 0, 4, 0.1)
    ps = [torch.nn.Parameter(v.clone()) for v in vals]
    opt = O.MultiAdamW(ps, lr=1e-3, state_bits=bits)

    def go(opt, ps, frm, to):
        for t in range(frm, to):
            for p, g in zip(ps, tensors(n, dtype, 0, 50 + t)[0]):
                p.grad = g
            opt.step(max_norm=1.0)
    go(opt, ps, 0, 3)
    torch.save({"opt": opt.state_dict(), "ps": [p.detach() for p in ps]}, tmp_path / "c.pt")
    go(opt, ps, 3, 6)
    saved = torch.load(tmp_path / "c.pt", weights_only=True, map_location="cpu")
    qs = [torch.nn.Parameter(x.to(DEV)) for x in saved["ps"]]
    again = O.MultiAdamW(qs, lr=5.0, state_bits=bits)
    again.load_state_dict(saved["opt"])
    go(again, qs, 3, 6)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and torch.equal(opt.flat_master(), again.flat_master())
    assert all(torch.equal(x, y) for x, y in zip(opt.flat_moments(), again.flat_moments()))


def test_conversion_between_the_two_forms(O):
    n = [700, 3, 256, 4097]
    vals, _, _ = tensors(n, F32, 0, 4, 0.1)
    ps = [torch.nn.Parameter(v) for v in vals]
    full = O.MultiAdamW(ps, lr=1e-3)
    for t in range(3):
        for p, g in zip(ps, tensors(n, F32, 0, 50 + t)[0]):
            p.grad = g
        full.step()
    small = O.MultiAdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], state_bits=8)
    small.load_state_dict(full.state_dict())
    sd, fd = small.state_dict()["state"], full.state_dict()["state"]
    for i in range(len(n)):
        for key, codes, signed in (("exp_avg", 127, True), ("exp_avg_sq", 254, False)):
            q, b = R.pack_tensor(fd[i][key].cpu().numpy(), 0, 0, codes, signed, nearest=True)
            assert np.array_equal(sd[i][key + "_q"].cpu().numpy(), q) and np.array_equal(sd[i][key + "_base"].cpu().numpy(), b)
    m, v = small.flat_moments()
    back = O.MultiAdamW([torch.nn.Parameter(p.detach().clone()) for p in ps])
    back.load_state_dict(small.state_dict())
    assert all(torch.equal(x, y.float()) for x, y in zip(back.flat_moments(), (m, v)))
    bad = small.state_dict()
    bad["state"][1]["exp_avg_base"] = torch.zeros(7, dtype=torch.int32)
    kept = [x.clone() for x in back.flat_moments()]
    with pytest.raises(ValueError, match="exp_avg_base"):
        back.load_state_dict(bad)
    assert all(torch.equal(x, y) for x, y in zip(back.flat_moments(), kept))


def test_every_code_is_read_back(O):
    """both conversions over all 256 codes and bases from the smallest to the largest, fp32 and bf16"""
    L = O._lib
    bases = np.array([[0, 0], [1, 1], [300, 400], [1016 - 127, 1016 - 254], [0x7F7 - 127, 0x7F7 - 254]], np.int16)
    nb = len(bases)
    q = torch.arange(256, dtype=torch.uint8).repeat(nb).to(DEV)
    b = torch.from_numpy(bases).to(DEV)
    want_m = np.concatenate([R.unpack(np.arange(256), int(x[0]), True) for x in bases])
    want_v = np.concatenate([R.unpack(np.arange(256), int(x[1]), False) for x in bases])
    for dtype in (F32, BF16):
        m, v = (torch.empty(256 * nb, dtype=dtype, device=DEV) for _ in range(2))
        L.call("vae_moments8_unpack", q.data_ptr(), q.data_ptr(), b.data_ptr(), m.data_ptr(), v.data_ptr(), nb, int(dtype is BF16), L.current_stream())
        # a subnormal level (base 0) is bits << 20, not mantissa and exponent: compared from the first normal number on
        for got, want in ((np64(m), want_m), (np64(v), want_v)):
            normal = ~(np.abs(want) < 2.0 ** -126) | (want == 0)
            assert np.array_equal(got[normal], want[normal], equal_nan=True)
        if dtype is F32:
            qm, qv, bb = torch.empty_like(q), torch.empty_like(q), torch.empty_like(b)
            L.call("vae_moments8_pack", m.data_ptr(), v.data_ptr(), qm.data_ptr(), qv.data_ptr(), bb.data_ptr(), nb, L.current_stream())
            assert torch.equal(qm, q) and torch.equal(qv, q) and torch.equal(bb, b)


def test_a_thousand_steps_in_eight_bits_are_the_definitions(O):
    """500 steps of a constant gradient, then 500 without one: codes and bases of every step's end are the restatement's, bit for bit.
    (How near the definition comes to moments in 32 bits is looked at in tests/test_multi_optim_host.py.)"""
    n = 600
    g = (torch.randn(n, generator=torch.Generator().manual_seed(3)).abs() + 0.1).to(DEV)
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = O.MultiAdamW([p], lr=0.0, state_bits=8)
    m, v = np.zeros(n, np.float32), np.zeros(n, np.float32)
    for t in range(1, 1001):
        p.grad = g if t <= 500 else torch.zeros_like(g)
        opt.step()
        m, v = R.moments32(p.grad.cpu().numpy(), m, v)
        qm, bm = R.pack_tensor(m, t, R.RATE_M, 127, True)
        qv, bv = R.pack_tensor(v, t, R.RATE_V, 254, False)
        m, v = R.unpack_tensor(qm, bm, True).astype(np.float32), R.unpack_tensor(qv, bv, False).astype(np.float32)
        if t % 50 == 0:
            got = state_of(opt)
            assert np.array_equal(got["exp_avg_q"].cpu().numpy(), qm) and np.array_equal(got["exp_avg_base"].cpu().numpy(), bm), t
            assert np.array_equal(got["exp_avg_sq_q"].cpu().numpy(), qv) and np.array_equal(got["exp_avg_sq_base"].cpu().numpy(), bv), t


# ------------------------------------------------------------------------------------------------ streams, graphs, the loop
@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_counts_on(O, bits):
    n = [700, 64, 5000]
    vals, _, _ = tensors(n, F32, 0, 4, 0.1)
    ps, qs = [torch.nn.Parameter(v.clone()) for v in vals], [torch.nn.Parameter(v.clone()) for v in vals]
    lr_a, lr_b = (torch.tensor(1e-3, device=DEV) for _ in range(2))
    a, b = O.MultiAdamW(ps, lr=lr_a, state_bits=bits), O.MultiAdamW(qs, lr=lr_b, state_bits=bits)
    static = [torch.zeros_like(v) for v in vals]
    for p, q, g in zip(ps, qs, static):
        p.grad, q.grad = g, g
    graph, norms = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        a.step(max_norm=1.0)
    for t in range(5):
        for g, new in zip(static, tensors(n, F32, 0, 70 + t)[0]):
            g.copy_(new)
        lr_a.fill_(1e-3 / (t + 1)), lr_b.fill_(1e-3 / (t + 1))
        graph.replay()
        b.step(max_norm=1.0)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), t
        assert torch.equal(a.grad_norm, b.grad_norm)
        assert all(torch.equal(x, y) for x, y in zip(a.flat_moments(), b.flat_moments()))
    a.step(max_norm=1.0), b.step(max_norm=1.0)       # eager again, on the same state
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert float(state_of(a)["step"]) == 6


def test_two_captured_clips_do_not_share_scratch(O):
    gs = [[torch.randn(k, device=DEV) for k in (5000, 70_000)] for _ in range(2)]
    ps = [params_of([torch.zeros_like(g) for g in x], x) for x in gs]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in gs], []
    for graph, p in zip(graphs, ps):
        with torch.cuda.graph(graph):
            outs.append(O.clip_grad_norm_(p, 1.0))
    for t in range(3):
        want = []
        for x in gs:
            for g in x:
                g.normal_(generator=torch.Generator(DEV).manual_seed(t + len(want)))
            want.append(R.norm([np64(g) for g in x]))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, x, w in zip(outs, gs, want):
            assert abs(float(out) - w) <= 1.01 * R.EPS24 * w
            assert abs(R.norm([np64(g) for g in x]) - R.coefficient(w, 1.0) * w) < 1e-6


def test_another_stream(O):
    vals, _, _ = tensors([5000, 70_000], F32, 0, 4, 0.1)
    ps, qs = [torch.nn.Parameter(v.clone()) for v in vals], [torch.nn.Parameter(v.clone()) for v in vals]
    a, b = O.MultiAdamW(ps), O.MultiAdamW(qs)
    side = torch.cuda.Stream()
    for t in range(3):
        gs = [torch.randn(v.shape, device=DEV) for v in vals]
        for p, q, g in zip(ps, qs, gs):
            p.grad, q.grad = g, g.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a.step(max_norm=1.0)
        torch.cuda.current_stream().wait_stream(side)
        b.step(max_norm=1.0)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_the_loop_with_the_conv_vae(O):
    """train_step, FusedStep and fit with MultiAdamW, against FlatAdamW on the same start: the same formulas, so the same losses and
    parameters up to fp32 roundings of the step, which the bf16 weight copies can amplify to their own last place"""
    from vae_amd.train import Config, FusedStep, train_step
    from vae_amd.vae import VAEConv
    conf = Config(kl_weight=1.0, percep_weight=0.0, recon_loss="l1")
    x = torch.rand(8, 3, 16, 16, generator=torch.Generator().manual_seed(2)).to(DEV)
    eps = torch.randn(8, 64, generator=torch.Generator().manual_seed(3)).to(DEV)

    def model():
        torch.manual_seed(1337)
        return VAEConv(3, 3, 64, 0.0, 16).to(DEV).train()
    losses = {}
    for kind in ("flat", "multi", "multi fused", "multi8"):
        m = model()
        opt = O.FlatAdamW(m, lr=1e-3) if kind == "flat" else O.MultiAdamW(m.parameters(), lr=1e-3, state_bits=8 if kind == "multi8" else 32)
        step = FusedStep(m, opt, conf) if kind in ("flat", "multi fused") else (lambda a, e, m=m, opt=opt: train_step(m, opt, a, conf, e))
        losses[kind] = [float(step(x, eps)) for _ in range(4)]
        if kind != "flat":
            assert float(opt.grad_norm) > 0 and [float(e["step"]) for e in opt.state_dict()["state"].values()] == [4.0] * 52
    assert losses["multi"][0] == losses["multi8"][0] == losses["multi fused"][0]
    for kind in ("multi", "multi fused"):
        assert np.allclose(losses[kind], losses["flat"], rtol=2.0 ** -8), losses       # a weight copy's last place: 2^-8 relative
    # a written parameter is seen: the packed weights follow, so a second forward differs from the first
    assert losses["multi"][1] != losses["multi"][0]


def test_the_loop_with_a_unet_of_the_drafts(O):
    from vae_amd import unet
    torch.manual_seed(7)
    m = unet.VAEUnet256(3, 64, 0.0, 16).to(DEV).train()
    x = torch.rand(4, 3, 16, 16, device=DEV)
    ref = [torch.nn.Parameter(p.detach().clone()) for p in m.parameters()]
    a = O.MultiAdamW(m.parameters(), lr=1e-3)
    b = torch.optim.AdamW(ref, lr=1e-3)
    for t in range(2):
        out, mu, lv = m(x)
        a.zero_grad()
        unet.vae_loss_mse(x, out, mu, lv, 1.0).backward()
        for q, p in zip(ref, m.parameters()):
            q.grad = None if p.grad is None else p.grad.detach().clone()
        tn = torch.nn.utils.clip_grad_norm_(ref, 1.0)
        b.step()
        a.step(max_norm=1.0)
        # torch sums in fp32: N terms, pairwise within blocks; its norm is off by some 1e-6 at most
        assert abs(float(a.grad_norm) / float(tn) - 1) < 1e-5
    for p, q in zip(m.parameters(), ref):
        # the clip's 1e-5 changes gradient and root alike and cancels but for eps; the rest are fp32 halves of steps of at most 2 lr
        within(p, np64(q), 10 * R.EPS24 * np.abs(np64(q)) + 2 * 2e-3 * 1e-4)
