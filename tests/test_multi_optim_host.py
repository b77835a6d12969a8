"""CPU checks of the many-tensor optimizer: what the C entry points and the Python layer refuse (no kernel is launched), sizes of the scratch,
the struct mirrors, and the 8-bit format's own arithmetic in the tests' restatement."""
import ctypes

import numpy as np
import pytest
import torch

import multi_optim_ref as R
from vae_amd import _lib as L
from vae_amd import optim


def job(n=8, param=4096, grad=8192, block=0, slot=0, flags=0):
    return L.MtTensor(param=param, grad=grad, n=n, block=block, slot=slot, flags=flags)


def group(jobs, **kw):
    arr = (L.MtTensor * len(jobs))(*jobs)
    base = dict(state_bits=32, tensors=ctypes.cast(arr, ctypes.c_void_p), count=len(jobs), nslots=len(jobs), exp_avg=4096, exp_avg_sq=8192,
                nblocks=4, steps=4096, scalars=4096, lr=1e-4, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01)
    base.update(kw)
    return (L.MtGroup * 1)(L.MtGroup(**base)), arr


def test_struct_mirrors_have_the_c_layout():
    assert ctypes.sizeof(L.MtTensor) == 40 == optim._JOB.itemsize
    for name, _ in L.MtTensor._fields_:
        assert getattr(L.MtTensor, name).offset == optim._JOB.fields[name][1]
    assert ctypes.sizeof(L.MtGroup) == 24 + 4 * 8 + 8 + 3 * 8 + 5 * 8


def test_partials_cover_every_launch():
    # at most 256 shares over all launches, and one for each launch whose share is smaller than one
    for n in (0, 1, 192, 193, 5000, 65536):
        assert L.call("vae_multi_partials", n) >= 256 + -(-n // 192) + 64 - 1


@pytest.mark.parametrize("bad, match", [
    (dict(n=-1), "n=-1"), (dict(flags=4), "unknown flags"), (dict(grad=None), "gradient is null"), (dict(grad=8194), "not aligned"),
    (dict(grad=8193, flags=2), "not aligned")])
def test_norm_and_clip_refuse(bad, match):
    arr = (L.MtTensor * 1)(job(**bad))
    with pytest.raises(RuntimeError, match=match):
        L.call("vae_multi_grad_norm", arr, 1, 4096, 1.0, 4096, None)
    with pytest.raises(RuntimeError, match=match):
        L.call("vae_multi_clip", arr, 1, 4096, 1.0, 1.0, 4096, None)


def test_norm_and_clip_refuse_scratch_and_counts():
    arr = (L.MtTensor * 1)(job())
    with pytest.raises(RuntimeError, match="null pointer"):
        L.call("vae_multi_grad_norm", arr, 1, None, 1.0, 4096, None)
    with pytest.raises(RuntimeError, match="null pointer"):
        L.call("vae_multi_clip", arr, 1, 4096, 1.0, 1.0, None, None)
    with pytest.raises(RuntimeError, match="out of range"):
        L.call("vae_multi_clip", arr, 65537, 4096, 1.0, 1.0, 4096, None)
    with pytest.raises(RuntimeError, match="out of range"):
        L.call("vae_multi_grad_norm", None, 1, 4096, 1.0, 4096, None)
    for bad in (-1.0, float("nan")):
        with pytest.raises(RuntimeError, match="max_norm"):
            L.call("vae_multi_clip", arr, 1, 4096, 1.0, bad, 4096, None)


@pytest.mark.parametrize("jobs, kw, match", [
    ([job()], dict(state_bits=16), "state_bits"), ([job()], dict(beta1=1.0), "betas"), ([job()], dict(beta2=-0.1), "betas"),
    ([job()], dict(eps=-1.0), "eps"), ([job()], dict(state_bits=8, eps=1e-13, bases=4096), "8-bit moments need"), ([job()], dict(lr=-1.0), "lr"), ([job()], dict(weight_decay=float("nan")), "weight_decay"),
    ([job()], dict(exp_avg=None), "null state"), ([job()], dict(state_bits=8), "null state"), ([job()], dict(exp_avg=4100), "16-byte"),
    ([job()], dict(steps=None), "step counts"), ([job()], dict(steps=4100), "not aligned"), ([job()], dict(lr_dev=4098), "not aligned"),
    ([job()], dict(nslots=65537), "nslots"), ([job()], dict(nslots=-1), "nslots"), ([job(n=1025)], {}, "reaches behind"), ([job(block=4)], {}, "reaches behind"),
    ([job(slot=1)], {}, "slot"), ([job(param=None)], {}, "parameter is null"), ([job(param=4098)], {}, "not aligned"),
    ([job(flags=1)], {}, "remainder"), ([job()], dict(struct_size=8), "struct_size")])
def test_step_refuses(jobs, kw, match):
    size = kw.pop("struct_size", None)
    g, arr = group(jobs, **kw)
    if size:
        g[0].struct_size = size
    with pytest.raises(RuntimeError, match=match):
        L.call("vae_multi_adamw_step", g, 1, 4096, 1.0, 1.0, 4096, None)


def test_step_refuses_its_own_arguments():
    g, arr = group([job()])
    for n in (0, 65):
        with pytest.raises(RuntimeError, match="ngroups"):
            L.call("vae_multi_adamw_step", g, n, 4096, 1.0, 1.0, 4096, None)
    with pytest.raises(RuntimeError, match="NaN"):
        L.call("vae_multi_adamw_step", g, 1, 4096, 1.0, float("nan"), 4096, None)
    with pytest.raises(RuntimeError, match="buffer"):
        L.call("vae_multi_adamw_step", g, 1, None, 1.0, 1.0, 4096, None)


def test_moment_conversions_refuse():
    for name, args in (("vae_moments8_unpack", (4096, 4096, 4096, 4096, 4096, -1, 0, None)), ("vae_moments8_pack", (4096, 4096, 4096, 4096, 4096, -1, None))):
        with pytest.raises(RuntimeError, match="nblocks"):
            L.call(name, *args)
    with pytest.raises(RuntimeError, match="null"):
        L.call("vae_moments8_unpack", 4096, None, 4096, 4096, 4096, 1, 0, None)
    with pytest.raises(RuntimeError, match="16-byte"):
        L.call("vae_moments8_pack", 4096, 4100, 4096, 4096, 4096, 1, None)
    L.call("vae_moments8_pack", None, None, None, None, None, 0, None)       # nothing to do: nothing is looked at
    with pytest.raises(RuntimeError, match="out is null"):
        L.call("vae_multi_master", (L.MtTensor * 1)(job()), 1, None, None, 1, None)
    with pytest.raises(RuntimeError, match="remainder"):
        L.call("vae_multi_master", (L.MtTensor * 1)(job(flags=3)), 1, None, 4096, 1, None)
    with pytest.raises(RuntimeError, match="reaches behind"):
        L.call("vae_multi_master", (L.MtTensor * 1)(job(n=257)), 1, None, 4096, 1, None)


def cpu_param(*shape, dtype=torch.float32):
    p = torch.nn.Parameter(torch.randn(*shape).to(dtype))
    p.grad = torch.randn_like(p)
    return p


def test_python_layer_refuses_on_the_cpu():
    p = cpu_param(4, 4)
    with pytest.raises(RuntimeError, match="MI355X only"):
        optim.MultiAdamW([p])
    with pytest.raises(RuntimeError, match="MI355X only"):
        optim.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="MI355X only"):
        optim.grad_norm(p)
    with pytest.raises(TypeError, match="float64"):
        optim.MultiAdamW([torch.nn.Parameter(torch.randn(3).double())])
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_([p], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_([p], float("nan"))
    with pytest.raises(ValueError, match="norm_type"):
        optim.clip_grad_norm_([p], 1.0, norm_type=1.0)
    p.grad = None
    assert float(optim.clip_grad_norm_([p], 1.0)) == 0.0 == float(optim.grad_norm([p]))


@pytest.mark.parametrize("kw, match", [
    (dict(lr=-1.0), "lr"), (dict(betas=(1.0, 0.9)), "betas"), (dict(betas=(0.9, -0.1)), "betas"), (dict(eps=-1e-8), "eps"),
    (dict(weight_decay=-1.0), "weight_decay"), (dict(state_bits=16), "state_bits"), (dict(lr=torch.tensor(1e-3)), "on the GPU"),
    (dict(lr=float("nan")), "lr"), (dict(eps=0.0, state_bits=8), "8-bit moments need")])
def test_python_layer_refuses_hyperparameters(kw, match):
    with pytest.raises(ValueError, match=match):
        optim.MultiAdamW([cpu_param(4)], **kw)


def test_dense_looks_at_gaps_not_at_the_order_of_dims():
    x = torch.zeros(4, 6, 5, 3)
    assert optim._dense(x) and optim._dense(x.permute(2, 0, 3, 1)) and optim._dense(x.to(memory_format=torch.channels_last))
    assert not optim._dense(x[:, ::2]) and not optim._dense(x[:, :3]) and not optim._dense(torch.zeros(1).expand(5))
    assert optim._dense(torch.zeros(())) and optim._dense(torch.zeros(1, 7)[:, :1]) and optim._dense(torch.zeros(0, 3))


# ------------------------------------------------------------------------------------------------ the 8-bit format itself
def test_levels_are_the_top_bits_of_fp32():
    rng = np.random.default_rng(0)
    x = np.abs(np.concatenate([rng.standard_normal(1000), 10.0 ** rng.uniform(-37, 38, 1000)])).astype(np.float32)
    lev, part = R._levels(x.astype(np.float64))
    bits = x.view(np.uint32).astype(np.int64)
    assert np.array_equal(lev, bits >> 20) and np.array_equal((part * 2 ** 20).astype(np.int64), bits & 0xFFFFF)
    assert np.array_equal(R.level_value(lev).astype(np.float32).view(np.uint32), ((bits >> 20) << 20).astype(np.uint32))


def test_every_code_survives_a_round_trip():
    for codes, signed in ((127, True), (254, False)):
        q = np.arange(codes + 1, dtype=np.int64)
        if signed:
            q = np.concatenate([q, np.arange(129, 256)])
        q = np.resize(q, 256).astype(np.uint8)
        for base in (0, 1, 700, 0x7F7 - codes):
            x = R.unpack(q, base, signed)
            for d in (0, 1 << 19, (1 << 20) - 1):
                back, b = R.pack(x, np.full(256, d), codes, signed)
                lowest = R.level_value(base + 1)
                # a subnormal level is not what a mantissa and an exponent describe: base 0 stops at the normal numbers
                ok = (np.abs(x) >= 2.0 ** -126) | (x == 0) if base == 0 else np.ones(256, bool)
                assert b == base and np.array_equal(back[ok], q[ok]), (codes, base, d, lowest)


def test_rounding_of_a_constant_is_unbiased_in_time():
    """mean over T steps of the rounded value of a constant.  u_t = frac(t * rate + c) is an additive recurrence; the share of t with
    u_t >= 1 - f is f up to the sequence's discrepancy, which for sqrt 2 and sqrt 3 (partial quotients at most 2) is below 3 (ln T + 1) / T;
    a level is at most 1/8 of the value wide."""
    T = 4096
    tol = 3 * (np.log(T) + 1) / T / 8
    for rate, codes, signed in ((R.RATE_M, 127, True), (R.RATE_V, 254, False)):
        for x in (1.0 + 1 / 77, 0.3, 1.5e-3, 0.02):
            lev, part = R._levels(np.array([x]))
            for i in (0, 1, 77):
                d = np.array([int(((i * R.A + t * rate) & 0xFFFFFFFF) >> 12) for t in range(1, T + 1)])
                up = part[0] * 2 ** 20 + d >= 2 ** 20
                mean = np.mean(R.level_value(lev[0] + up))
                assert abs(mean - x) <= tol * x, (rate, x, i, mean)


def test_second_moment_never_becomes_zero_and_first_is_kept_small():
    x = np.zeros(256)
    x[0], x[1], x[2] = 1.0, 1e-20, 2.0 ** -40
    q, b = R.pack(x, np.zeros(256, np.int64), 254, False)
    assert q[0] == 254 and q[1] == 1 and q[2] == 1 and not q[3:].any()
    q, b = R.pack(x, np.full(256, (1 << 20) - 1), 127, True)
    assert q[0] == 127 and q[1] == 0 and q[2] == 0


def test_second_moment_decays_where_nearest_would_stand_still():
    """no gradient, beta2 = 0.999: a step takes 0.001 off the value, which is between 9/1000 and 16/1000 of the level below it, and the value
    falls a level where the dither's fraction is below that share (seen from the far end).  For sqrt 2 the multiples of q = 2, 5, 12, 29, 70,
    169 come nearest to whole numbers, to within 0.172, 0.071, 0.029, 0.012, 0.0051, 0.0021.  Two falls are therefore at least 29
    steps apart (no smaller multiple comes within 0.016), and any 169 steps hit every interval longer than 0.0051 + 0.0021 < 0.009.  So 500
    steps take between 2 and 18 levels (exactly 5.8 in 64 bits); rounding to nearest takes none."""
    n = 256
    x = np.float32(10.0) ** np.random.default_rng(1).uniform(-4, 0, n).astype(np.float32)
    for nearest, low, high in ((False, 2, 18), (True, 0, 0)):
        q, b = R.pack_tensor(x, 0, 0, 254, False, nearest=True)
        start = R._levels(R.unpack_tensor(q, b, False))[0]
        for t in range(1, 501):
            v = R.unpack_tensor(q, b, False).astype(np.float32) * np.float32(0.999)
            q, b = R.pack_tensor(v, t, R.RATE_V, 254, False, nearest=nearest)
        fell = start - R._levels(R.unpack_tensor(q, b, False))[0]
        assert fell.min() >= low and fell.max() <= high, (nearest, fell.min(), fell.max())


# ------------------------------------------------------------------------------------------------ the native walk over the lists (on host tensors)
def step_table(params, layout=None):
    n = len(params)
    if layout is None:
        layout = np.array([[p.numel(), 10 * k, k, int(p.dtype is torch.bfloat16)] for k, p in enumerate(params)], np.int64).reshape(n, 4)
    jobs = np.zeros(n, optim._JOB)
    return L.host().collect_step(params, jobs, layout, -1), jobs


def test_the_walk_fills_the_table_and_advances_versions():
    ps = [cpu_param(3, 4), cpu_param(7, dtype=torch.bfloat16), cpu_param(0), cpu_param(())]
    ps.insert(1, torch.nn.Parameter(torch.zeros(5)))       # without a gradient
    before = [p._version for p in ps]
    n, jobs = step_table(ps)
    have = [k for k, p in enumerate(ps) if p.grad is not None]
    assert n == 4 and [p._version - b for p, b in zip(ps, before)] == [1, 0, 1, 1, 1]
    for row, k in zip(jobs, have):
        p = ps[k]
        assert (row["param"], row["grad"], row["n"], row["block"], row["slot"]) == (p.data_ptr(), p.grad.data_ptr(), p.numel(), 10 * k, k)
        assert row["flags"] == (3 if p.dtype is torch.bfloat16 else 0) and row["reserved"] == 0
    table = np.zeros(5, optim._JOB)
    assert L.host().collect_grads(ps, table, -1, False) == 4
    assert list(table["grad"][:4]) == list(jobs["grad"][:4]) and list(table["flags"][:4]) == [0, 2, 0, 0] and list(table["n"][:4]) == [12, 7, 0, 1]


def test_the_walk_over_all_parameters_reads_only():
    ps = [cpu_param(3, 4), torch.nn.Parameter(torch.zeros(5)), cpu_param(7, dtype=torch.bfloat16)]
    layout = np.array([[12, 0, 0, 0], [5, 1, 1, 0], [7, 2, 2, 1]], np.int64)
    jobs, before = np.zeros(3, optim._JOB), [p._version for p in ps]
    assert L.host().collect_params(ps, jobs, layout, -1) == 3 and [p._version for p in ps] == before
    assert list(jobs["param"]) == [p.data_ptr() for p in ps] and list(jobs["flags"]) == [0, 0, 3] and list(jobs["block"]) == [0, 1, 2]
    assert L.host().collect_params([ps[0], strided()], jobs, np.array([[12, 0, 0, 0], [24, 1, 1, 0]], np.int64), -1) == -1


def test_the_walk_leaves_everything_else_to_the_general_way():
    def one(p, **kw):
        row = dict(n=p.numel(), flags=int(p.dtype is torch.bfloat16))
        row.update(kw)
        before = p._version
        n, _ = step_table([cpu_param(2), p], np.array([[2, 0, 0, 0], [row["n"], 1, 1, row["flags"]]], np.int64))
        assert n == -1 and p._version == before
    p = cpu_param(4, 6)
    one(p, n=23)                                             # another size than the state was made for
    one(p, flags=1)                                          # another type
    one(strided())
    q = cpu_param(4, 6)
    q.grad = torch.zeros(6, 4).t()
    one(q)                                                   # the gradient in another order
    q.grad = torch.zeros(1, 1).expand(4, 6)
    one(q)
    h = cpu_param(4, dtype=torch.float16)
    one(h)
    s = torch.nn.Parameter(torch.zeros(3, 3))
    s.grad = torch.eye(3).to_sparse()
    one(s)
    c = cpu_param(4)
    assert L.host().collect_step([c], np.zeros(1, optim._JOB), np.array([[4, 0, 0, 0]], np.int64), 0) == -1       # not on that GPU
    assert L.host().collect_step(["no tensor"], np.zeros(1, optim._JOB), np.zeros((1, 4), np.int64), -1) == -1
    assert L.host().collect_step([], np.zeros(0, optim._JOB), np.zeros((0, 4), np.int64), -1) == 0


def strided():
    p = torch.nn.Parameter(torch.zeros(6, 4).t())
    p.grad = torch.zeros(6, 4).t()
    return p


def test_the_walk_finds_gradients_that_overlap():
    flat = torch.zeros(20)
    ps = [torch.nn.Parameter(torch.zeros(8)) for _ in range(2)]
    for shift, ok in ((8, True), (7, False), (0, False)):
        ps[0].grad, ps[1].grad = flat[:8], flat[shift:shift + 8]
        before = flat._version
        n = L.host().collect_grads(ps, np.zeros(2, optim._JOB), -1, True)
        assert n == (2 if ok else -1) and (flat._version > before) == ok
        assert L.host().collect_grads(ps, np.zeros(2, optim._JOB), -1, False) == 2       # reading them is no matter


def test_the_walk_refuses_tables_that_are_too_short():
    ps = [cpu_param(2), cpu_param(2)]
    with pytest.raises(ValueError, match="shorter"):
        L.host().collect_step(ps, np.zeros(1, optim._JOB), np.zeros((2, 4), np.int64), -1)
    with pytest.raises(ValueError, match="shorter"):
        L.host().collect_step(ps, np.zeros(2, optim._JOB), np.zeros((1, 4), np.int64), -1)
    with pytest.raises(ValueError, match="shorter"):
        L.host().collect_grads(ps, np.zeros(1, optim._JOB), -1, False)
    with pytest.raises((TypeError, BufferError, ValueError)):
        L.host().collect_grads(ps, 7, -1, False)


def test_the_extension_is_refused_under_another_torch(monkeypatch):
    L.host()
    monkeypatch.setattr(L, "_host", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    with pytest.raises(RuntimeError, match="rebuild"):
        L.host()
    monkeypatch.setattr(L, "HOST_PATH", "/nowhere/_host.so")
    with pytest.raises(RuntimeError, match="not found"):
        L.host()


def test_each_thread_has_a_table_of_its_own():
    import threading
    t, seen = optim._tables, []
    t.room(100)
    mine = t.addr
    assert len(t.jobs) >= 100 and t.jobs.ctypes.data == mine and t.room(3) is t.jobs

    def other():
        seen.append((t.room(10).ctypes.data, t.addr))
    th = threading.Thread(target=other)
    th.start()
    th.join()
    assert seen[0][0] == seen[0][1] != mine and t.addr == mine
