"""More CPU checks of the many-tensor optimizer: calls that have to be refused before anything is launched or written."""
import numpy as np
import pytest
import torch

from test_multi_optim_host import group, job
from vae_amd import _lib as L
from vae_amd import optim


@pytest.mark.parametrize("max_norm, norm", [(1.0, 4096), (-1.0, None)])
@pytest.mark.parametrize("slot", [1, 60000])
def test_step_refuses_the_slot_of_an_empty_tensor(max_norm, norm, slot):
    """an empty tensor's step count is advanced too, so its slot has to be one of the group's"""
    g, arr = group([job(), job(n=0, param=None, grad=None, slot=slot)], nslots=1)
    with pytest.raises(RuntimeError, match=f"tensor 1 has slot {slot} of 1"):
        L.call("vae_multi_adamw_step", g, 1, 4096, 1.0, max_norm, norm, None)


# ------------------------------------------------------------------------------------------------ a group's tensors (on host tensors)
def held(monkeypatch, params, bits=32):
    """the state of a param group, on the host"""
    monkeypatch.setattr(L, "current_stream", lambda device=None: 0)
    st = optim._GroupState(params, bits)
    st.index = -1
    return st


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_parameter_in_another_memory_order_than_its_state_is_refused(monkeypatch, bits, dtype):
    """the state of a channels_last or transposed parameter is in that order: element k of it belongs to another element of the contiguous one"""
    for make in (lambda: torch.randn(4, 6, 3, 3).to(dtype).to(memory_format=torch.channels_last), lambda: torch.randn(7, 5).to(dtype).t()):
        p, q = torch.nn.Parameter(make()), torch.nn.Parameter(torch.zeros(3))
        st = held(monkeypatch, [q, p], bits)
        p.grad, q.grad = torch.randn_like(p), torch.zeros(3)
        assert st.collect()[0] == 2
        p.data = p.data.contiguous()
        p.grad = torch.zeros(p.shape, dtype=dtype)
        with pytest.raises(RuntimeError, match="make a new optimizer"):
            st.collect()
        assert L.host().collect_params(st.params, np.zeros(2, optim._JOB), st.layout, -1) == -1       # what flat_master asks first
        p.grad = None       # without a gradient it is not stepped
        assert st.collect()[0] == 1


def test_lists_are_compared_by_identity():
    """a group's list as it is now against the tensors the state was made for"""
    ps = [torch.nn.Parameter(torch.zeros(4)) for _ in range(3)]
    same, new = L.host().same_tensors, torch.nn.Parameter(torch.zeros(4))
    assert same(list(ps), ps) and same(ps, ps) and same([], [])
    for now in ([ps[0], new, ps[2]], [ps[1], ps[0], ps[2]], ps[:2], [*ps, new], [], [ps[0], None, ps[2]]):
        assert not same(now, ps)
    assert same(tuple(ps), ps)       # any sequence will do
    with pytest.raises(TypeError):
        same(3, ps)


def test_moments_unpack_refuses_unknown_flags():
    for flags in (2, 4, -1, 257 + 2):
        with pytest.raises(RuntimeError, match="unknown flags"):
            L.call("vae_moments8_unpack", 4096, 4096, 4096, 4096, 4096, 1, flags, None)


def test_strides_of_dims_of_one_element_do_not_matter(monkeypatch):
    """a 1x1 convolution in channels_last and contiguous: the same order of elements, other strides"""
    x = torch.randn(8, 6, 1, 1)
    a, b = x.to(memory_format=torch.channels_last), x.clone()
    assert a.stride() != b.stride()
    st = held(monkeypatch, [torch.nn.Parameter(a)], 8)
    codes, bases = torch.zeros(48, dtype=torch.uint8), torch.zeros(1, dtype=torch.int16)
    e = {"step": 1, "exp_avg_q": codes, "exp_avg_sq_q": codes, "exp_avg_base": bases, "exp_avg_sq_base": bases, "stride": b.stride()}
    optim.MultiAdamW._check_entry(st, 0, e)
    other = held(monkeypatch, [torch.nn.Parameter(torch.randn(6, 8).t())], 8)
    for stride in ((6, 1), (1, 6), (8, 1)):
        with pytest.raises(ValueError, match="order of strides"):
            optim.MultiAdamW._check_entry(other, 0, {**e, "stride": stride})
    optim.MultiAdamW._check_entry(other, 0, {**e, "stride": (1, 8)})


# ------------------------------------------------------------------------------------------------ the build
def test_the_library_builds_where_torch_is_not_installed(tmp_path):
    """_host.so needs torch's headers; without them make says so and goes on, as libvae_hip.so needs none"""
    import os
    import subprocess
    src = os.path.join(os.path.dirname(L.__file__), "csrc")
    out = tmp_path / "_host.so"
    run = lambda python: subprocess.run(["make", "-C", src, f"PYTHON={python}", f"HOST_OUT={out}", str(out)], capture_output=True, text=True)  # noqa: E731
    r = run("false")
    assert r.returncode == 0 and not out.exists() and "torch" in r.stdout, r.stdout + r.stderr


def test_the_walk_takes_the_address_that_may_be_written():
    """a lazily cloned tensor shares its memory until one of the two is written: what a launch will write has to be its own by then"""
    a, b = torch.ones(64), torch.ones(64)
    p = torch.nn.Parameter(torch._lazy_clone(a))
    p.grad = torch._lazy_clone(b)
    shared = torch._C._data_address(a), torch._C._data_address(b)
    jobs = np.zeros(1, optim._JOB)
    assert L.host().collect_step([p], jobs, np.array([[64, 0, 0, 0]], np.int64), -1) == 1
    assert jobs["param"][0] != shared[0] and jobs["grad"][0] == shared[1]       # the gradient is only read
    assert L.host().collect_grads([p], jobs, -1, False) == 1 and jobs["grad"][0] == shared[1]
    assert L.host().collect_grads([p], jobs, -1, True) == 1 and jobs["grad"][0] != shared[1]
