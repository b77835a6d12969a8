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
