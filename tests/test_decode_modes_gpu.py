"""GPU: memory_recurrence of one token under forward-mode differentiation (refused, as for longer calls) and
torch.jit.trace (the call's results, by the kernels of longer calls: within fp32 rounding of the decode kernel's)."""
import warnings

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from atlas_rnn_b200 import memory_recurrence
from atlas_rnn_b200.workloads import Workload, make_inputs
from tests.helpers import TOL_F32, rel_l2

pytestmark = pytest.mark.gpu
NAMES = ("k", "q", "v", "lr", "decay", "beta", "S0", "Z0")


def inputs(seed):
    w = Workload("one", 2, 3, 1, 32, 32, 32, 1, "none", "off", 1, True, torch.float32, 0)
    inp = make_inputs(w, seed=seed, device="cuda", state_scale=0.1)
    return [inp[n] for n in NAMES]


def call(k, q, v, lr, decay, beta, S0, Z0):
    return memory_recurrence(k, q, v, lr, decay, beta, S_ref=S0, S0=S0, Z0=Z0)[:3]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_of_one_token_is_refused(native_lib, name):
    x = inputs(1)
    with forward_ad.dual_level(), torch.no_grad():
        call(*x)  # no tangent: runs
        at = NAMES.index(name)
        x[at] = forward_ad.make_dual(x[at], torch.ones_like(x[at]))
        with pytest.raises(NotImplementedError):
            call(*x)


def test_traced_one_token(native_lib):
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        m = torch.jit.trace(call, tuple(inputs(1)))
    for got, want in zip(m(*inputs(2)), call(*inputs(2))):
        assert rel_l2(got, want) <= TOL_F32
