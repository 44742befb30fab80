"""CPU: the language-model operators' autograd functions check what they are given themselves: a traced call runs them alone,
on the inputs of its own run, and nothing that is no row of a CUDA tensor may reach a kernel."""
import pytest
import torch

from atlas_rnn_b200.distill import DistillLossFn
from atlas_rnn_b200.sampling import SampleTokensFn
from atlas_rnn_b200.selective_scan import CausalConv1dFn, SelectiveScanFn

Z = torch.zeros


def scan(**change):
    x = dict(u=Z(2, 3, 6), delta=Z(2, 3, 6), A=Z(6, 4), B=Z(2, 3, 4), C=Z(2, 3, 4), D=None, z=None, bias=None, h0=None,
             lengths=None, softplus=False, chunk=0)
    SelectiveScanFn.apply(*{**x, **change}.values())


def conv(**change):
    x = dict(x=Z(2, 3, 6), w=Z(6, 4), bias=None, init=None, lengths=None, activation=None)
    CausalConv1dFn.apply(*{**x, **change}.values())


def sample(**change):
    x = dict(logits=Z(2, 5), noise=Z(2, 5), temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    SampleTokensFn.apply(*{**x, **change}.values())


def distill(**change):
    x = dict(logits=Z(2, 5), values=Z(2, 3), indices=Z(2, 3, dtype=torch.int64), temperature=1.0)
    DistillLossFn.apply(*{**x, **change}.values())


@pytest.mark.parametrize("call", [scan, conv, sample, distill])
def test_tensors_of_the_host_are_refused(call):
    with pytest.raises(RuntimeError, match="must be on a CUDA device"):
        call()


@pytest.mark.parametrize("call, change, error", [
    (scan, dict(delta=Z(1, 3, 6)), ValueError),
    (scan, dict(B=Z(2, 3, 4, dtype=torch.bfloat16)), TypeError),
    (scan, dict(A=Z(6, 65), B=Z(2, 3, 65), C=Z(2, 3, 65)), ValueError),
    (conv, dict(w=Z(5, 4)), ValueError),
    (conv, dict(init=Z(2, 2, 6)), ValueError),
    (sample, dict(noise=Z(1, 5)), ValueError),
    (sample, dict(top_k=Z(1, dtype=torch.int64)), ValueError),
    (distill, dict(values=Z(1, 3)), ValueError),
    (distill, dict(indices=Z(1, 3, dtype=torch.int64)), ValueError),
    (distill, dict(indices=Z(2, 2, dtype=torch.int64)), ValueError),
    (distill, dict(indices=Z(2, 3)), TypeError),
    (distill, dict(logits=Z(2, 5, dtype=torch.float16)), TypeError),
    (distill, dict(values=Z(2, 1025), indices=Z(2, 1025, dtype=torch.int64)), ValueError),
])
def test_other_sizes_and_types_are_refused(call, change, error):
    with pytest.raises(error, match="atlas_rnn_b200"):
        call(**change)


@pytest.mark.parametrize("settings", [dict(top_k=-1), dict(top_p=float("nan")), dict(top_p=1.5), dict(top_p=-0.5),
                                      dict(top_k=5, min_p=2.0), dict(top_k=0.5)])
def test_generate_refuses_settings_out_of_range(settings, monkeypatch):
    import atlas_rnn_b200 as A
    m = A.RNNMemoryTransformer(num_tokens=8, dim=8, depth=1, heads=1, dim_head=8)
    monkeypatch.setattr(m, "forward", lambda x, **_: (Z(*x.shape, 8), None, None))
    with pytest.raises((ValueError, TypeError), match="top_k|top_p|min_p|integer"):
        m.generate(Z(1, 3, dtype=torch.int64), max_length=4, **settings)
