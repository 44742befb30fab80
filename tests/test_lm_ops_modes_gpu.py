"""GPU: the language-model operators under torch's other ways of calling a function: forward-mode differentiation is
refused, as by the package's other operators."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def rand(*shape, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


def scan_inputs(b, t, d, n, seed, dtype=torch.float32):
    return dict(u=rand(b, t, d, seed=seed, dtype=dtype), delta=rand(b, t, d, seed=seed + 1, dtype=dtype),
                A=-rand(d, n, seed=seed + 2).abs(), B=rand(b, t, n, seed=seed + 3, dtype=dtype),
                C=rand(b, t, n, seed=seed + 4, dtype=dtype), z=rand(b, t, d, seed=seed + 5, dtype=dtype),
                initial_state=rand(b, d, n, seed=seed + 6))


@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("name", ["u", "delta", "A", "B", "C", "z", "initial_state"])
def test_forward_mode_of_the_scan_is_refused(native_lib, t, name):
    from atlas_rnn_b200 import selective_scan
    x = scan_inputs(2, t, 6, 4, seed=1)
    with forward_ad.dual_level():
        selective_scan(**x, delta_softplus=True)  # no tangent: runs
        x[name] = forward_ad.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises(NotImplementedError):
            selective_scan(**x, delta_softplus=True)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            selective_scan(**x, delta_softplus=True)


@pytest.mark.parametrize("t", [1, 40])
@pytest.mark.parametrize("name", ["x", "weight", "bias", "initial_state"])
def test_forward_mode_of_the_convolution_is_refused(native_lib, t, name):
    from atlas_rnn_b200 import causal_conv1d
    x = dict(x=rand(2, t, 6, seed=1), weight=rand(6, 4, seed=2), bias=rand(6, seed=3), initial_state=rand(2, 3, 6, seed=4))
    with forward_ad.dual_level():
        causal_conv1d(**x, activation="silu")
        x[name] = forward_ad.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises(NotImplementedError):
            causal_conv1d(**x, activation="silu")
        with torch.no_grad(), pytest.raises(NotImplementedError):
            causal_conv1d(**x, activation="silu")


@pytest.mark.parametrize("t", [1, 40])
def test_dual_level_keeps_the_bits(native_lib, t):
    from atlas_rnn_b200 import causal_conv1d, selective_scan
    x = scan_inputs(2, t, 6, 4, seed=2)
    want = *selective_scan(**x, delta_softplus=True), *causal_conv1d(x["u"], x["A"])
    with forward_ad.dual_level():
        got = *selective_scan(**x, delta_softplus=True), *causal_conv1d(x["u"], x["A"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
