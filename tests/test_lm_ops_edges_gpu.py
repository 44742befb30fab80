"""GPU: calls of the language-model operators at the edges of what their documentation allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,t", [(0, 5), (2, 0)])
def test_calls_without_steps_carry_gradients(native_lib, b, t):
    """No rows or no steps: every input gets a gradient, of zeros but for what passes the state through."""
    from atlas_rnn_b200 import causal_conv1d, selective_scan
    leaf = lambda *s: torch.randn(*s, device="cuda").requires_grad_()
    x = dict(u=leaf(b, t, 6), delta=leaf(b, t, 6), A=leaf(6, 4), B=leaf(b, t, 4), C=leaf(b, t, 4), D=leaf(6), z=leaf(b, t, 6),
             delta_bias=leaf(6), initial_state=leaf(b, 6, 4))
    out, hT = selective_scan(**x)
    assert out.shape == (b, t, 6) and torch.equal(hT, x["initial_state"])
    (out.sum() + 3 * hT.sum()).backward()
    for k, v in x.items():
        assert torch.equal(v.grad, torch.full_like(v, 3.0 if k == "initial_state" else 0.0)), k
    c = dict(x=leaf(b, t, 6), weight=leaf(6, 1, 4), bias=leaf(6), initial_state=leaf(b, 3, 6))
    y, final = causal_conv1d(**c)
    assert y.shape == (b, t, 6) and torch.equal(final, c["initial_state"])
    (y.sum() + 3 * final.sum()).backward()
    for k, v in c.items():
        assert torch.equal(v.grad, torch.full_like(v, 3.0 if k == "initial_state" else 0.0)), k
    u = leaf(b, t, 6)
    causal_conv1d(u, c["weight"])[0].sum().backward()  # the outputs alone, without a state
    assert torch.equal(u.grad, torch.zeros_like(u))


@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 3)])
def test_distillation_of_no_rows(native_lib, lead):
    from atlas_rnn_b200 import distill_loss
    for reduction, shape in (("none", lead), ("sum", ()), ("mean", ())):
        x = torch.zeros(*lead, 50, device="cuda", requires_grad=True)
        loss = distill_loss(x, torch.zeros(*lead, 4, device="cuda", requires_grad=True),
                            torch.zeros(*lead, 4, dtype=torch.int64, device="cuda"), reduction=reduction)
        assert loss.shape == shape and loss.sum() == 0
        loss.sum().backward()
        assert x.grad.shape == x.shape


@pytest.mark.parametrize("rows,V", [(4, 300), (2, 40000)])
def test_settings_per_row_that_are_nan_give_the_first_token(native_lib, rows, V):
    """As a comparison with a NaN keeps nothing but the first token: in each of the three settings that have NaNs."""
    from atlas_rnn_b200 import sample_tokens
    g = torch.Generator().manual_seed(5)
    l, u = torch.randn(rows, V, generator=g).cuda(), torch.rand(rows, V, generator=g).cuda()
    want = sample_tokens(l, u)
    bad = torch.full((rows,), float("nan"), device="cuda")
    bad[1::2] = 1.0
    want[::2] = l.argmax(-1)[::2]
    assert not torch.equal(sample_tokens(l, u)[::2], want[::2])  # the draw itself is another token
    for name in ("temperature", "top_p", "min_p"):
        x = bad.clone()
        if name == "min_p":
            x[1::2] = 0.0
        assert torch.equal(sample_tokens(l, u, **{name: x}), want), name
