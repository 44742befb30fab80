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


def growth(dt, A, n, T, live, dtype=torch.float64, h0=None):
    """One channel group of states that grow: delta dt [T], A > 0, inputs u only at the steps `live`."""
    g = torch.Generator().manual_seed(3)
    pos = lambda *s: 0.5 + torch.rand(*s, generator=g, dtype=dtype)
    u = torch.zeros(1, T, 5, dtype=dtype)
    u[:, live] = pos(1, len(live), 5)
    x = dict(u=u, delta=dt.to(dtype)[None, :, None].expand(1, T, 5).contiguous(), A=torch.full((5, n), A, dtype=dtype),
             B=pos(1, T, n), C=pos(1, T, n), initial_state=h0)
    return {k: None if v is None else v.float().double() for k, v in x.items()}


def steps(x):
    """The recurrence in float64, one step after another."""
    h = torch.zeros(1, 5, x["A"].shape[1], dtype=torch.float64) if x["initial_state"] is None else x["initial_state"]
    out = []
    for t in range(x["u"].shape[1]):
        dt = x["delta"][:, t, :, None]
        h = torch.exp(dt * x["A"]) * h + dt * x["u"][:, t, :, None] * x["B"][:, t, None]
        out.append((h * x["C"][:, t, None]).sum(-1))
    return torch.stack(out, 1), h


def scan(x, chunk):
    from atlas_rnn_b200 import selective_scan
    return selective_scan(**{k: None if v is None else v.float().cuda() for k, v in x.items()}, chunk=chunk)


@pytest.mark.parametrize("n", [3, 16])
def test_growing_states_whose_factor_over_a_chunk_overflows(native_lib, n):
    """e^(dt A) = e^4 a step: e^128, beyond fp32, over a chunk of 32, whose entering state is 0 (inputs in the last 8 steps
    alone). All terms are positive. A step's factor is off by at most 2^-22 (the hardware's exp2) + 4 2^-23 (the roundings of
    its argument) < 2^-20, over 7 steps, and the sums by n 2^-24: 2^-16 covers both."""
    x = growth(torch.full((96,), 4.0), 1.0, n, 96, list(range(88, 96)))
    out, hT = steps(x)
    for chunk in (0, 32, 64, 96):
        got = scan(x, chunk)
        torch.testing.assert_close(got[0].double().cpu(), out, rtol=2.0 ** -16, atol=0)
        torch.testing.assert_close(got[1].double().cpu(), hT, rtol=2.0 ** -16, atol=0)


def test_growing_gradients_whose_factor_over_a_chunk_overflows(native_lib):
    """The same backwards: outputs are used in the first 8 steps, and no gradient enters from behind."""
    x = growth(torch.full((96,), 4.0), 1.0, 3, 96, [])
    x["u"][:, 88:] = 1.0
    leaf = {k: None if v is None else v.clone().requires_grad_() for k, v in x.items()}
    steps(leaf)[0][:, :8].sum().backward()
    from atlas_rnn_b200 import selective_scan
    for chunk in (0, 32, 64, 96):
        mine = {k: None if v is None else v.float().cuda().requires_grad_() for k, v in x.items()}
        selective_scan(**mine, chunk=chunk)[0][:, :8].sum().backward()
        for k, v in leaf.items():
            if v is not None:
                torch.testing.assert_close(mine[k].grad.double().cpu(), v.grad, rtol=2.0 ** -16, atol=0, msg=lambda m: f"{k}: {m}")


def test_a_tiny_state_that_grows_by_more_than_the_largest_number(native_lib):
    """A chunk's factor of e^92.8 = 2^133.9 overflows; times the state of 1.2e-37 it does not. dt A is added over 32 steps
    and multiplied by log2(e), 6 roundings of 2^-24 of 133.9 ln 2 = 93 at most: 4e-5; step by step as much. 2^-13."""
    dt = torch.full((64,), 2.9)
    dt[32:] = 0.0
    x = growth(dt, 1.0, 3, 64, [], h0=torch.full((1, 5, 3), 1.2e-37, dtype=torch.float64))
    out, hT = steps(x)
    for chunk in (32, 64):
        got = scan(x, chunk)
        torch.testing.assert_close(got[0][:, 32:].double().cpu(), out[:, 32:], rtol=2.0 ** -13, atol=0)
        torch.testing.assert_close(got[1].double().cpu(), hT, rtol=2.0 ** -13, atol=0)


def test_more_groups_than_a_grid_is_high(native_lib):
    """70000 groups of one channel: gradients of B and C against float64. Sums of 1 channel over at most 3 steps: products
    of up to 6 factors each rounded, exponentials off by 2^-20; 2^-17 of the largest term covers them."""
    from atlas_rnn_b200 import selective_scan
    g = torch.Generator().manual_seed(0)
    b, t, d, n = 1, 3, 70000, 2
    rn = lambda *s: torch.randn(*s, generator=g)
    x = dict(u=rn(b, t, d), delta=rn(b, t, d).abs(), A=-rn(d, n).abs(), B=rn(b, t, d, n), C=rn(b, t, d, n))
    ref = {k: v.double().requires_grad_() for k, v in x.items()}
    h, out = 0, []
    for i in range(t):
        dt = ref["delta"][:, i, :, None]
        h = torch.exp(dt * ref["A"]) * h + dt * ref["u"][:, i, :, None] * ref["B"][:, i]
        out.append((h * ref["C"][:, i]).sum(-1))
    torch.stack(out, 1).sum().backward()
    mine = {k: v.cuda().requires_grad_() for k, v in x.items()}
    got = selective_scan(**mine)[0]
    got.sum().backward()
    torch.testing.assert_close(got.double().cpu(), torch.stack(out, 1), rtol=0, atol=2.0 ** -17 * 100)
    for k, v in ref.items():
        torch.testing.assert_close(mine[k].grad.double().cpu(), v.grad, rtol=0, atol=2.0 ** -17 * v.grad.abs().max().item(),
                                   msg=lambda m: f"{k}: {m}")


def test_short_chunks_of_a_long_row(native_lib):
    """More chunks than a grid is high (65535). dt A = -1 a step: what a state was 64 steps ago is left by e^-64, so the last
    steps are those of a scan of the last 256 alone, bit for bit up to the cut's roundings (2^-20 a step, 2^-17 in all)."""
    from atlas_rnn_b200 import selective_scan
    g = torch.Generator(device="cuda").manual_seed(0)
    T = 65536 * 32 + 5
    pos = lambda *s: 0.5 + torch.rand(*s, device="cuda", generator=g)
    x = dict(u=pos(1, T, 2), delta=torch.ones(1, T, 2, device="cuda"), B=pos(1, T, 1), C=pos(1, T, 1))
    A = -torch.ones(2, 1, device="cuda")
    tail = {k: v[:, -256:].clone().requires_grad_() for k, v in x.items()}
    want, hT = selective_scan(A=A, **tail, chunk=256)
    (want[:, 64:].sum() + hT.sum()).backward()
    x = {k: v.requires_grad_() for k, v in x.items()}
    got, last = selective_scan(A=A, **x, chunk=32)
    (got[:, -192:].sum() + last.sum()).backward()
    torch.testing.assert_close(got[:, -192:], want[:, 64:], rtol=2.0 ** -17, atol=0)
    torch.testing.assert_close(last, hT, rtol=2.0 ** -17, atol=0)
    for k, v in tail.items():
        torch.testing.assert_close(x[k].grad[:, -192:], v.grad[:, 64:], rtol=2.0 ** -17, atol=2.0 ** -17 * v.grad.abs().max().item())


def test_generate_passes_every_filter_on(native_lib):
    """At temperature 1, each filter alone leaves the most likely token; and with all of them the tokens are those of a loop
    over sample_tokens with the same uniforms."""
    import atlas_rnn_b200 as A
    torch.manual_seed(0)
    m = A.RNNMemoryTransformer(num_tokens=64, dim=32, depth=1, heads=1, dim_head=32, omega_window=2).cuda()
    prompt = torch.randint(0, 64, (3, 5), device="cuda")
    greedy = m.generate(prompt, max_length=20, temperature=0.0)
    free = dict(max_length=20, temperature=1.0, min_p=0.0)
    assert not torch.equal(m.generate(prompt, **free, top_k=63), greedy)
    assert torch.equal(m.generate(prompt, **free, top_p=1e-9), greedy)
    assert torch.equal(m.generate(prompt, **free, top_k=1), greedy)
    assert torch.equal(m.generate(prompt, max_length=20, temperature=1.0, min_p=1.0, top_k=63), greedy)

    cfg = dict(temperature=0.7, top_k=30, top_p=0.8, min_p=0.01)
    torch.manual_seed(1)
    got = m.generate(prompt, max_length=20, **cfg)
    torch.manual_seed(1)
    full, x, states = prompt, prompt, None
    with torch.no_grad():
        for _ in range(15):
            logits, states, _ = m(x, mem_states=states, return_cache=True)
            last = logits[:, -1:].float()
            x = A.sample_tokens(last, torch.rand(last.shape, device="cuda"), **cfg)
            full = torch.cat([full, x], dim=-1)
    assert torch.equal(got, full) and not torch.equal(got, greedy)
