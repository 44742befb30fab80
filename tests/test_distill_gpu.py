"""GPU: distill_loss (atlas_distill_forward / _backward) against its definition in float64 with torch autograd.

Tolerances (rel-L2). The loss is a difference of logarithms of size about 10 (log p - log q), each rounded to fp32 at
2^-23 of about 20 in units of log2: 2^-18 absolute, against losses of 0.1 and more here: 2^-14. Gradients are
tau g (q - p): q's exponent is rounded at 2^-23 of about 30, so 2^-18 of q; where q and p cancel the difference keeps the
error of the larger: 2^-16 over a row. A bf16 gradient adds half a step, 2^-8."""
import pytest
import torch

from tests.helpers import rel_l2

pytestmark = pytest.mark.gpu

LOSS_TOL, GRAD_TOL = 2.0 ** -14, 2.0 ** -16


def reference(logits, values, indices, tau):
    """(leaf, per-row losses, rows with entries)."""
    V, K = logits.shape[-1], values.shape[-1]
    x = logits.detach().double().cpu().reshape(-1, V).requires_grad_(True)
    v, i = values.detach().double().cpu().reshape(-1, K), indices.cpu().long().reshape(-1, K)
    logq = torch.log_softmax(x / tau, -1)
    losses, some = [], []
    for r in range(x.shape[0]):
        on = (i[r] >= 0) & (i[r] < V) & (v[r] > -float("inf"))
        some.append(bool(on.any()))
        if not some[-1]:
            losses.append(0.0 * x[r, 0].detach())
            continue
        logp = torch.log_softmax(v[r][on] / tau, -1)
        losses.append(tau ** 2 * (logp.exp() * (logp - logq[r, i[r][on]])).sum())
    return x, torch.stack(losses), torch.tensor(some)


def make(rows, V, K, dtype, seed, ragged=True, repeat=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (2 * torch.randn(rows, V, device="cuda", generator=g)).to(dtype)
    v = 3 + 2 * torch.randn(rows, K, device="cuda", generator=g)
    i = torch.randint(0, max(1, V // 4) if repeat else V, (rows, K), device="cuda", generator=g)
    if ragged:
        n = torch.randint(0, K + 1, (rows, 1), device="cuda", generator=g)
        i = torch.where(torch.arange(K, device="cuda") < n, i, -1)
    return x, v, i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,K,tau,repeat", [
    (1, 1, 1, 1.0, False), (3, 2, 5, 1.0, True), (7, 256, 17, 2.0, False), (33, 257, 64, 0.5, True),
    (5, 1001, 1024, 1.0, True), (2, 50001, 20, 2.0, False), (3, 32768, 100, 1.0, False), (300, 4096, 8, 1.5, False),
])
def test_loss_and_gradient(native_lib, rows, V, K, tau, repeat, dtype):
    from atlas_rnn_b200 import distill_loss
    x, v, i = make(rows, V, K, dtype, V + K, repeat=repeat)
    x.requires_grad_(True)
    leaf, ref, some = reference(x, v, i, tau)
    loss = distill_loss(x, v, i, temperature=tau, reduction="none")
    assert loss.dtype == torch.float32 and loss.shape == (rows,)
    assert rel_l2(loss, ref) <= LOSS_TOL or ref.norm() < 1e-3
    g = torch.Generator(device="cuda").manual_seed(1)
    up = torch.randn(rows, device="cuda", generator=g)
    (got,) = torch.autograd.grad(loss, [x], up)
    assert got.dtype == dtype
    if some.any() and V > 1:
        (want,) = torch.autograd.grad(ref, [leaf], up.double().cpu())
        assert rel_l2(got.float(), want) <= GRAD_TOL + (2.0 ** -8 if dtype == torch.bfloat16 else 0)
    assert (got.cpu()[~some] == 0).all() and (loss.cpu()[~some] == 0).all()


def test_reductions_and_shapes(native_lib):
    from atlas_rnn_b200 import distill_loss
    x, v, i = make(12, 300, 9, torch.float32, 2)
    i[0] = i[5] = -1
    each = distill_loss(x, v, i, reduction="none")
    n = (i >= 0).any(-1).sum()
    assert torch.allclose(distill_loss(x, v, i, reduction="sum"), each.sum())
    assert torch.allclose(distill_loss(x, v, i), each.sum() / n)
    assert torch.equal(distill_loss(x.view(3, 4, 300), v.view(3, 4, 9), i.view(3, 4, 9), reduction="none"), each.view(3, 4))
    assert torch.equal(distill_loss(x, v.double(), i.int(), reduction="none"), each)
    nothing = torch.full_like(i, -1)
    y = x.clone().requires_grad_(True)
    loss = distill_loss(y, v, nothing)
    assert loss == 0 and (torch.autograd.grad(loss, [y])[0] == 0).all()
    assert distill_loss(x[:0], v[:0], i[:0], reduction="none").shape == (0,) and distill_loss(x[:0], v[:0], i[:0]) == 0


def test_absent_entries_infinities_and_masked_students(native_lib):
    from atlas_rnn_b200 import distill_loss
    inf, nan = float("inf"), float("nan")
    x, v, i = make(6, 500, 10, torch.float32, 3, ragged=False)
    i[0, 3], i[0, 4], v[0, 5], v[0, 6] = 500, 1 << 40, -inf, nan
    x[1, ::2] = -inf           # masked students: their tokens carry no gradient
    i[1] = i[1] | 1
    v[2] = -inf                # no entry left
    x[2] = nan                 # .. so the row is not looked at
    v[3, 1:] = v[3, 0] - 200.0  # the others' weights underflow
    x[3, i[3, 4]] = -inf
    i[3, 4] = (i[3, 0] + 1) % 500
    i[4] = 7                   # one token, ten times
    x[5] = x[5] * 0 + torch.finfo(torch.float32).min / 2
    x.requires_grad_(True)
    leaf, ref, some = reference(torch.where(torch.arange(6, device="cuda")[:, None] == 2, 0.0, x.detach()), v, i, 1.0)
    loss = distill_loss(x, v, i, reduction="none")
    keep = torch.tensor([0, 1, 3, 4, 5])
    assert rel_l2(loss.cpu()[keep], ref[keep]) <= LOSS_TOL and loss[2] == 0
    (got,) = torch.autograd.grad(loss.sum(), [x])
    (want,) = torch.autograd.grad(ref.sum(), [leaf])
    assert (got[2] == 0).all() and (got[1, ::2] == 0).all()
    assert rel_l2(got.cpu()[keep], want[keep]) <= GRAD_TOL


def test_strided_unaligned_streams_and_replay(native_lib):
    from atlas_rnn_b200 import distill_loss
    x, v, i = make(10, 5000, 20, torch.bfloat16, 4)

    def run(t):
        t = t.detach().requires_grad_(True)
        loss = distill_loss(t, v, i, reduction="none")
        return loss, torch.autograd.grad(loss.sum(), [t])[0]
    want = run(x)
    wide = torch.zeros(10, 5003, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:] = x
    for t in (wide[:, 3:], x.t().contiguous().t()):
        got = run(t)
        assert rel_l2(got[0], want[0]) <= 2.0 ** -20  # other lanes add other parts
        assert rel_l2(got[1].float(), want[1].float()) <= 2.0 ** -8
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = run(x)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = distill_loss(x, v, i, reduction="none")
        x.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, distill_loss(x, v, i, reduction="none"))


def test_gradient_against_differences(native_lib):
    """Central differences along the gradient, step 0.05: the third derivative costs about 1e-3 of it, the loss's rounding
    (1e-6 of about 30) over 0.1 another 1e-3 of a gradient of size 1."""
    from atlas_rnn_b200 import distill_loss
    x, v, i = make(16, 300, 12, torch.float32, 5)
    x.requires_grad_(True)
    (gr,) = torch.autograd.grad(distill_loss(x, v, i, reduction="sum", temperature=2.0), [x])
    d = gr / gr.norm()
    f = lambda s: distill_loss(x.detach() + s * d, v, i, reduction="none", temperature=2.0).double().sum().item()
    assert abs((f(0.05) - f(-0.05)) / 0.1 - gr.norm().item()) <= 1e-2 * gr.norm().item()


def test_language_model_loss_with_a_teacher(native_lib):
    import atlas_rnn_b200 as A
    torch.manual_seed(0)
    m = A.RNNMemoryTransformer(num_tokens=64, dim=32, depth=1, heads=1, dim_head=32, omega_window=2).cuda()
    x = torch.randint(0, 64, (2, 9), device="cuda")
    values, indices = torch.randn(2, 8, 5, device="cuda"), torch.randint(0, 64, (2, 8, 5), device="cuda")
    plain = m(x, return_loss=True)
    assert torch.equal(m(x, return_loss=True, teacher=(values, indices), distill_weight=0.0), plain)
    logits = m(x[:, :-1])
    want = 0.75 * plain + 0.25 * A.distill_loss(logits, values, indices, temperature=2.0)
    got = m(x, return_loss=True, teacher=(values, indices), distill_weight=0.25, distill_temperature=2.0)
    assert torch.allclose(got, want, rtol=1e-5)
    got.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
