"""GPU: the language-model operators under torch's other ways of calling a function: forward-mode differentiation is
refused, as by the package's other operators; torch.jit.trace has the call in it, so a traced call gives the same bits, checks
its inputs, and takes other sizes and strides than the traced ones."""
import warnings

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


def traced(f, *example):
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        return torch.jit.trace(f, example)


def same(f, module, *args):
    got, want = module(*args), f(*args)
    got, want = (got, want) if isinstance(got, tuple) else ((got,), (want,))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and len(got) == len(want)


@pytest.mark.parametrize("t", [1, 40])
def test_traced_scan(native_lib, t):
    from atlas_rnn_b200 import selective_scan
    names = ("u", "delta", "A", "B", "C", "z", "initial_state")
    f = lambda *a: selective_scan(**dict(zip(names, a)), delta_softplus=True)
    args = lambda *s, seed: [scan_inputs(*s, seed=seed)[k] for k in names]
    m = traced(f, *args(2, t, 6, 4, seed=1))
    same(f, m, *args(2, t, 6, 4, seed=10))
    other = args(3, t + 2, 10, 5, seed=20)
    same(f, m, *other)
    other[0] = other[0].transpose(1, 2).contiguous().transpose(1, 2)  # channels far apart
    other[2] = other[2].double()
    same(f, m, *other)
    leaves = [[v.detach().clone().requires_grad_() for v in other] for _ in range(2)]
    for out, hT in (f(*leaves[0]), m(*leaves[1])):
        (out.sum() + hT.sum()).backward()
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(*leaves))
    with pytest.raises(Exception, match="delta must have shape"):
        m(other[0], other[1][:, :-1], *other[2:])


@pytest.mark.parametrize("t", [1, 40])
def test_traced_convolution(native_lib, t):
    from atlas_rnn_b200 import causal_conv1d
    f = lambda x, w, b, s: causal_conv1d(x, w, b, initial_state=s, activation="silu")
    args = lambda b, t, c, seed: [rand(b, t, c, seed=seed), rand(c, 1, 4, seed=seed + 1), rand(c, seed=seed + 2),
                                  rand(b, 3, c, seed=seed + 3)]
    m = traced(f, *args(2, t, 6, seed=1))
    same(f, m, *args(2, t, 6, seed=10))
    other = args(3, t + 2, 9, seed=20)
    same(f, m, *other)
    other[0] = other[0].transpose(1, 2).contiguous().transpose(1, 2)
    other[1] = other[1].to(torch.bfloat16)
    same(f, m, *other)
    leaves = [[v.detach().clone().requires_grad_() for v in other] for _ in range(2)]
    for y, final in (f(*leaves[0]), m(*leaves[1])):
        (y.sum() + final.sum()).backward()
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(*leaves))
    with pytest.raises(Exception, match="initial_state must have shape"):
        m(*other[:3], other[3][:, :-1])


def test_traced_sampling(native_lib):
    from atlas_rnn_b200 import sample_tokens
    f = lambda l, u, k: sample_tokens(l, u, temperature=0.8, top_p=0.9, top_k=k)
    args = lambda rows, V, seed: [rand(rows, V, seed=seed), rand(rows, V, seed=seed + 1).sigmoid(),
                                  torch.arange(1, rows + 1, device="cuda")]
    m = traced(f, *args(3, 50, seed=1))
    same(f, m, *args(3, 50, seed=10))
    l, u, k = args(5, 700, seed=20)
    same(f, m, l, u, k)
    same(f, m, l.t().contiguous().t(), u, k)
    with pytest.raises(Exception, match="noise must have shape"):
        m(l, u[:, :-1], k)


def test_traced_distillation(native_lib):
    from atlas_rnn_b200 import distill_loss
    f = lambda x, v, i: distill_loss(x, v, i, temperature=2.0)

    def args(rows, V, K, seed):
        g = torch.Generator().manual_seed(seed)
        return [rand(rows, V, seed=seed), rand(rows, K, seed=seed + 1), torch.randint(0, V, (rows, K), generator=g).cuda()]

    m = traced(f, *args(3, 50, 4, seed=1))
    same(f, m, *args(3, 50, 4, seed=10))
    x, v, i = args(5, 700, 6, seed=20)
    same(f, m, x, v, i)
    same(f, m, x.t().contiguous().t(), v.double(), i.int())
    with pytest.raises(Exception, match="teacher_values must have shape"):
        m(x, v[:3], i)


@pytest.mark.parametrize("t", [1, 40])
def test_function_transforms_are_refused(native_lib, t):
    """torch.func's wrappers have no storage that a kernel could read."""
    from atlas_rnn_b200 import causal_conv1d, distill_loss, sample_tokens, selective_scan
    x = scan_inputs(2, t, 6, 4, seed=1)
    w, v = rand(6, 4, seed=2), rand(t, 3, seed=3)
    i = torch.zeros(t, 3, dtype=torch.int64, device="cuda")
    calls = [lambda u: selective_scan(**{**x, "u": u})[0], lambda u: causal_conv1d(u, w)[0],
             lambda u: distill_loss(u, v.expand(2, t, 3), i.expand(2, t, 3))]
    for f in calls:
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x["u"],), (torch.ones_like(x["u"]),))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda u: f(u).sum())(x["u"])
    for f in calls[:2] + [lambda u: sample_tokens(u, u.sigmoid())]:
        with pytest.raises(RuntimeError):
            torch.vmap(f)(x["u"][None].expand(3, *x["u"].shape).contiguous())


def test_recomputed_and_offloaded_training_steps(native_lib):
    """Gradients under activation checkpointing and with the kept tensors moved to the host are the plain step's bits."""
    from torch.utils.checkpoint import checkpoint
    from atlas_rnn_b200 import causal_conv1d, selective_scan
    x, w = scan_inputs(2, 70, 6, 4, seed=1), rand(6, 4, seed=2)
    names = list(x)

    def layer(*a):
        s = dict(zip(names, a[1:]))
        s["u"] = causal_conv1d(s["u"], a[0], activation="silu")[0]
        out, hT = selective_scan(**s, delta_softplus=True)
        return out.square().sum() + hT.sum()

    def grads(run):
        leaves = [w.clone().requires_grad_()] + [v.clone().requires_grad_() for v in x.values()]
        run(leaves).backward()
        return [v.grad for v in leaves]

    want = grads(lambda a: layer(*a))
    offloaded = grads(lambda a: offload(layer, a))
    for got in (grads(lambda a: checkpoint(layer, *a, use_reentrant=False)), offloaded):
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def offload(f, args):
    with torch.autograd.graph.save_on_cpu():
        return f(*args)
