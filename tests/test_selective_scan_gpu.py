"""GPU: selective_scan and causal_conv1d (atlas_sscan_*, atlas_causal_conv_*) against the recurrence
and the convolution written step by step in float64 with torch autograd.

Tolerances (rel-L2). Inputs are exact in both, the kernels accumulate in fp32. A step multiplies the state by
an exponential off by up to 2^-22 (the hardware's exp2) plus the rounding of its argument; such errors are
independent from step to step, so k remembered steps leave sqrt(k) 2^-22, and steps are remembered at most 1000
deep (dt >= 0.001, |A| >= 1 as drawn here): F32(T) = 8 sqrt(min(T, 1000)) 2^-22 + 2^-20 with a factor for the
sums' own roundings. A bf16 output adds its one rounding, half a step: 2^-8."""
import math

import pytest
import torch

from tests.helpers import rel_l2

pytestmark = pytest.mark.gpu

NAMES = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial_state")


def tol(T, dtype):
    f32 = 8 * math.sqrt(min(T, 1000)) * 2.0 ** -22 + 2.0 ** -20
    return f32 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)


def make(B, T, D, G, N, dtype=torch.float32, z=True, skip=True, bias=True, state=True, lengths=None, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * T + D)
    rn = lambda *s: torch.randn(*s, generator=g)
    step = torch.exp(torch.rand(D, generator=g) * math.log(100.0) + math.log(1e-3))
    x = dict(u=rn(B, T, D).to(dtype), delta=(0.5 * rn(B, T, D)).to(dtype),
             A=-torch.arange(1, N + 1).float() * torch.exp(0.2 * rn(D, N)), B=rn(B, T, G, N).to(dtype),
             C=rn(B, T, G, N).to(dtype), D=1 + 0.1 * rn(D) if skip else None, z=rn(B, T, D).to(dtype) if z else None,
             delta_bias=torch.log(torch.expm1(step)) if bias else None,
             initial_state=rn(B, D, N) if state else None)
    if not bias:
        x["delta"] = (x["delta"] - 3).to(dtype)
    x = {k: None if v is None else v.cuda() for k, v in x.items()}
    x["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return x


def call(x, softplus=True, chunk=0, **over):
    from atlas_rnn_b200 import selective_scan
    x = {**x, **over}
    return selective_scan(x["u"], x["delta"], x["A"], x["B"], x["C"], x["D"], x["z"], delta_bias=x["delta_bias"],
                          delta_softplus=softplus, initial_state=x["initial_state"], lengths=x["lengths"], chunk=chunk)


def reference(x, softplus=True):
    """Leaves in float64 on the CPU, (out, final state) by the recurrence."""
    leaf = {k: None if x[k] is None else x[k].detach().double().cpu().requires_grad_(True) for k in NAMES}
    u, A, B, C = leaf["u"], leaf["A"], leaf["B"], leaf["C"]
    b, t, d = u.shape
    g, n = B.shape[2:]
    pre = leaf["delta"] if leaf["delta_bias"] is None else leaf["delta"] + leaf["delta_bias"]
    dt = torch.nn.functional.softplus(pre, threshold=1e9) if softplus else pre
    h = torch.zeros(b, d, n, dtype=torch.float64) if leaf["initial_state"] is None else leaf["initial_state"]
    ends = [t] * b if x["lengths"] is None else x["lengths"].clamp(0, t).tolist()
    live = torch.tensor([[float(i < e) for i in range(t)] for e in ends], dtype=torch.float64)
    wide = lambda m: m.repeat_interleave(d // g, dim=1)
    outs = []
    for i in range(t):
        on = live[:, i, None]
        nh = torch.exp(dt[:, i, :, None] * A) * h + (dt[:, i] * u[:, i])[..., None] * wide(B[:, i])
        h = torch.where(on[..., None] > 0, nh, h)
        y = (h * wide(C[:, i])).sum(-1)
        if leaf["D"] is not None:
            y = y + leaf["D"] * u[:, i]
        if leaf["z"] is not None:
            y = y * torch.nn.functional.silu(leaf["z"][:, i])
        outs.append(torch.where(on > 0, y, torch.zeros_like(y)))
    return leaf, torch.stack(outs, 1), h


CASES = [
    # B, T, D, G, N, dtype, z, skip, bias, state, softplus, lengths, chunk
    (2, 1, 5, 1, 16, torch.float32, True, True, True, True, True, None, 0),
    (2, 2, 33, 1, 16, torch.float32, False, False, False, False, True, None, 0),
    (1, 31, 16, 1, 16, torch.float32, True, True, True, True, True, None, 0),
    (3, 33, 40, 2, 1, torch.float32, True, True, True, True, True, (33, 0, 17), 0),
    (2, 65, 70, 1, 3, torch.float32, True, False, True, False, True, None, 32),
    (2, 100, 36, 3, 8, torch.float32, False, True, True, True, True, (100, 31), 32),
    (1, 200, 64, 1, 10, torch.float32, True, True, True, True, False, None, 64),
    (2, 130, 24, 2, 17, torch.float32, True, True, False, True, True, (5, 130), 0),
    (1, 97, 12, 1, 33, torch.float32, True, True, True, True, True, None, 32),
    (2, 70, 20, 1, 64, torch.float32, True, True, True, True, True, (70, 64), 32),
    (1, 1024, 8, 1, 16, torch.float32, True, True, True, True, True, None, 0),
    (2, 300, 128, 1, 16, torch.bfloat16, True, True, True, True, True, None, 0),
    (2, 96, 65, 1, 16, torch.bfloat16, True, True, True, True, True, (96, 40), 32),
    (3, 37, 66, 3, 5, torch.bfloat16, False, True, True, False, True, (0, 1, 37), 0),
    (1, 257, 48, 1, 64, torch.bfloat16, True, True, True, True, True, None, 64),
    (1, 64, 130, 1, 24, torch.bfloat16, True, True, True, True, True, None, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])) + ("_bf16" if c[5] == torch.bfloat16
                                                                                     else "") + f"_c{c[12]}")
def test_scan_and_gradients(native_lib, case):
    B, T, D, G, N, dtype, z, skip, bias, state, softplus, lengths, chunk = case
    x = make(B, T, D, G, N, dtype, z, skip, bias, state, lengths)
    if not softplus:
        x["delta"] = x["delta"].float().abs().mul(0.1).to(dtype)
        x["delta_bias"] = None if x["delta_bias"] is None else x["delta_bias"].abs() * 0.01
    leaf, ref, ref_h = reference(x, softplus)
    with torch.no_grad():
        out0, h0 = call(x, softplus, chunk)
    for k in NAMES:
        if x[k] is not None:
            x[k].requires_grad_(True)
    out, h = call(x, softplus, chunk)
    assert out.dtype == dtype and h.dtype == torch.float32
    if T > 1:  # one step without gradients is another kernel
        assert torch.equal(out, out0) and torch.equal(h, h0)
    assert rel_l2(out0.float(), ref) <= tol(T, dtype) and rel_l2(h0, ref_h) <= tol(T, torch.float32)
    assert rel_l2(out.float(), ref) <= tol(T, dtype) and rel_l2(h, ref_h) <= tol(T, torch.float32)
    g = torch.Generator().manual_seed(1)
    up, uph = torch.randn(ref.shape, generator=g).to(dtype), torch.randn(ref_h.shape, generator=g)
    names = [k for k in NAMES if x[k] is not None]
    got = torch.autograd.grad((out, h), [x[k] for k in names], (up.cuda(), uph.cuda()))
    want = torch.autograd.grad((ref, ref_h), [leaf[k] for k in names], (up.double(), uph.double()))
    for k, a, w in zip(names, got, want):
        assert a.dtype == x[k].dtype and a.shape == x[k].shape
        assert rel_l2(a.float(), w) <= 2 * tol(T, a.dtype), (k, rel_l2(a.float(), w))


def test_rows_past_their_length_are_never_read(native_lib):
    x = make(3, 70, 40, 1, 16, lengths=(70, 33, 0))
    base = call(x)
    for k in ("u", "delta", "z", "B", "C"):
        x[k] = x[k].clone()
        x[k][1, 33:] = float("nan")
        x[k][2] = float("inf")
    leaves = [x[k].requires_grad_(True) for k in NAMES]
    out, h = call(x)
    assert torch.equal(out, base[0]) and torch.equal(h, base[1])
    assert (out[1, 33:] == 0).all() and (out[2] == 0).all() and torch.equal(h[2], x["initial_state"][2])
    up = torch.ones_like(out)
    up[1, 33:] = float("nan")
    for k, gr in zip(NAMES, torch.autograd.grad((out, h), leaves, (up, torch.ones_like(h)))):
        assert torch.isfinite(gr).all(), k
        if k in ("u", "delta", "z", "B", "C"):
            assert (gr[1, 33:] == 0).all() and (gr[2] == 0).all(), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_unaligned_inputs(native_lib, dtype):
    """u and z as halves of one projection, B and C inside another at an odd offset: same bits as dense copies."""
    B, T, D, N = 2, 75, 48, 16
    x = make(B, T, D, 1, N, dtype)
    uz = torch.cat([x["u"], x["z"]], -1)
    bc = torch.cat([torch.zeros(B, T, 3, dtype=dtype, device="cuda"), x["B"][:, :, 0], x["C"][:, :, 0]], -1)
    y = {**x, "u": uz[..., :D], "z": uz[..., D:], "B": bc[..., 3:3 + N].unsqueeze(2), "C": bc[..., 3 + N:].unsqueeze(2),
         "delta": x["delta"].transpose(0, 1).contiguous().transpose(0, 1)}
    leaves = lambda m: [m[k].requires_grad_(True) for k in NAMES]
    outs = []
    for m in (x, y):
        lv = leaves(m)
        o = call(m)
        outs.append([*o, *torch.autograd.grad(o, lv, [torch.ones_like(v) for v in o])])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    # channels that are not dense are copied
    t = {**x, "u": x["u"].detach().transpose(1, 2).contiguous().transpose(1, 2)}
    assert torch.equal(call(t)[0], outs[0][0])


def test_three_dimensional_b_and_c(native_lib):
    x = make(2, 20, 12, 1, 7)
    flat = call(x, B=x["B"][:, :, 0], C=x["C"][:, :, 0])
    assert all(torch.equal(a, b) for a, b in zip(flat, call(x)))


def test_a_prompt_cut_anywhere_and_single_tokens_continue_it(native_lib):
    from atlas_rnn_b200 import causal_conv1d
    B, T, D, N, K = 2, 45, 24, 16, 4
    x = make(B, T, D, 1, N)
    g = torch.Generator(device="cuda").manual_seed(5)
    w, bias = torch.randn(D, 1, K, device="cuda", generator=g), torch.randn(D, device="cuda", generator=g)

    def run(xs, conv_state, state):  # the convolution in front of the scan, as a layer runs them
        u, conv_state = causal_conv1d(xs["u"], w, bias, activation="silu", initial_state=conv_state)
        out, state = call({**xs, "u": u, "initial_state": state, "lengths": None})
        return out, conv_state, state

    cut = lambda lo, hi: {k: v[:, lo:hi] if k in ("u", "delta", "z", "B", "C") else v for k, v in x.items()}
    whole, wc, wh = run(x, None, x["initial_state"])
    outs, cs, st = [], None, x["initial_state"]
    for lo, hi in [(0, 1), (1, 20), (20, 21), (21, 22), (22, 44), (44, 45)]:
        o, cs, st = run(cut(lo, hi), cs, st)
        outs.append(o)
    assert torch.equal(cs, wc)
    assert rel_l2(torch.cat(outs, 1), whole) <= 2 * tol(T, torch.float32) and rel_l2(st, wh) <= 2 * tol(T, torch.float32)


@pytest.mark.parametrize("N", [1, 4, 10, 16, 24, 64])
def test_one_token(native_lib, N):
    x = make(5, 1, 12, 2, N, lengths=(1, 0, 1, 1, 1))
    _, ref, ref_h = reference(x)
    with torch.no_grad():
        out, h = call(x)
    assert rel_l2(out, ref) <= tol(1, torch.float32) and rel_l2(h, ref_h) <= tol(1, torch.float32)
    assert (out[1] == 0).all() and torch.equal(h[1], x["initial_state"][1])


def test_same_bits_twice_and_on_another_stream(native_lib):
    x = make(2, 300, 64, 1, 16, torch.bfloat16)
    leaves = [x[k].requires_grad_(True) for k in NAMES]

    def run():
        o = call(x, chunk=64)
        return [*o, *torch.autograd.grad(o, leaves, [torch.ones_like(v) for v in o])]

    first = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = run()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_captured_and_replayed(native_lib):
    x = make(2, 40, 32, 1, 16)
    one = {k: v[:, :1].clone() if k in ("u", "delta", "z", "B", "C") else v for k, v in x.items()}
    with torch.no_grad():
        call(x, chunk=32), call(one)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, h = call(x, chunk=32)
            o1, h1 = call({**one, "initial_state": h})
        x["u"].mul_(-0.5)
        one["u"].add_(1.0)
        graph.replay()
        want, wh = call(x, chunk=32)
        w1, wh1 = call({**one, "initial_state": wh})
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(h, wh) and torch.equal(o1, w1) and torch.equal(h1, wh1)


def test_gradient_against_differences(native_lib):
    """Directional derivative of a random weighting of the outputs, central differences over the kernel's own forward.
    With step s the difference is off by O(s^2) of the third derivative (1e-4 of it at s = 0.01) and by the forward's
    2^-20 relative rounding over 2 s: 5e-5 of the sum's size, which is sqrt(values) times the derivative at most."""
    x = make(2, 40, 16, 1, 8)
    g = torch.Generator(device="cuda").manual_seed(9)
    rn = lambda t: torch.randn(t.shape, device="cuda", generator=g)
    leaves = [x[k].requires_grad_(True) for k in NAMES]
    out, h = call(x)
    wo, wh = rn(out), rn(h)
    grads = torch.autograd.grad((out, h), leaves, (wo, wh))
    for k, leaf, gr in zip(NAMES, leaves, grads):
        v = gr / gr.norm()  # along the gradient the derivative is its norm

        def f(s):
            with torch.no_grad():
                o, hh = call({**x, k: leaf.detach() + s * v})
                return ((o.double() * wo).sum() + (hh.double() * wh).sum()).item()
        s = 0.01
        got = (f(s) - f(-s)) / (2 * s)
        assert abs(got - gr.norm().item()) <= 1e-2 * gr.norm().item(), (k, got, gr.norm().item())


def test_only_some_gradients_wanted(native_lib):
    x = make(2, 34, 16, 1, 16)
    full = {k: v for k, v in zip(NAMES, torch.autograd.grad(call({**x, **{k: x[k].requires_grad_(True) for k in NAMES}})[0].sum(),
                                                             [x[k] for k in NAMES]))}
    for k in NAMES:
        y = {n: v.detach() if v is not None and n in NAMES else v for n, v in x.items()}
        y[k] = y[k].clone().requires_grad_(True)
        (gr,) = torch.autograd.grad(call(y)[0].sum(), [y[k]])
        assert torch.equal(gr, full[k]), k
    y = {n: v.detach() if v is not None and n in NAMES else v for n, v in x.items()}
    y["u"] = y["u"].clone().requires_grad_(True)
    h = call(y)[1]  # the final state alone
    (gr,) = torch.autograd.grad(h.sum(), [y["u"]])
    leaf, _, ref_h = reference(y)
    (want,) = torch.autograd.grad(ref_h.sum(), [leaf["u"]])
    assert rel_l2(gr, want) <= 2 * tol(34, torch.float32)


def test_no_steps_and_no_rows(native_lib):
    x = make(2, 4, 8, 1, 16)
    none = {k: v[:, :0] if k in ("u", "delta", "z", "B", "C") else v for k, v in x.items()}
    out, h = call(none)
    assert out.shape == (2, 0, 8) and torch.equal(h, x["initial_state"])
    empty = {k: v[:0] if k in ("u", "delta", "z", "B", "C", "initial_state") else v for k, v in x.items()}
    out, h = call(empty)
    assert out.shape == (0, 4, 8) and h.shape == (0, 8, 16)


def test_large_step_arguments_stay_finite(native_lib):
    """softplus far out on both sides (0 and x itself), decays that underflow, gates that saturate."""
    x = make(1, 40, 8, 1, 16)
    x["delta"][0, ::3] = 60.0
    x["delta"][0, 1::3] = -120.0
    x["z"][0, ::2] = 200.0
    x["z"][0, 1::2] = -200.0
    leaves = [x[k].requires_grad_(True) for k in NAMES]
    leaf, ref, ref_h = reference(x)
    out, h = call(x)
    assert rel_l2(out, ref) <= tol(40, torch.float32) and rel_l2(h, ref_h) <= tol(40, torch.float32)
    got = torch.autograd.grad((out, h), leaves, (torch.ones_like(out), torch.ones_like(h)))
    want = torch.autograd.grad((ref, ref_h), [leaf[k] for k in NAMES], (torch.ones_like(ref), torch.ones_like(ref_h)))
    for k, a, w in zip(NAMES, got, want):
        assert torch.isfinite(a).all() and rel_l2(a, w) <= 2 * tol(40, torch.float32), (k, rel_l2(a, w))


# ---- causal convolution ----------------------------------------------------------------------

def conv_reference(x, w, bias, silu, init, lengths):
    f = lambda t: None if t is None else t.detach().double().cpu().requires_grad_(True)
    x, w, bias, init = f(x), f(w), f(bias), f(init)
    b, t, c = x.shape
    k = w.shape[-1]
    first = torch.zeros(b, k - 1, c, dtype=torch.float64) if init is None else init
    full = torch.cat([first, x], 1)
    pre = sum(full[:, j:j + t] * w.reshape(c, k)[:, j] for j in range(k))
    if bias is not None:
        pre = pre + bias
    y = torch.nn.functional.silu(pre) if silu else pre
    ends = [t] * b if lengths is None else lengths.clamp(0, t).tolist()
    y = torch.stack([torch.cat([y[i, :e], torch.zeros_like(y[i, e:])]) for i, e in enumerate(ends)])
    final = torch.stack([full[i, e:e + k - 1] for i, e in enumerate(ends)])
    return (x, w, bias, init), y, final


@pytest.mark.parametrize("B,T,C,K,dtype,silu,bias,state,lengths", [
    (2, 1, 5, 4, torch.float32, True, True, True, None),
    (1, 2, 8, 4, torch.float32, True, True, False, None),
    (3, 37, 33, 2, torch.float32, False, False, True, (37, 0, 2)),
    (2, 300, 130, 3, torch.float32, True, True, True, (300, 299)),
    (2, 129, 64, 4, torch.bfloat16, True, True, True, None),
    (2, 700, 256, 4, torch.bfloat16, True, True, True, (700, 3)),
    (1, 90, 17, 5, torch.bfloat16, False, True, True, (31,)),
    (2, 65, 40, 6, torch.float32, True, True, True, None),
    (1, 64, 7, 7, torch.float32, True, False, False, None),
    (2, 50, 96, 8, torch.bfloat16, True, True, True, (4, 50)),
])
def test_conv_and_gradients(native_lib, B, T, C, K, dtype, silu, bias, state, lengths):
    from atlas_rnn_b200 import causal_conv1d
    g = torch.Generator(device="cuda").manual_seed(T + K)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, w = rn(B, T, C).to(dtype).requires_grad_(True), rn(C, 1, K).requires_grad_(True)
    b = rn(C).requires_grad_(True) if bias else None
    init = rn(B, K - 1, C).to(dtype).requires_grad_(True) if state else None
    ln = None if lengths is None else torch.tensor(lengths, device="cuda")
    leaf, ref, ref_f = conv_reference(x, w, b, silu, init, ln)
    y, final = causal_conv1d(x, w, b, activation="silu" if silu else None, initial_state=init, lengths=ln)
    # K products and the activation in fp32: (K + 4) 2^-24 of the largest term, against a sum that may cancel: 2^-18
    bound = 2.0 ** -18 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    assert y.dtype == dtype and rel_l2(y.float(), ref) <= bound
    assert torch.equal(final.double().cpu(), ref_f)  # copies
    dy, df = rn(*y.shape).to(dtype), rn(*final.shape).to(dtype)
    pairs = [(n, a, l) for n, a, l in zip(("x", "w", "bias", "init"), (x, w, b, init), leaf) if a is not None]
    got = torch.autograd.grad((y, final), [p[1] for p in pairs], (dy, df))
    want = torch.autograd.grad((ref, ref_f), [p[2] for p in pairs], (dy.double().cpu(), df.double().cpu()))
    for (n, a, _), gr, wt in zip(pairs, got, want):
        lim = 2.0 ** -18 + (2.0 ** -8 if gr.dtype == torch.bfloat16 else 0.0)
        assert gr.dtype == a.dtype and rel_l2(gr.float(), wt) <= lim, (n, rel_l2(gr.float(), wt))


def test_conv_strides_dead_rows_and_bits(native_lib):
    from atlas_rnn_b200 import causal_conv1d
    g = torch.Generator(device="cuda").manual_seed(2)
    wide = torch.randn(3, 80, 2 * 66 + 1, device="cuda", generator=g)
    w, bias = torch.randn(66, 4, device="cuda", generator=g), torch.randn(66, device="cuda", generator=g)
    ln = torch.tensor([80, 7, 0], device="cuda")
    x = wide[..., 1:67]
    leaves = [t.requires_grad_(True) for t in (w, bias)]
    run = lambda v: causal_conv1d(v, w, bias, activation="silu", lengths=ln)
    a, b = run(x), run(x.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    bad = x.clone()
    bad[1, 7:], bad[2] = float("nan"), float("inf")
    bad.requires_grad_(True)
    c = run(bad)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    grads = torch.autograd.grad(c[0].sum(), [bad] + leaves)
    again = torch.autograd.grad(run(bad)[0].sum(), [bad] + leaves)
    assert all(torch.isfinite(t).all() and torch.equal(t, s) for t, s in zip(grads, again))
    assert (grads[0][1, 7:] == 0).all() and (grads[0][2] == 0).all()


def test_second_derivatives_are_refused(native_lib):
    x = make(1, 8, 8, 1, 8)
    x["u"].requires_grad_(True)
    (gr,) = torch.autograd.grad(call(x)[0].sum(), [x["u"]], create_graph=True)
    with pytest.raises(RuntimeError):
        gr.sum().backward()
