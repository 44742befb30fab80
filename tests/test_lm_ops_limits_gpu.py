"""GPU: the language-model operators at the ends of their ranges: elements past 2^31, batches past a grid's second
dimension, decays of -inf, repeated tokens among many entries, several streams at once, captured training steps."""
import pytest
import torch

from tests.helpers import rel_l2
from tests.test_distill_gpu import GRAD_TOL, make as distill_case, reference as distill_reference
from tests.test_sampling_gpu import reference as sample_reference
from tests.test_selective_scan_gpu import NAMES, call, make, reference, tol

pytestmark = pytest.mark.gpu
FAR = (1 << 31) + 64  # elements between two rows


def gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, device="cuda", generator=g)


def test_rows_more_than_31_bits_apart(native_lib):
    """The second row of every strided operand lies behind 2^31 elements of the first."""
    from atlas_rnn_b200 import causal_conv1d, distill_loss, sample_tokens, selective_scan
    rn = gen(1)
    store = torch.zeros(FAR + 40000, dtype=torch.bfloat16, device="cuda")

    def far(x):  # [2, ...] with its rows FAR apart
        v = store.as_strided(x.shape, (FAR, *x.stride()[1:]))
        v.copy_(x)
        return v
    T, D, N = 40, 64, 16
    x, A = rn(2, T, D).bfloat16(), -rn(D, N).exp()
    bc = rn(2, T, 2 * N).bfloat16()
    near = selective_scan(x, x, A, bc[..., :N], bc[..., N:], z=x, delta_softplus=True)
    v = far(x)
    assert all(torch.equal(a, b) for a, b in zip(near, selective_scan(v, v, A, bc[..., :N], bc[..., N:], z=v, delta_softplus=True)))
    w = far(bc)
    assert all(torch.equal(a, b) for a, b in zip(near, selective_scan(x, x, A, w[..., :N], w[..., N:], z=x, delta_softplus=True)))
    one = [selective_scan(p[:, :1], p[:, :1], A, q[:, :1, :N], q[:, :1, N:], delta_softplus=True) for p, q in ((x, bc), (x, w))]
    assert all(torch.equal(a, b) for a, b in zip(*one))
    taps = rn(D, 4)
    want = causal_conv1d(x, taps, activation="silu")
    assert all(torch.equal(a, b) for a, b in zip(want, causal_conv1d(far(x), taps, activation="silu")))
    logits, noise = rn(2, 30000).bfloat16(), torch.rand(2, 30000, device="cuda")
    v, i = rn(2, 20), torch.randint(0, 30000, (2, 20), device="cuda")
    want = sample_tokens(logits, noise, top_p=0.9), distill_loss(logits, v, i, reduction="none")
    y = far(logits)
    assert torch.equal(want[0], sample_tokens(y, noise, top_p=0.9))
    assert torch.equal(want[1], distill_loss(y, v, i, reduction="none"))


def test_results_of_more_than_31_bits(native_lib):
    """Rows that are one row in memory (stride 0): all results equal, those past 2^31 elements too."""
    from atlas_rnn_b200 import causal_conv1d, distill_loss, selective_scan
    rn = gen(2)
    B, T, D, N = 1100, 1024, 2048, 8
    x, bc, A = rn(1, T, D).bfloat16(), rn(1, T, N).bfloat16(), -rn(D, N).exp()
    r = lambda t: t.expand(B, *t.shape[1:])
    out, h = selective_scan(r(x), r(x), A, r(bc), r(bc), delta_softplus=True)
    for i in (B // 2, B - 1):
        assert torch.equal(out[0], out[i]) and torch.equal(h[0], h[i])
    del out
    y, final = causal_conv1d(r(x), rn(D, 4), activation="silu")
    assert torch.equal(y[0], y[B - 1]) and torch.equal(final[0], final[B - 1])
    del y
    rows, V = 70000, 32000
    one = rn(1, V).bfloat16()
    logits = one.expand(rows, V).detach().requires_grad_(True)
    v, i = rn(1, 8).expand(rows, 8), torch.randint(0, V, (1, 8), device="cuda").expand(rows, 8)
    loss = distill_loss(logits, v, i, reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), [logits])
    assert (loss == loss[0]).all()
    for k in (rows // 2, rows - 1):
        assert torch.equal(grad[0], grad[k])


@pytest.mark.parametrize("T", [1, 3])
def test_more_rows_than_a_grid_is_high(native_lib, T):
    from atlas_rnn_b200 import causal_conv1d, selective_scan
    rn = gen(3)
    B, D, N = 70001, 6, 5
    x, bc, A, w = rn(B, T, D), rn(B, T, N), -rn(D, N).exp(), rn(D, 3)
    out, h = selective_scan(x, x, A, bc, bc, delta_softplus=True)
    y, final = causal_conv1d(x, w)
    for i in (0, 65534, 65535, B - 1):
        s = slice(i, i + 1)
        o1, h1 = selective_scan(x[s], x[s], A, bc[s], bc[s], delta_softplus=True)
        # the one-step kernel and the walking one round differently: a few of 2^-24 of terms that may cancel
        assert rel_l2(out[s], o1) <= 2.0 ** -18 and rel_l2(h[s], h1) <= 2.0 ** -18
        y1, f1 = causal_conv1d(x[s], w)
        assert rel_l2(y[s], y1) <= 2.0 ** -18 and torch.equal(final[s], f1)


@pytest.mark.parametrize("T,lengths", [(1, None), (1, (0, 1)), (37, (30, 0)), (700, (700, 350))])
def test_decays_of_minus_infinity(native_lib, T, lengths):
    """exp(dt A) = 0 for dt > 0, 1 for the steps that are none: against a finite A whose exponentials are 0 as well."""
    x = make(2, T, 16, 1, 16)
    x["lengths"] = None if lengths is None else torch.tensor(lengths, device="cuda")
    x["A"][::3, ::2] = -float("inf")
    finite = {**x, "A": torch.where(x["A"].isinf(), -1e30, x["A"])}
    leaves = [x[k].requires_grad_(True) for k in NAMES]
    leaf, ref, ref_h = reference(finite)
    out, h = call(x)
    with torch.no_grad():
        again = call(x)
    for o, hh in ((out, h), again):
        assert rel_l2(o, ref) <= tol(T, torch.float32) and rel_l2(hh, ref_h) <= tol(T, torch.float32)
    got = torch.autograd.grad((out, h), leaves, (torch.ones_like(out), torch.ones_like(h)))
    want = torch.autograd.grad((ref, ref_h), [leaf[k] for k in NAMES], (torch.ones_like(ref), torch.ones_like(ref_h)))
    for k, a, w in zip(NAMES, got, want):
        assert torch.isfinite(a).all() and rel_l2(a, w) <= 2 * tol(T, torch.float32), (k, rel_l2(a, w))


def test_lengths_of_64_bits(native_lib):
    from atlas_rnn_b200 import causal_conv1d
    x, w = gen(4)(4, 9, 8), gen(5)(8, 4)
    long = torch.tensor([-(1 << 40), 1 << 40, 5, 0], device="cuda")
    short = torch.tensor([0, 9, 5, 0], dtype=torch.int32, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(causal_conv1d(x, w, lengths=long), causal_conv1d(x, w, lengths=short)))


@pytest.mark.parametrize("K", [33, 128, 1000])
@pytest.mark.parametrize("tokens", [1, 40, 16384])
def test_repeated_tokens_among_many_entries(native_lib, K, tokens):
    """All entries one token, many repeats, and tokens whose low 14 bits agree without being equal."""
    from atlas_rnn_b200 import distill_loss
    V = 40000
    x, v, i = distill_case(3, V, K, torch.float32, K + tokens, ragged=False)
    i = i % tokens
    i[1] = i[1] + 16384 * (torch.arange(K, device="cuda") % 2)
    i[2, K // 2:] = -1
    x.requires_grad_(True)
    leaf, ref, _ = distill_reference(x, v, i, 1.0)
    (got,) = torch.autograd.grad(distill_loss(x, v, i, reduction="sum"), [x])
    (want,) = torch.autograd.grad(ref.sum(), [leaf])
    assert rel_l2(got, want) <= GRAD_TOL


def test_the_longest_row_of_equal_logits(native_lib):
    """The masses of a row add up to nearly 2^64."""
    from atlas_rnn_b200 import sample_tokens
    V = (1 << 24) - 16
    x, u = torch.zeros(1, V, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, V, device="cuda")
    u[0, V // 2 - 1], u[0, V // 2 + 1], u[0, V - 1] = 0.5, 0.9, 0.95
    # top-p keeps ceil(p V) tokens by index
    assert sample_tokens(x, u).item() == V - 1
    assert sample_tokens(x, u, top_p=0.5).item() == V // 2 - 1
    assert sample_tokens(x, u, top_p=0.75).item() == V // 2 + 1
    assert sample_tokens(x, u, top_k=V // 2).item() == V // 2 - 1


def test_calls_on_several_streams_at_once(native_lib):
    from atlas_rnn_b200 import causal_conv1d, distill_loss, sample_tokens
    rn = gen(6)
    x = make(2, 900, 96, 1, 16)
    for k in NAMES:
        x[k].requires_grad_(True)
    taps = rn(96, 4).requires_grad_(True)
    v, i = rn(64, 50), torch.randint(0, 20000, (64, 50), device="cuda")
    logits, noise = rn(64, 20000).requires_grad_(True), torch.rand(64, 20000, device="cuda")

    def work():
        out, h = call(x)
        y, _ = causal_conv1d(out, taps, activation="silu")
        loss = distill_loss(logits, v, i)
        token = sample_tokens(logits, noise, top_k=40, top_p=0.9)
        return [out, h, y, loss, token, *torch.autograd.grad((y, loss), [x[k] for k in NAMES] + [taps, logits],
                                                             (torch.ones_like(y), torch.ones_like(loss)))]
    want = work()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_a_captured_training_step(native_lib):
    """Forward and backward of the operators together in one graph, replayed on new inputs (the leaves have no eager graph)."""
    from atlas_rnn_b200 import causal_conv1d, distill_loss, selective_scan
    rn = gen(7)
    b, t, d, n, V = 2, 70, 32, 16, 1000
    x = rn(b, t, d)
    params = [p.requires_grad_(True) for p in (rn(d, 4), -rn(d, n).exp().detach(), rn(d), rn(d, 2 * n) * 0.2, rn(d, V) * 0.1)]
    v, i = rn(b, t, 12), torch.randint(0, V, (b, t, 12), device="cuda")

    def step():
        w, A, D, proj, head = params
        u, _ = causal_conv1d(x, w, activation="silu")
        bc = u @ proj
        y, _ = selective_scan(u, u, A, bc[..., :n], bc[..., n:], D, z=x, delta_softplus=True)
        return torch.autograd.grad(distill_loss(y @ head, v, i), params)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (8, 9):
        x.copy_(gen(seed)(b, t, d))
        graph.replay()
        torch.cuda.synchronize()
        kept = [g.clone() for g in got]
        want = step()
        # the library products may take other kernels outside the graph: fp32 products of 32 terms, 2^-20
        for g, w in zip(kept, want):
            assert rel_l2(g, w) <= 2.0 ** -16


def test_extreme_temperatures(native_lib):
    from atlas_rnn_b200 import distill_loss, sample_tokens
    x, v, i = distill_case(4, 300, 6, torch.float32, 10, ragged=False)
    for tau in (1e-3, 1e3):
        y = x.clone().requires_grad_(True)
        leaf, ref, _ = distill_reference(y, v, i, tau)
        loss = distill_loss(y, v, i, temperature=tau, reduction="none")
        # tau 1000: differences of 1e-3 between logarithms of size 10 (2^-20 each), times tau^2
        assert (loss.cpu().double() - ref.detach()).norm() <= 2.0 ** -14 * ref.norm() + 2.0 ** -19 * tau ** 2
        (got,) = torch.autograd.grad(loss.sum(), [y])
        (want,) = torch.autograd.grad(ref.sum(), [leaf])
        assert rel_l2(got, want) <= GRAD_TOL
    u = torch.rand(4, 300, device="cuda")
    for t in (1e-29, 1e-6, 1e30):
        assert torch.equal(sample_tokens(x, u, temperature=t).cpu(), sample_reference(x, u, temperature=t))
    assert torch.equal(sample_tokens(x, u, temperature=1e-40), x.argmax(-1))


@pytest.mark.parametrize("N,G,z,dtype", [(5, 1, True, torch.float32), (8, 3, False, torch.bfloat16), (16, 1, True, torch.bfloat16),
                                         (17, 2, True, torch.float32), (32, 1, False, torch.float32),
                                         (64, 1, True, torch.bfloat16)])
def test_one_token_for_many_rows(native_lib, N, G, z, dtype):
    """Several rows a thread, the last ones fewer; rows without a step hold NaN."""
    B, D = 1190 + 3, 6
    g = torch.Generator().manual_seed(N)
    x = make(B, 1, D, G, N, dtype, z=z)
    x["lengths"] = (torch.rand(B, generator=g) < 0.8).int().cuda()
    _, ref, ref_h = reference(x)
    dead = x["lengths"] == 0
    for k in ("u", "delta", "B", "C", "z"):
        if x[k] is not None:
            x[k][dead] = float("nan")
    with torch.no_grad():
        out, h = call(x)
    assert rel_l2(out.float(), ref) <= tol(1, dtype) and rel_l2(h, ref_h) <= tol(1, torch.float32)
    assert (out[dead] == 0).all() and torch.equal(h[dead], x["initial_state"][dead])
    x["lengths"] = None
    x = {k: v if v is None else v[~dead] if v.shape[0] == B else v for k, v in x.items()}
    with torch.no_grad():
        again = call(x)
    assert torch.equal(again[0], out[~dead]) and torch.equal(again[1], h[~dead])


@pytest.mark.parametrize("C,K,dtype", [(6, 2, torch.float32), (1028, 3, torch.bfloat16), (64, 4, torch.bfloat16),
                                       (7, 5, torch.float32), (130, 6, torch.float32), (9, 7, torch.bfloat16),
                                       (36, 8, torch.float32)])
def test_one_convolution_step_for_many_rows(native_lib, C, K, dtype):
    from atlas_rnn_b200 import causal_conv1d
    from tests.test_selective_scan_gpu import conv_reference
    B = 303
    rn = gen(C)
    x, w, bias, init = rn(B, 1, C).to(dtype), rn(C, K), rn(C), rn(B, K - 1, C).to(dtype)
    lengths = (torch.rand(B, device="cuda") < 0.8).int()
    _, ref, ref_f = conv_reference(x, w, bias, True, init, lengths)
    x[lengths == 0] = float("nan")
    y, final = causal_conv1d(x, w, bias, activation="silu", initial_state=init, lengths=lengths)
    # K products and the activation in fp32, as for longer rows: 2^-18, and half a step of bf16
    assert rel_l2(y.float(), ref) <= 2.0 ** -18 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    assert torch.equal(final.double().cpu(), ref_f)
    # taps at any alignment, few rows
    shifted = torch.empty(C * K + 1, device="cuda")[1:].view(C, K).copy_(w)
    some = slice(0, 5)
    for v in (w, shifted):
        o, f = causal_conv1d(x[some], v, bias, activation="silu", initial_state=init[some], lengths=lengths[some])
        assert torch.equal(o, y[some]) and torch.equal(f, final[some])


@pytest.mark.parametrize("K,dtype,C", [(2, torch.bfloat16, 8192), (3, torch.float32, 8192), (4, torch.bfloat16, 8192),
                                       (4, torch.float32, 8190), (4, torch.bfloat16, 8191), (8, torch.bfloat16, 8192)])
def test_convolution_of_long_runs(native_lib, K, dtype, C):
    """Sizes that fill the machine, where a thread walks its longest runs, against float64 on the GPU."""
    from atlas_rnn_b200 import causal_conv1d
    B, T = 2, 4133
    rn = gen(K)
    x, w, bias = rn(B, T, C).to(dtype).requires_grad_(True), rn(C, K).requires_grad_(True), rn(C).requires_grad_(True)
    init = rn(B, K - 1, C).to(dtype).requires_grad_(True)
    lengths = torch.tensor([T, 1030], device="cuda")
    dy, df = rn(B, T, C).to(dtype), rn(B, K - 1, C).to(dtype)
    y, final = causal_conv1d(x, w, bias, activation="silu", initial_state=init, lengths=lengths)
    got = torch.autograd.grad((y, final), (x, w, bias, init), (dy, df))
    leaf = [t.detach().double().requires_grad_(True) for t in (x, w, bias, init)]
    full = torch.cat([leaf[3], leaf[0]], 1)
    ref = torch.nn.functional.silu(leaf[2] + sum(full[:, j:j + T] * leaf[1][:, j] for j in range(K)))
    ref = ref * (torch.arange(T, device="cuda")[:, None] < lengths[:, None, None])
    ref_f = torch.stack([full[b, e:e + K - 1] for b, e in enumerate(lengths.tolist())])
    want = torch.autograd.grad((ref, ref_f), leaf, (dy.double(), df.double()))
    # as for short rows: 2^-18, half a step of bf16; the parameters' sums of 5163 terms in fp32 by runs, records and CTAs keep
    # to 2^-18 of the sum of their sizes, against a sum that cancels to its square root (1/72 of it): 2^-12
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    rel = lambda a, b: ((a.double() - b).norm() / b.norm()).item()
    assert rel(y, ref) <= 2.0 ** -18 + half and torch.equal(final.double(), ref_f)
    for name, g, r in zip(("x", "w", "bias", "init"), got, want):
        assert rel(g, r) <= (2.0 ** -12 if name in ("w", "bias") else 2.0 ** -18 + half), (name, rel(g, r))


def test_cuts_of_the_time_axis_agree(native_lib):
    """The library's own cut at a size that fills the machine, short and long pieces, and none."""
    x = make(3, 2500, 1536, 1, 16, lengths=(2500, 1111, 0))
    leaves = [x[k].requires_grad_(True) for k in NAMES]
    rn = gen(11)
    w, wh = rn(3, 2500, 1536), rn(3, 1536, 16)
    runs = []
    for chunk in (2528, 0, 64, 1024):  # the first: one piece
        out, h = call(x, chunk=chunk)
        runs.append([out, h, *torch.autograd.grad((out, h), leaves, (w, wh))])
    for r in runs[1:]:
        for name, a, b in zip(("out", "state", *NAMES), r, runs[0]):
            # either side is within tol of the exact result (twice that for gradients, as in the tests of short sequences)
            assert rel_l2(a, b) <= 4 * tol(2500, torch.float32), (name, rel_l2(a, b))
