"""GPU: sample_tokens (atlas_sample_tokens) against its definition in float64, row by row with numpy: tokens must be
equal. A row could differ only where two scores, or a mass and its cut, are closer than the kernel's resolution: scores are
compared in fp64, masses are exact to 2^-41 of the largest token's and exp's fp32 rounding (2^-23), so a draw is disputed
with a chance of about 1e-6 a row; the inputs here are fixed."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(logits, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    V = logits.shape[-1]
    L = logits.detach().double().cpu().numpy().reshape(-1, V)
    U = noise.detach().double().cpu().numpy().reshape(-1, V)
    pick = lambda v, r: float(v.reshape(-1)[r]) if torch.is_tensor(v) else v
    out = []
    for r in range(L.shape[0]):
        t, k, p, m = (pick(v, r) for v in (temperature, top_k, top_p, min_p))
        l = np.where(np.isnan(L[r]), -np.inf, L[r])
        if not (l > -np.inf).any():
            out.append(0)
            continue
        order = np.lexsort((np.arange(V), -l))
        if k > 0:
            order = order[:int(k)]
        top = l[order[0]]
        with np.errstate(invalid="ignore"):
            w = np.where(l[order] == top, 1.0, np.exp(l[order] - top))
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        ok = (before < p * w.sum()) & (w >= m)
        ok[0] = True
        kept = np.sort(order[ok])
        kept = kept[l[kept] > -np.inf]
        s = l[kept]
        if t > 0:
            s = s / t - np.log(np.maximum(-np.log(np.maximum(U[r][kept], 1e-20)), 1e-20))
        out.append(int(kept[int(np.argmax(s))]))
    return torch.tensor(out).reshape(logits.shape[:-1])


def draw(rows, V, seed, dtype=torch.float32, spread=2.0, masked=1 / 16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda: torch.rand(rows, V, device="cuda", generator=g)
    l = spread * torch.randn(rows, V, device="cuda", generator=g) + 3.0 * (rn() < 40.0 / V)
    l = l.masked_fill(rn() < masked, float("-inf"))
    return l.to(dtype), rn()


SETTINGS = [
    dict(),
    dict(min_p=0.1),
    dict(temperature=0.7, top_k=1),
    dict(temperature=0.0, top_k=20, top_p=0.5),
    dict(temperature=1.3, top_k=50, top_p=0.9, min_p=0.02),
    dict(top_p=0.95, temperature=0.8),
    dict(top_p=0.2),
    dict(top_k=511),
    dict(top_k=700, top_p=0.99),
    dict(top_p=0.0),
    dict(top_p=1e-9, min_p=1.0),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (16, 256), (5, 1000), (2, 4097), (40, 8191), (1, 50001), (3, 131072)])
def test_tokens_equal_the_definition(native_lib, rows, V, dtype):
    from atlas_rnn_b200 import sample_tokens
    for n, cfg in enumerate(SETTINGS):
        l, u = draw(rows, V, 100 * n + V, dtype)
        got = sample_tokens(l, u, **cfg)
        assert got.shape == (rows,) and got.dtype == torch.int64
        assert torch.equal(got.cpu(), reference(l, u, **cfg)), cfg


@pytest.mark.parametrize("V", [700, 20000, 131072])
def test_many_equal_logits(native_lib, V):
    """Ties beyond the list's size: the cut goes down to the index."""
    from atlas_rnn_b200 import sample_tokens
    g = torch.Generator(device="cuda").manual_seed(V)
    u = torch.rand(4, V, device="cuda", generator=g)
    flat = torch.zeros(4, V, device="cuda")
    flat[1] = torch.randint(0, 2, (V,), device="cuda", generator=g).float()
    flat[2] = torch.randint(0, 40, (V,), device="cuda", generator=g).float() / 64
    flat[3, ::2] = -0.0  # the same as 0
    for cfg in (dict(top_k=3), dict(top_k=V // 2 + 1), dict(top_p=0.5), dict(top_k=V - 1, top_p=0.3), dict(top_k=600, min_p=0.5),
                dict(top_p=0.75, min_p=0.3, temperature=0.5), dict(temperature=0.0)):
        for dtype in (torch.float32, torch.bfloat16):
            l = flat.to(dtype)
            assert torch.equal(sample_tokens(l, u, **cfg).cpu(), reference(l, u, **cfg)), (cfg, dtype)


def test_sorted_and_clustered_rows(native_lib):
    """The largest tokens side by side, in one thread's or one CTA's share."""
    from atlas_rnn_b200 import sample_tokens
    V = 70000
    g = torch.Generator(device="cuda").manual_seed(1)
    l = (3 * torch.randn(4, V, device="cuda", generator=g)).sort(dim=-1).values
    l[1] = l[1].flip(0)
    l[2, 8:] = l[2, 8:] - 100.0
    l[3, ::8192] = 60.0
    u = torch.rand(4, V, device="cuda", generator=g)
    for cfg in (dict(top_k=40), dict(top_k=512, top_p=0.9), dict(top_k=5000, top_p=0.9), dict(top_p=0.9), dict(min_p=0.01)):
        assert torch.equal(sample_tokens(l, u, **cfg).cpu(), reference(l, u, **cfg)), cfg


def test_infinities_nan_and_empty_rows(native_lib):
    from atlas_rnn_b200 import sample_tokens
    inf, nan = float("inf"), float("nan")
    V = 300
    l, u = draw(7, V, 3)
    l[0] = -inf
    l[1] = nan
    l[2, 5:] = -inf
    l[3, 17] = l[3, 200] = inf
    l[4, ::3] = nan
    l[5] = -inf
    l[5, 299] = -3e38
    l[6] = torch.finfo(torch.float32).min  # a mask of the type's lowest value everywhere: like any equal logits
    for cfg in (dict(), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.5), dict(temperature=0.0), dict(top_k=2, temperature=0.01)):
        assert torch.equal(sample_tokens(l, u, **cfg).cpu(), reference(l, u, **cfg)), cfg
    assert sample_tokens(l, u)[0] == 0 and sample_tokens(l, u)[5] == 299


def test_extreme_noise_and_temperature(native_lib):
    from atlas_rnn_b200 import sample_tokens
    l, u = draw(6, 500, 4)
    u[0] = 0.0
    u[1] = 1.0 - 2.0 ** -24
    u[2, ::2] = 0.0
    u[3] = 0.5
    u[4, 7] = 1.0
    for t in (1e-6, 0.01, 1.0, 100.0, 1e6):
        assert torch.equal(sample_tokens(l, u, temperature=t).cpu(), reference(l, u, temperature=t)), t
        assert torch.equal(sample_tokens(l, u, temperature=t, top_k=30).cpu(), reference(l, u, temperature=t, top_k=30)), t


def test_settings_per_row(native_lib):
    from atlas_rnn_b200 import sample_tokens
    l, u = draw(64, 9000, 5, torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(6)
    r = lambda: torch.rand(64, device="cuda", generator=g)
    cfg = dict(temperature=(2 * r() - 0.3).clamp(min=0), top_k=(200 * r() - 50).int(), top_p=1.2 * r(), min_p=0.3 * r() - 0.05)
    assert torch.equal(sample_tokens(l, u, **cfg).cpu(), reference(l, u, **cfg))
    cfg["top_k"] = cfg["top_k"].long().clamp(min=0) + (1 << 40) * (r() < 0.2)
    cfg["top_p"] = cfg["top_p"].double()
    got = sample_tokens(l, u, **cfg)
    cfg["top_p"] = cfg["top_p"].float()
    assert torch.equal(got.cpu(), reference(l, u, **cfg))


def test_layouts_streams_and_replay(native_lib):
    from atlas_rnn_b200 import sample_tokens
    l, u = draw(6, 5000, 7)
    cfg = dict(top_k=40, top_p=0.8)
    want = sample_tokens(l, u, **cfg)
    assert torch.equal(sample_tokens(l.view(2, 3, 5000), u.view(2, 3, 5000), **cfg), want.view(2, 3))
    assert sample_tokens(l[0], u[0], **cfg) == want[0]
    wide = torch.zeros(6, 5003, device="cuda")
    wide[:, 3:] = l
    assert torch.equal(sample_tokens(wide[:, 3:], u, **cfg), want)       # unaligned rows
    assert torch.equal(sample_tokens(l.t().contiguous().t(), u, **cfg), want)
    assert sample_tokens(l[:0], u[:0]).shape == (0,)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = sample_tokens(l, u, **cfg)
    s.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(l, u, **cfg)
    l.copy_(l.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, sample_tokens(l, u, **cfg))


def test_frequencies_follow_the_softmax(native_lib):
    """Over many draws each token's share is its probability, within 5 standard deviations."""
    from atlas_rnn_b200 import sample_tokens
    g = torch.Generator(device="cuda").manual_seed(8)
    l = torch.tensor([2.0, 1.0, 0.0, -1.0, 0.5], device="cuda").expand(20000, 5)
    n = torch.bincount(sample_tokens(l, torch.rand(20000, 5, device="cuda", generator=g)), minlength=5).cpu().double()
    p = torch.softmax(l[0].double().cpu(), -1)
    assert ((n - 20000 * p).abs() <= 5 * (20000 * p * (1 - p)).sqrt()).all()


def test_generate_with_top_k_and_top_p(native_lib):
    import atlas_rnn_b200 as A
    torch.manual_seed(0)
    m = A.RNNMemoryTransformer(num_tokens=64, dim=32, depth=1, heads=1, dim_head=32, omega_window=2).cuda()
    prompt = torch.randint(0, 64, (2, 5), device="cuda")
    greedy = m.generate(prompt, max_length=12, temperature=0.0)
    assert torch.equal(m.generate(prompt, max_length=12, temperature=0.0, top_k=10, top_p=0.9), greedy)
    assert torch.equal(m.generate(prompt, max_length=12, temperature=1.0, top_k=1), greedy)
    out = m.generate(prompt, max_length=12, temperature=1.0, top_k=10, top_p=0.9)
    assert out.shape == (2, 12) and torch.equal(out[:, :5], prompt) and (out < 64).all()
