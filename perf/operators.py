"""Performance cases of the language-model operators: the selective state space scan with its
short causal convolution (training, prompts, single tokens), token sampling from given random
numbers, and the distillation loss over a teacher's top logits.

``run`` calls the package's entry points when ``own`` is set, and otherwise computes the same
results with elementary torch operations in 32 bits (64 where sums or borders need it), rounded
once at the end. ``exact`` gives the results from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------

def listed():
    return [
        # one layer's convolution in a training step of a 768-wide model with expansion 2, T 8192
        dict(name="conv_train", op="conv", b=4, t=8192, c=1536, k=4, dtype="bf16", silu=True, lengths=False),
        # a ragged batch in full precision: odd sizes, a carried state, rows of their own lengths
        dict(name="conv_ragged_f32", op="conv", b=3, t=1001, c=201, k=3, dtype="f32", silu=True, lengths=True),
        # the scan of the same layer in the same training step, forward and backward
        dict(name="scan_train", op="scan_train", b=4, t=8192, d=1536, n=16, g=1, dtype="bf16", z=True, lengths=False),
        # a small full-precision model with grouped B and C, no gate, and odd sizes
        dict(name="scan_train_odd_f32", op="scan_train", b=3, t=1021, d=202, n=10, g=2, dtype="f32", z=False,
             lengths=True),
        # one long prompt: few channels in flight, the time axis has to carry the parallelism
        dict(name="scan_prompt_long", op="scan_prompt", b=1, t=65536, d=1536, n=16, g=1, dtype="bf16", z=True,
             lengths=False),
        # a batch of prompts of their own lengths, continued from earlier states
        dict(name="scan_prompt_ragged", op="scan_prompt", b=16, t=1500, d=1536, n=16, g=1, dtype="bf16", z=True,
             lengths=True),
        # one token of one sequence: latency only
        dict(name="step_1", op="step", b=1, d=1536, n=16, g=1, k=4, dtype="bf16"),
        # one token of a full serving batch: the states are the traffic
        dict(name="step_256", op="step", b=256, d=1536, n=16, g=1, k=4, dtype="bf16"),
        # one sequence of a chat: nucleus sampling over a large odd vocabulary in full precision
        dict(name="sample_1", op="sample", rows=1, v=100003, dtype="f32", per_row=False, temperature=0.8, top_k=0,
             top_p=0.95, min_p=0.0),
        # a serving batch, each row with its own settings
        dict(name="sample_64", op="sample", rows=64, v=131072, dtype="bf16", per_row=True, temperature=1.0, top_k=50,
             top_p=0.9, min_p=0.02),
        # a student with a 32k vocabulary over one batch of tokens, forward and backward
        dict(name="distill_32k", op="distill", rows=8192, v=32000, k=64, dtype="bf16", temperature=2.0),
        # the byte-level model, a short batch in full precision
        dict(name="distill_bytes_f32", op="distill", rows=500, v=256, k=17, dtype="f32", temperature=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "scan_train", "scan_train", "scan_prompt", "scan_prompt", "step", "sample", "sample",
                     "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "conv":
        b, c = _log(rng, 1, 16), _log(rng, 8, 4096)
        t = _log(rng, 1, max(2, min(32768, 40_000_000 // (b * c))))
        return dict(op=op, b=b, t=t, c=c, k=rng.randint(2, 8), dtype=dtype, silu=rng.random() < 0.7,
                    lengths=rng.random() < 0.4)
    if op in ("scan_train", "scan_prompt"):
        g = rng.choice([1, 1, 2])
        n = rng.choice([16, 16, rng.randint(1, 40)])
        b, d = _log(rng, 1, 16), g * _log(rng, 16, 1024)
        t = _log(rng, 1, max(2, min(32768, 400_000_000 // (b * d * n))))
        return dict(op=op, b=b, t=t, d=d, n=n, g=g, dtype=dtype, z=rng.random() < 0.7, lengths=rng.random() < 0.4)
    if op == "step":
        g = rng.choice([1, 1, 2])
        return dict(op=op, b=_log(rng, 1, 256), d=g * _log(rng, 16, 768), n=rng.choice([16, rng.randint(1, 40)]),
                    g=g, k=rng.randint(2, 8), dtype=dtype)
    if op == "sample":
        v = _log(rng, 100, 131072)
        return dict(op=op, rows=_log(rng, 1, 64), v=v, dtype=dtype, per_row=rng.random() < 0.5,
                    temperature=rng.choice([0.0, 0.7, 1.0, 1.3]), top_k=rng.choice([0, 1, 20, 300]),
                    top_p=rng.choice([1.0, 0.95, 0.5]), min_p=rng.choice([0.0, 0.1]))
    v = _log(rng, 100, 65536)
    rows = _log(rng, 1, min(8192, 200_000_000 // v))
    return dict(op=op, rows=rows, v=v, k=_log(rng, 1, 256 if v >= 256 else v), dtype=dtype,
                temperature=rng.choice([1.0, 2.0, 0.7]))


# ---- inputs --------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed % (1 << 62))


def _lengths(case, gen):
    """Row lengths from nothing up to all of t (the first row is whole)."""
    if not case["lengths"]:
        return None
    r = torch.randint(0, case["t"] + 1, (case["b"],), device="cuda", generator=gen, dtype=torch.int32)
    r[0] = case["t"]
    return r


def _scan_inputs(case, gen, t):
    """Values as such a layer meets them: A = -(1 .. N) times a learned spread, step sizes from 0.001 to
    0.1 through the bias, B and C side by side in one projection, u and z as halves of another."""
    b, d, n, g, dt = case["b"], case["d"], case["n"], case["g"], _TYPES[case["dtype"]]
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    with_z = case.get("z", True)
    uz = rn(b, t, 2 * d).to(dt)
    bc = rn(b, t, 2 * g * n).to(dt)
    step = torch.exp(torch.rand(d, device="cuda", generator=gen) * math.log(100.0) + math.log(1e-3))
    return dict(u=uz[..., :d], z=uz[..., d:] if with_z else None, delta=(0.5 * rn(b, t, d)).to(dt),
                A=-torch.arange(1, n + 1, device="cuda", dtype=torch.float32) * torch.exp(0.2 * rn(d, n)),
                B=bc[..., :g * n].unflatten(-1, (g, n)), C=bc[..., g * n:].unflatten(-1, (g, n)),
                D=1 + 0.1 * rn(d), delta_bias=torch.log(torch.expm1(step)), initial_state=0.5 * rn(b, d, n))


def prepare(case, seed):
    gen = _gen(seed)
    op = case["op"]
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    s = {"case": case}
    if op in ("conv", "step"):
        b, c, k, dt = case["b"], case.get("c", case.get("d")), case["k"], _TYPES[case["dtype"]]
        t = case.get("t", 1)
        s.update(x=rn(b, t, c).to(dt), weight=rn(c, 1, k) / math.sqrt(k), bias=0.1 * rn(c),
                 conv_state=rn(b, k - 1, c).to(dt))
    if op == "conv":
        s.update(lengths=_lengths(case, gen), dy=rn(b, t, c).to(dt), d_state=rn(b, k - 1, c).to(dt))
        s["leaves"] = [s[n].requires_grad_(True) for n in ("x", "weight", "bias", "conv_state")]
    elif op in ("scan_train", "scan_prompt", "step"):
        t = case.get("t", 1)
        s.update(_scan_inputs(case, gen, t), lengths=_lengths(case, gen) if "lengths" in case else None)
        if op == "scan_train":
            s.update(dout=rn(case["b"], t, case["d"]).to(s["u"].dtype), d_state=rn(case["b"], case["d"], case["n"]))
            names = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial_state")
            s["leaves"] = [s[n].requires_grad_(True) for n in names if s[n] is not None]
    elif op == "sample":
        rows, v = case["rows"], case["v"]
        # a peaked head over a wide tail, one token in sixteen masked out
        logits = 2.0 * rn(rows, v) + 3.0 * (torch.rand(rows, v, device="cuda", generator=gen) < 40.0 / v)
        masked = torch.rand(rows, v, device="cuda", generator=gen) < 1 / 16
        s["logits"] = logits.masked_fill_(masked, float("-inf")).to(_TYPES[case["dtype"]])
        s["noise"] = torch.rand(rows, v, device="cuda", generator=gen)
        s["settings"] = {n: case[n] for n in ("temperature", "top_k", "top_p", "min_p")}
        if case["per_row"]:  # each request's own, around the case's
            r = lambda: torch.rand(rows, device="cuda", generator=gen)
            s["settings"] = dict(temperature=case["temperature"] * (0.5 + r()),
                                 top_k=(case["top_k"] * 2 * r()).to(torch.int32),
                                 top_p=1 - (1 - case["top_p"]) * 2 * r(), min_p=case["min_p"] * 2 * r())
    else:
        rows, v, k = case["rows"], case["v"], case["k"]
        s["logits"] = (2.0 * rn(rows, v)).to(_TYPES[case["dtype"]]).requires_grad_(True)
        base = torch.randint(0, v, (rows, 1), device="cuda", generator=gen)
        stride = 2 * torch.randint(0, max(1, v // (2 * k) // 2), (rows, 1), device="cuda", generator=gen) + 1
        at = (base + stride * torch.arange(k, device="cuda")) % v
        # rows with fewer entries than k, and now and then a row without any
        count = torch.randint(1, k + 1, (rows, 1), device="cuda", generator=gen)
        count = torch.where(torch.rand(rows, 1, device="cuda", generator=gen) < 0.05, 0, count)
        s["indices"] = torch.where(torch.arange(k, device="cuda") < count, at, -1)
        s["values"] = 3.0 + 2.0 * rn(rows, k)
        s["dloss"] = rn(rows)
    return s


# ---- the plain forms -----------------------------------------------------------------------

def _linear_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, by doubling."""
    s, t = 1, a.shape[1]
    while s < t:
        b2 = b.clone()
        b2[:, s:].addcmul_(a[:, s:], b[:, :-s])
        b = b2
        if 2 * s < t:
            a2 = a.clone()
            a2[:, s:].mul_(a[:, :-s])
            a = a2
        s *= 2
    return b


def _live(s, t):
    """[b, t, 1]: whether a row is within its sequence's length."""
    at = torch.arange(t, device="cuda")
    return None if s["lengths"] is None else (at < s["lengths"][:, None])[..., None]


def _over_channels(x, d):
    """[b, t, g, n] -> [b, t, d, n] in 32 bits."""
    return x.float().repeat_interleave(d // x.shape[2], dim=2)


def _plain_scan(s, grads):
    case = s["case"]
    d, g, n = case["d"], case["g"], case["n"]
    u, delta, A, h0 = s["u"].float(), s["delta"].float(), s["A"], s["initial_state"]
    z = None if s["z"] is None else s["z"].float()
    t = u.shape[1]
    live = _live(s, t)
    keep = (lambda x: x) if live is None else (lambda x: torch.where(live, x, 0.0))
    x = delta + s["delta_bias"]
    dt = keep(x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())))
    Bd, Cd = _over_channels(s["B"], d), _over_channels(s["C"], d)
    a = torch.exp(dt[..., None] * A)
    b = (dt * u)[..., None] * Bd
    b[:, 0] += a[:, 0] * h0
    h = _linear_scan(a, b)
    del b
    y = (h * Cd).sum(-1) + s["D"] * u
    sg = None if z is None else 1 / (1 + torch.exp(-z))
    out = keep(y if z is None else y * z * sg).to(s["u"].dtype)
    if not grads:
        return out, h[:, -1]
    dout = keep(s["dout"].float())
    dy = dout if z is None else dout * z * sg
    gr = dy[..., None] * Cd
    gr[:, -1] += s["d_state"]
    nxt = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    gr = _linear_scan(nxt.flip(1), gr.flip(1)).flip(1)
    del nxt
    per_group = lambda v: v.unflatten(2, (g, d // g)).sum(3)
    dC = per_group(h * dy[..., None]).to(s["C"].dtype)
    dB = per_group(gr * (dt * u)[..., None]).to(s["B"].dtype)
    s1 = (gr * Bd).sum(-1)
    gah = torch.cat([h0[:, None], h[:, :-1]], 1).mul_(a).mul_(gr)
    dA = (gah * dt[..., None]).sum((0, 1))
    ddelta = keep(((gah * A).sum(-1) + u * s1) / (1 + torch.exp(-x)))
    got = [(dt * s1 + s["D"] * dy).to(s["u"].dtype), ddelta.to(s["delta"].dtype), dA, dB, dC, (dy * u).sum((0, 1))]
    if z is not None:
        got.append((dout * y * sg * (1 + z * (1 - sg))).to(s["z"].dtype))
    return [out, h[:, -1]] + got + [ddelta.sum((0, 1)), a[:, 0] * gr[:, 0]]


def _plain_conv(s, silu, grads):
    x, w, st = s["x"].float(), s["weight"].float()[:, 0], s["conv_state"].float()
    t, k = x.shape[1], w.shape[-1]
    live = _live(s, t)
    keep = (lambda v: v) if live is None else (lambda v: torch.where(live, v, 0.0))
    full = torch.cat([st, x], 1)  # x[t] is full[t + k - 1]
    windows = full.unfold(1, k, 1)
    pre = (windows * w).sum(-1) + s["bias"]
    sg = 1 / (1 + torch.exp(-pre))
    y = keep(pre * sg if silu else pre).to(s["x"].dtype)
    ends = s["lengths"].long() if live is not None else torch.full((x.shape[0],), t, device="cuda")
    last = (ends[:, None] + torch.arange(k - 1, device="cuda"))[..., None].expand(-1, -1, x.shape[-1])
    final = full.gather(1, last).to(s["x"].dtype)
    if not grads:
        return y, final
    dp = keep(s["dy"].float())
    if silu:
        dp = dp * sg * (1 + pre * (1 - sg))
    pad = torch.nn.functional.pad(dp, (0, 0, k - 1, k - 1))
    dfull = (pad.unfold(1, k, 1) * w.flip(-1)).sum(-1)
    dfull = dfull.scatter_add(1, last, s["d_state"].float())
    dw = (windows * dp[..., None]).sum((0, 1))
    return [y, final, dfull[:, k - 1:].to(s["x"].dtype), dw[:, None], dp.sum((0, 1)),
            dfull[:, :k - 1].to(s["x"].dtype)]


def _column(v, dtype=torch.float64):
    return v.to(dtype)[:, None] if torch.is_tensor(v) else v


def _plain_sample(s):
    """In 64 bits: a token next to a border must fall on its own side."""
    p = {n: _column(v) for n, v in s["settings"].items()}
    v = s["logits"].shape[-1]
    l, order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    w = torch.exp(l - l[:, :1])
    rank = torch.arange(v, device="cuda")
    k = torch.as_tensor(p["top_k"], device="cuda")
    keep = ((k <= 0) | (rank < k)).expand_as(l)
    w = torch.where(keep, w, 0.0)
    before = torch.cumsum(w, -1) - w
    keep = keep & ((before < p["top_p"] * w.sum(-1, keepdim=True)) | (rank == 0))
    keep = keep & ((w >= p["min_p"]) | (rank == 0))
    noise = s["noise"].double().gather(1, order).clamp(min=1e-20)
    gumbel = -torch.log((-torch.log(noise)).clamp(min=1e-20))
    temp = torch.as_tensor(p["temperature"], device="cuda", dtype=torch.float64)
    score = torch.where(temp > 0, l / temp + gumbel, l)
    score = torch.where(keep, score, float("-inf"))
    at = torch.where(score == score.amax(-1, keepdim=True), order, v).amin(-1)
    return at


def _plain_distill(s):
    tau = s["case"]["temperature"]
    x, at = s["logits"].float() / tau, s["indices"]
    there = at >= 0
    tv = torch.where(there, s["values"] / tau, float("-inf"))
    some = there.any(-1, keepdim=True)
    top = torch.where(some, tv.amax(-1, keepdim=True), 0.0)
    e = torch.exp(tv - top)
    total = torch.where(some, e.sum(-1, keepdim=True), 1.0)
    p = e / total
    m = x.amax(-1, keepdim=True)
    lse = torch.log(torch.exp(x - m).sum(-1, keepdim=True))
    logq = x.gather(1, at.clamp(min=0)) - m - lse
    logp = torch.where(there, tv - top, 0.0) - torch.log(total)
    loss = tau * tau * (p * (logp - logq)).sum(-1)
    grad = torch.where(some, torch.exp(x - m - lse), 0.0).scatter_add_(1, at.clamp(min=0), -p)
    grad *= (s["dloss"] * tau)[:, None]
    return loss, grad.to(s["logits"].dtype)


# ---- one pass ------------------------------------------------------------------------------

def _scan_call(s):
    from atlas_rnn_b200 import selective_scan
    return selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"], delta_bias=s["delta_bias"],
                          delta_softplus=True, initial_state=s["initial_state"], lengths=s["lengths"])


def _conv_call(s, silu, lengths):
    from atlas_rnn_b200 import causal_conv1d
    return causal_conv1d(s["x"], s["weight"], s["bias"], activation="silu" if silu else None,
                         initial_state=s["conv_state"], lengths=lengths)


def _run_own(s):
    op = s["case"]["op"]
    if op == "conv":
        y, final = _conv_call(s, s["case"]["silu"], s["lengths"])
        return [y, final, *torch.autograd.grad((y, final), s["leaves"], (s["dy"], s["d_state"]))]
    if op == "scan_train":
        out, final = _scan_call(s)
        return [out, final, *torch.autograd.grad((out, final), s["leaves"], (s["dout"], s["d_state"]))]
    if op == "distill":
        from atlas_rnn_b200 import distill_loss
        loss = distill_loss(s["logits"], s["values"], s["indices"], temperature=s["case"]["temperature"],
                            reduction="none")
        return [loss, *torch.autograd.grad(loss, [s["logits"]], s["dloss"])]
    with torch.no_grad():
        if op == "scan_prompt":
            return list(_scan_call(s))
        if op == "step":
            return [*_conv_call(s, True, None), *_scan_call(s)]
        from atlas_rnn_b200 import sample_tokens
        return [sample_tokens(s["logits"], s["noise"], **s["settings"])]


@torch.no_grad()
def _run_plain(s):
    op = s["case"]["op"]
    if op == "conv":
        return _plain_conv(s, s["case"]["silu"], True)
    if op == "scan_train":
        return _plain_scan(s, True)
    if op == "scan_prompt":
        return list(_plain_scan(s, False))
    if op == "step":
        return [*_plain_conv(s, True, False), *_plain_scan(s, False)]
    if op == "sample":
        return [_plain_sample(s)]
    return list(_plain_distill(s))


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    op, size = case["op"], {"bf16": 2, "f32": 4}[case["dtype"]]

    def conv(b, t, c, k, train):
        rows = b * t * c
        states = 2 * b * (k - 1) * c * size
        # forward x -> y; backward x, dy -> dx
        return (rows * size * (5 if train else 2) + states * (2 if train else 1) + 4 * c * (k + 1) * (3 if train else 1),
                rows * k * (6 if train else 2))

    def scan(b, t, d, n, g, z, train):
        rows = b * t * d
        wide, narrow = (4 if z else 3), 2 * b * t * g * n  # u, delta, z, out; B, C
        nbytes = rows * size * wide + narrow * size + 2 * 4 * b * d * n + 4 * d * (n + 2)
        if train:  # u, delta, z, dout, B, C again; du, ddelta, dz, dB, dC out; the states' gradients
            nbytes += rows * size * (7 if z else 5) + 2 * narrow * size + 2 * 4 * b * d * n + 2 * 4 * d * (n + 2)
        return nbytes, rows * n * (22 if train else 8)  # an exponential counts as one

    if op == "conv":
        nbytes, flops = conv(case["b"], case["t"], case["c"], case["k"], True)
    elif op in ("scan_train", "scan_prompt"):
        nbytes, flops = scan(case["b"], case["t"], case["d"], case["n"], case["g"], case["z"], op == "scan_train")
    elif op == "step":
        one = conv(case["b"], 1, case["d"], case["k"], False)
        two = scan(case["b"], 1, case["d"], case["n"], case["g"], True, False)
        nbytes, flops = one[0] + two[0], one[1] + two[1]
    elif op == "sample":
        cells = case["rows"] * case["v"]
        # the noise of the tokens that can be drawn: top-k of them, or all
        noise = case["rows"] * (case["top_k"] or case["v"]) * 4
        nbytes, flops = cells * size + noise + 8 * case["rows"], 4 * cells
    else:
        cells = case["rows"] * case["v"]
        nbytes = 3 * cells * size + 2 * case["rows"] * case["k"] * 12 + 8 * case["rows"]
        flops = 8 * cells
    return {"bytes": int(nbytes), "flops": int(flops)}


# ---- the definitions in 64 bits ------------------------------------------------------------

def _exact_scan(s, grads):
    """Step by step, as the recurrence is written."""
    case = s["case"]
    f = lambda x: x.detach().double()
    u, A, h = f(s["u"]), f(s["A"]), f(s["initial_state"]).clone()
    bsz, t, d = u.shape
    g, n = case["g"], case["n"]
    x = f(s["delta"]) + f(s["delta_bias"])
    dt = torch.logaddexp(x, torch.zeros_like(x))
    ends = torch.full((bsz,), t, device="cuda") if s["lengths"] is None else s["lengths"].long()
    live = (torch.arange(t, device="cuda")[None] < ends[:, None]).double()[..., None]
    dt = dt * live
    dtu = dt * u
    each = lambda m, i: f(m[:, i])[:, :, None].expand(-1, -1, d // g, -1).reshape(bsz, d, n)
    y = torch.empty_like(u)
    hist = [] if grads else None
    for i in range(t):
        if grads:
            hist.append(h)
        h = torch.exp(dt[:, i, :, None] * A) * h + dtu[:, i, :, None] * each(s["B"], i)
        y[:, i] = torch.einsum("bdn,bdn->bd", h, each(s["C"], i))
    final = h
    y = y + f(s["D"]) * u
    gate = torch.ones_like(u) if s["z"] is None else f(s["z"]) * torch.sigmoid(f(s["z"]))
    out = y * gate * live
    if not grads:
        return out, final
    dout = f(s["dout"]) * live
    dy = dout * gate
    q = f(s["d_state"]).clone()
    du, ddt = f(s["D"]) * dy, torch.zeros_like(u)
    dA = torch.zeros_like(A)
    dB = torch.zeros(bsz, t, g, n, device="cuda", dtype=torch.float64)
    dC = torch.zeros_like(dB)
    cut = lambda m: m.view(bsz, g, d // g, n).sum(2)
    for i in reversed(range(t)):
        before = hist.pop()
        Bi = each(s["B"], i)
        decay = torch.exp(dt[:, i, :, None] * A)
        carried = decay * before
        after = carried + dtu[:, i, :, None] * Bi
        q = q + dy[:, i, :, None] * each(s["C"], i)
        dC[:, i] = cut(after * dy[:, i, :, None])
        dB[:, i] = cut(q * dtu[:, i, :, None])
        inner = torch.einsum("bdn,bdn->bd", q, Bi)
        du[:, i] += dt[:, i] * inner
        flow = q * carried
        ddt[:, i] = torch.einsum("bdn,dn->bd", flow, A) + u[:, i] * inner
        dA += torch.einsum("bdn,bd->dn", flow, dt[:, i])
        q = q * decay
    ddelta = ddt * torch.sigmoid(x) * live
    got = [out, final, du, ddelta, dA, dB, dC, (dy * u).sum((0, 1))]
    if s["z"] is not None:
        zz = f(s["z"])
        sg = torch.sigmoid(zz)
        got.append(dout * y * (sg + zz * sg * (1 - sg)))
    return got + [ddelta.sum((0, 1)), q]


def _exact_conv(s, silu, grads):
    """By torch's differentiation of the definition."""
    f = lambda v: v.detach().double().requires_grad_(grads)
    x, w, bias, st = f(s["x"]), f(s["weight"]), f(s["bias"]), f(s["conv_state"])
    with torch.enable_grad():
        full = torch.cat([st, x], 1)
        t, k = x.shape[1], w.shape[-1]
        pre = bias + 0.0
        pre = sum(full[:, j:j + t] * w[:, 0, j] for j in range(k)) + pre
        y = pre * torch.sigmoid(pre) if silu else pre
        ends = [t] * x.shape[0] if s.get("lengths") is None else s["lengths"].tolist()
        y = torch.stack([torch.cat([y[i, :e], torch.zeros_like(y[i, e:])]) for i, e in enumerate(ends)])
        final = torch.stack([full[i, e:e + k - 1] for i, e in enumerate(ends)])
        if not grads:
            return y, final
        return [y.detach(), final.detach(),
                *torch.autograd.grad((y, final), (x, w, bias, st), (s["dy"].double(), s["d_state"].double()))]


def _exact_sample(s):
    rows = []
    for r in range(s["logits"].shape[0]):
        p = {n: float(v[r]) if torch.is_tensor(v) else v for n, v in s["settings"].items()}
        l = s["logits"][r].double().cpu().numpy()
        u = np.maximum(s["noise"][r].double().cpu().numpy(), 1e-20)
        order = np.lexsort((np.arange(l.size), -l))
        if p["top_k"] > 0:
            order = order[:int(p["top_k"])]
        mass = np.exp(l[order] - l[order[0]])
        below = np.concatenate([[0.0], np.cumsum(mass)[:-1]])
        ok = (below < p["top_p"] * mass.sum()) & (mass >= p["min_p"])
        ok[0] = True
        left = np.sort(order[ok])
        score = l[left]
        if p["temperature"] > 0:
            score = score / p["temperature"] - np.log(np.maximum(-np.log(u[left]), 1e-20))
        rows.append(int(left[int(np.argmax(score))]))
    return torch.tensor(rows)


def _exact_distill(s):
    tau = s["case"]["temperature"]
    with torch.enable_grad():
        x = s["logits"].detach().double().requires_grad_(True)
        logq = torch.log_softmax(x / tau, -1)
        there = s["indices"] >= 0
        row = torch.arange(x.shape[0], device="cuda")[:, None].expand_as(there)[there]
        tv = s["values"].double() / tau
        denom = torch.zeros(x.shape[0], device="cuda", dtype=torch.float64)
        shift = tv.amax(-1)
        denom = denom.index_add(0, row, torch.exp(tv[there] - shift[row]))
        logp = tv[there] - shift[row] - torch.log(denom[row])
        term = torch.exp(logp) * (logp - logq[row, s["indices"][there]])
        loss = tau ** 2 * torch.zeros_like(denom).index_add(0, row, term)
        return [loss.detach(), *torch.autograd.grad(loss, [x], s["dloss"].double())]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "conv":
        return _exact_conv(s, case["silu"], True)
    if op == "distill":
        return _exact_distill(s)
    with torch.no_grad():
        if op == "sample":
            return [_exact_sample(s)]
        if op == "step":
            return [*_exact_conv(s, True, False), *_exact_scan(s, False)]
        return list(_exact_scan(s, op == "scan_train"))
