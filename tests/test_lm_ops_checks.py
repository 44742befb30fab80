"""CPU: argument checks of the language-model operators (they come before any launch, so CPU tensors reach them),
and the layout of their argument records against the header."""
import os
import subprocess
import tempfile

import pytest
import torch

import atlas_rnn_b200 as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def scan_args(b=2, t=3, d=6, g=2, n=4, dtype=torch.float32):
    z = lambda *s: torch.zeros(*s, dtype=dtype)
    return dict(u=z(b, t, d), delta=z(b, t, d), A=torch.zeros(d, n), B=z(b, t, g, n), C=z(b, t, g, n))


def test_scan_argument_record_matches_header():
    from atlas_rnn_b200.selective_scan import _SCAN
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "atlas_mem.h"\nint main(void) {\n' \
           'printf("%zu %zu %zu %zu\\n", sizeof(AtlasSelScan), offsetof(AtlasSelScan, u), offsetof(AtlasSelScan, len),' \
           ' offsetof(AtlasSelScan, dout));\nreturn 0; }\n'
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "t.c"), os.path.join(td, "t")
        open(c, "w").write(prog)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        size, at_u, at_len, at_dout = map(int, subprocess.run([exe], capture_output=True, text=True).stdout.split())
    assert _SCAN.size == size
    fields = list(range(1, 1 + 2 + 5 + 1 + 5 + 12 + 5 + 4 + 2 + 1 + 2 + 10))
    assert len(fields) == len(_SCAN.unpack(bytes(size)))
    marks = [0] * len(fields)
    for where, index in ((at_u, 8), (at_len, 29), (at_dout, 36)):  # u, len, dout
        m = list(marks)
        m[index] = 0x1122
        raw = _SCAN.pack(*m)
        assert int.from_bytes(raw[where:where + 8], "little") == 0x1122, index


def test_scan_without_cuda_is_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        A.selective_scan(**scan_args())


@pytest.mark.parametrize("change, error", [
    (dict(u=torch.zeros(2, 3)), ValueError),
    (dict(u=torch.zeros(2, 3, 6, dtype=torch.float16)), TypeError),
    (dict(delta=torch.zeros(2, 3, 5)), ValueError),
    (dict(delta=torch.zeros(2, 3, 6, dtype=torch.bfloat16)), TypeError),
    (dict(A=torch.zeros(6, 5)), ValueError),
    (dict(A=torch.zeros(6, 4, dtype=torch.int32)), TypeError),
    (dict(B=torch.zeros(2, 3, 4)), ValueError),                       # C has four dimensions
    (dict(B=torch.zeros(2, 3, 4, 4), C=torch.zeros(2, 3, 4, 4)), ValueError),  # 6 channels in 4 groups
    (dict(A=torch.zeros(6, 65), B=torch.zeros(2, 3, 2, 65), C=torch.zeros(2, 3, 2, 65)), ValueError),
    (dict(A=torch.zeros(6, 0), B=torch.zeros(2, 3, 2, 0), C=torch.zeros(2, 3, 2, 0)), ValueError),
    (dict(D=torch.zeros(5)), ValueError),
    (dict(z=torch.zeros(2, 4, 6)), ValueError),
    (dict(delta_bias=torch.zeros(6, 1)), ValueError),
    (dict(initial_state=torch.zeros(2, 4, 6)), ValueError),
    (dict(lengths=torch.zeros(2)), TypeError),
    (dict(lengths=[1, 2]), TypeError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(chunk=33), ValueError),
    (dict(chunk=-32), ValueError),
])
def test_scan_refusals(change, error):
    with pytest.raises(error):
        A.selective_scan(**{**scan_args(), **change})


@pytest.mark.parametrize("change, error", [
    (dict(x=torch.zeros(3, 6)), ValueError),
    (dict(x=torch.zeros(2, 3, 6, dtype=torch.float64)), TypeError),
    (dict(weight=torch.zeros(6, 1)), ValueError),
    (dict(weight=torch.zeros(6, 9)), ValueError),
    (dict(weight=torch.zeros(5, 4)), ValueError),
    (dict(weight=torch.zeros(6, 2, 4)), ValueError),
    (dict(bias=torch.zeros(5)), ValueError),
    (dict(activation="relu"), ValueError),
    (dict(initial_state=torch.zeros(2, 4, 6)), ValueError),
    (dict(initial_state=torch.zeros(2, 3, 6, dtype=torch.bfloat16)), TypeError),
    (dict(lengths=torch.zeros(2)), TypeError),
    (dict(), RuntimeError),
])
def test_conv_refusals(change, error):
    with pytest.raises(error):
        A.causal_conv1d(**{**dict(x=torch.zeros(2, 3, 6), weight=torch.zeros(6, 1, 4)), **change})


def test_native_calls_refuse_bad_arguments(native_lib):
    """The C entries return an error code before any launch."""
    from atlas_rnn_b200.selective_scan import _SCAN
    import ctypes
    s = [ctypes.c_size_t() for _ in range(3)]
    refs = [ctypes.byref(v) for v in s]
    fields = lambda B=1, T=8, D=4, N=16, G=1, dt=0, chunk=0: [B, T, D, N, G, 1, dt, chunk] + [0] * 41
    assert native_lib.atlas_sscan_workspace(None, *refs) == 1
    assert native_lib.atlas_sscan_forward(None, None) == 1 and native_lib.atlas_sscan_backward(None, None) == 1
    assert native_lib.atlas_sscan_workspace(_SCAN.pack(*fields()), *refs) == 0 and s[0].value == 1 * 1 * 4 * 16 * 4
    for bad in (dict(B=0), dict(T=0), dict(D=0), dict(N=0), dict(N=65), dict(G=3), dict(dt=2), dict(chunk=5)):
        assert native_lib.atlas_sscan_workspace(_SCAN.pack(*fields(**bad)), *refs) == 1, bad
    assert native_lib.atlas_sscan_forward(_SCAN.pack(*fields()), None) == 1  # null operands
    assert native_lib.atlas_causal_conv_scratch(1, 8, 4, 9) == 0
    assert native_lib.atlas_causal_conv_forward(*([None, 0, 0] + [None] * 6 + [4, 1, 0, 1, 8, 4, None])) == 1


def test_sample_argument_record_matches_header():
    from atlas_rnn_b200.sampling import _SAMPLE
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "atlas_mem.h"\nint main(void) {\n' \
           'printf("%zu %zu %zu\\n", sizeof(AtlasSample), offsetof(AtlasSample, top_k), offsetof(AtlasSample, dtype));\n' \
           'return 0; }\n'
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "t.c"), os.path.join(td, "t")
        open(c, "w").write(prog)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        size, at_k, at_dtype = map(int, subprocess.run([exe], capture_output=True, text=True).stdout.split())
    assert _SAMPLE.size == size
    raw = _SAMPLE.pack(0, 0, 0, 0, 0, 0, 0, 0.0, 0.0, 0.0, 0x1122, 0, 0, 0, 0, 0x3344)
    assert int.from_bytes(raw[at_k:at_k + 8], "little") == 0x1122
    assert int.from_bytes(raw[at_dtype:at_dtype + 4], "little") == 0x3344


@pytest.mark.parametrize("change, error", [
    (dict(logits=torch.zeros(2, 5, dtype=torch.float16)), TypeError),
    (dict(logits=torch.zeros(())), ValueError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(noise=torch.zeros(2, 4)), ValueError),
    (dict(noise=torch.zeros(2, 5, dtype=torch.float64)), TypeError),
    (dict(temperature=-0.1), ValueError),
    (dict(temperature=float("nan")), ValueError),
    (dict(top_k=-1), ValueError),
    (dict(top_p=1.1), ValueError),
    (dict(top_p=-0.1), ValueError),
    (dict(min_p=2.0), ValueError),
    (dict(top_k=torch.zeros(2)), TypeError),
    (dict(top_p=torch.zeros(2, dtype=torch.int32)), TypeError),
    (dict(temperature=torch.zeros(3)), ValueError),
    (dict(), RuntimeError),
])
def test_sample_refusals(change, error):
    args = dict(logits=torch.zeros(2, 5), noise=torch.zeros(2, 5))
    with pytest.raises(error):
        A.sample_tokens(**{**args, **change})


def test_native_sample_refuses_bad_arguments(native_lib):
    from atlas_rnn_b200.sampling import _SAMPLE
    assert native_lib.atlas_sample_tokens(None, None) == 1
    for rows, V, dt in ((0, 5, 0), (1, 0, 0), (1, 5, 7), (1, 1 << 31, 0)):
        assert native_lib.atlas_sample_tokens(_SAMPLE.pack(16, 16, 16, rows, V, 5, 5, 1.0, 1.0, 0.0, 0, 0, 0, 0, 0, dt), None) == 1
    assert native_lib.atlas_sample_tokens(_SAMPLE.pack(0, 16, 16, 1, 5, 5, 5, 1.0, 1.0, 0.0, 0, 0, 0, 0, 0, 0), None) == 1


def test_distill_argument_record_matches_header():
    from atlas_rnn_b200.distill import _DISTILL
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "atlas_mem.h"\nint main(void) {\n' \
           'printf("%zu %zu %zu\\n", sizeof(AtlasDistill), offsetof(AtlasDistill, rows), offsetof(AtlasDistill, dtype));\n' \
           'return 0; }\n'
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "t.c"), os.path.join(td, "t")
        open(c, "w").write(prog)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        size, at_rows, at_dtype = map(int, subprocess.run([exe], capture_output=True, text=True).stdout.split())
    assert _DISTILL.size == size
    raw = _DISTILL.pack(*[0] * 8, 0x1122, 0, 0, 0, 0.0, 0x3344)
    assert int.from_bytes(raw[at_rows:at_rows + 8], "little") == 0x1122
    assert int.from_bytes(raw[at_dtype:at_dtype + 4], "little") == 0x3344


@pytest.mark.parametrize("change, error", [
    (dict(logits=torch.zeros(2, 5, dtype=torch.float16)), TypeError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(teacher_values=torch.zeros(2, 0)), ValueError),
    (dict(teacher_values=torch.zeros(2, 1025), teacher_indices=torch.zeros(2, 1025, dtype=torch.int64)), ValueError),
    (dict(teacher_values=torch.zeros(2, 3, dtype=torch.int32)), TypeError),
    (dict(teacher_indices=torch.zeros(2, 3)), TypeError),
    (dict(teacher_indices=torch.zeros(2, 4, dtype=torch.int64)), ValueError),
    (dict(teacher_values=torch.zeros(3, 3)), ValueError),
    (dict(temperature=0.0), ValueError),
    (dict(temperature=float("inf")), ValueError),
    (dict(reduction="batchmean"), ValueError),
    (dict(), RuntimeError),
])
def test_distill_refusals(change, error):
    args = dict(logits=torch.zeros(2, 5), teacher_values=torch.zeros(2, 3),
                teacher_indices=torch.zeros(2, 3, dtype=torch.int64))
    with pytest.raises(error):
        A.distill_loss(**{**args, **change})


def test_teacher_without_a_loss_is_refused():
    m = A.RNNMemoryTransformer(num_tokens=8, dim=8, depth=1, heads=1, dim_head=8)
    with pytest.raises(ValueError):
        m(torch.zeros(1, 3, dtype=torch.int64), teacher=(torch.zeros(1, 2, 1), torch.zeros(1, 2, 1, dtype=torch.int64)))


def test_native_distill_refuses_bad_arguments(native_lib):
    from atlas_rnn_b200.distill import _DISTILL
    assert native_lib.atlas_distill_forward(None, None) == 1 and native_lib.atlas_distill_backward(None, None) == 1
    ok = dict(rows=1, V=5, K=2, t=1.0, dt=0)
    for bad in (dict(rows=0), dict(V=0), dict(K=0), dict(K=1025), dict(t=0.0), dict(t=float("nan")), dict(dt=3)):
        f = {**ok, **bad}
        raw = _DISTILL.pack(*[16] * 8, f["rows"], f["V"], f["K"], 5, f["t"], f["dt"])
        assert native_lib.atlas_distill_forward(raw, None) == 1 and native_lib.atlas_distill_backward(raw, None) == 1, bad
    assert native_lib.atlas_distill_forward(_DISTILL.pack(*[0] * 8, 1, 5, 2, 5, 1.0, 0), None) == 1


def vast(*shape, dtype=torch.float32):
    return torch.zeros((), dtype=dtype).expand(*shape)


def test_sizes_beyond_the_kernels_are_refused():
    for b, t, d in ((1, 1 << 31, 1), (1 << 24 | 1, 1, 1), (1, 1, 1 << 30 | 1)):
        r = lambda *s: vast(b, t, *s)
        with pytest.raises(ValueError, match="at most"):
            A.selective_scan(r(d), r(d), vast(d, 4), r(4), r(4))
    for b, t, c in ((1, 1 << 31, 1), (1 << 24 | 1, 1, 1), (1, 1, 1 << 20 | 1)):
        with pytest.raises(ValueError, match="at most"):
            A.causal_conv1d(vast(b, t, c), vast(c, 4))
    with pytest.raises(ValueError, match="at most"):
        A.sample_tokens(vast(1, 1 << 24), vast(1, 1 << 24))
    with pytest.raises(TypeError):
        A.sample_tokens(vast(1, 8), vast(1, 8), top_k=0.5)
    for tau in (1e-7, 1e7, float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            A.distill_loss(vast(1, 8), vast(1, 2), vast(1, 2, dtype=torch.int64), temperature=tau)


def test_native_calls_refuse_unaligned_workspaces(native_lib):
    from atlas_rnn_b200.selective_scan import _SCAN
    f = [1, 8, 4, 16, 1, 1, 0, 0] + [16] * 5 + [0] * 12 + [16, 0, 0, 0] + [0] + [16, 16] + [0] * 17
    assert len(f) == 8 + 41
    saved, scratch = 32, 33  # fields
    for at in (saved, scratch):
        g = list(f)
        g[at] = 24
        assert native_lib.atlas_sscan_forward(_SCAN.pack(*g), None) == 1
