"""The 64-bit references of the short convolution, the selective scan and the query/key norm: their
gradients against differences, on the CPU; and what the C entry points refuse without a device."""
from __future__ import annotations

import ctypes

import pytest
import torch

from _rows_ref import conv_ref, qk_ref, scan_ref


def _differences(f, t, h=1e-6):
    """d f / d t by central differences (f: a scalar of the tensors it closes over)."""
    g = torch.zeros_like(t)
    for i in range(t.numel()):
        at = t.view(-1)
        keep = at[i].item()
        at[i] = keep + h
        up = f()
        at[i] = keep - h
        down = f()
        at[i] = keep
        g.view(-1)[i] = (up - down) / (2 * h)
    return g


def _match(name, got, diff):
    assert torch.allclose(got, diff, atol=1e-7, rtol=1e-6), f"{name}: {(got - diff).abs().max():.2e}"


def _rn(gen, *s):
    return torch.randn(*s, generator=gen, dtype=torch.float64)


@pytest.mark.parametrize("cu", [None, [0, 4, 4, 5]])
@pytest.mark.parametrize("act", [0, 1])
def test_conv_gradients_against_differences(cu, act):
    gen = torch.Generator().manual_seed(3)
    B = 1 if cu else 2
    N = len(cu) - 1 if cu else B
    x, w, b, st = _rn(gen, B, 5, 3), _rn(gen, 3, 4), _rn(gen, 3), _rn(gen, N, 3, 3)
    dy, df = _rn(gen, B, 5, 3), _rn(gen, N, 3, 3)
    f = lambda: sum((r[k][0] * g).sum() for r in [conv_ref(x, w, b, st, act, cu)]  # noqa: E731
                    for k, g in (("y", dy), ("final", df)))
    r = conv_ref(x, w, b, st, act, cu, dy, df)
    for name, t in (("dx", x), ("dw", w), ("db", b), ("dstate", st)):
        _match(name, r[name][0], _differences(f, t))


@pytest.mark.parametrize("cu,G", [(None, 1), (None, 2), ([0, 3, 3, 4, 6], 1)])
def test_scan_gradients_against_differences(cu, G):
    gen = torch.Generator().manual_seed(5)
    B, T, ch, N = (1 if cu else 2), 6, 4, 3
    S = len(cu) - 1 if cu else B
    x, dt, z = (_rn(gen, B, T, ch) for _ in range(3))
    A, D, bias = -torch.rand(ch, N, generator=gen, dtype=torch.float64) - 0.2, _rn(gen, ch), _rn(gen, ch)
    Bm, Cm, h0 = _rn(gen, B, T, G, N), _rn(gen, B, T, G, N), _rn(gen, S, ch, N)
    dout, dht = _rn(gen, B, T, ch), _rn(gen, S, ch, N)
    a = (x, dt, A, Bm, Cm, D, z, bias, h0, True, cu)
    f = lambda: sum((r[k][0] * g).sum() for r in [scan_ref(*a)] for k, g in (("out", dout), ("ht", dht)))  # noqa: E731
    r = scan_ref(*a, dout, dht)
    for name, t in (("dx", x), ("ddt", dt), ("dA", A), ("dB", Bm), ("dC", Cm), ("dD", D), ("dz", z), ("dbias", bias),
                    ("dh0", h0)):
        _match(name, r[name][0], _differences(f, t))


@pytest.mark.parametrize("pairs", [False, True])
def test_qk_norm_gradients_against_differences(pairs):
    gen = torch.Generator().manual_seed(7)
    x, w, dy = _rn(gen, 2, 3, 2, 6), _rn(gen, 6), _rn(gen, 2, 3, 2, 6)
    angle = _rn(gen, 5, 2)
    pos = torch.tensor([[0, 4, 2], [1, 1, 3]])
    a = (angle.cos(), angle.sin(), pos, 1e-3, pairs)
    f = lambda: (qk_ref(x, w, *a)[0] * dy).sum()  # noqa: E731
    _, _, dx, _, dw, _ = qk_ref(x, w, *a, dy)
    _match("dx", dx, _differences(f, x))
    _match("dw", dw, _differences(f, w))


@pytest.fixture(scope="module")
def C():
    import build as B  # pallas-kernel_b200/build.py (incremental)
    B.build()
    from tops import _C
    return _C


def _refused(C, name, args, status, text):
    assert getattr(C.lib(), name)(ctypes.byref(args), None) == status
    assert text in C.lib().tops_gla_last_error().decode()


def _conv(C, **kw):
    a = C.ConvArgs(B=1, T=4, D=8, W=4, N=1, dtype=C.BF16, w_dtype=C.BF16, x=16, w=16, y=16, x_stride_b=32, x_stride_t=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_conv_refusals_without_a_device(C):
    for kw, st, text in (({"W": 5}, -2, "width"), ({"W": 1}, -2, "width"), ({"dtype": 7}, -1, "dtype"),
                         ({"w_dtype": C.F16}, -1, "w_dtype"), ({"activation": 2}, -1, "activation"),
                         ({"N": 2}, -1, "N must equal B"), ({"D": 0}, -1, "dimension"), ({"B": -1}, -1, "dimension"),
                         ({"x": None}, -1, "required"), ({"y": None}, -1, "required"),
                         ({"cu_seqlens": 16, "B": 2, "N": 2}, -1, "B == 1"),
                         ({"cu_seqlens": 16, "N": 0}, -1, "N >= 1")):
        _refused(C, "tops_gla_causal_conv_fwd", _conv(C, **kw), st, text)
    _refused(C, "tops_gla_causal_conv_step", _conv(C), -1, "T must be 1")
    _refused(C, "tops_gla_causal_conv_step", _conv(C, T=1), -1, "required")
    b = C.ConvBwdArgs(f=_conv(C), dy=16, dy_stride_b=32, dy_stride_t=8, dx=16, dw=16)
    assert C.lib().tops_gla_causal_conv_bwd_workspace_size(ctypes.byref(b)) > 0
    _refused(C, "tops_gla_causal_conv_bwd", b, -4, "workspace")


def _scan(C, **kw):
    a = C.ScanArgs(B=1, T=4, D=8, N=16, G=1, S=1, dtype=C.BF16, x=16, dt=16, Bm=16, Cm=16, A=16, y=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_scan_refusals_without_a_device(C):
    for kw, st, text in (({"N": 65}, -2, "64 states"), ({"N": 0}, -2, "64 states"), ({"G": 3}, -1, "multiple of G"),
                         ({"G": 0}, -1, "multiple of G"), ({"dtype": 9}, -1, "dtype"), ({"S": 2}, -1, "S must equal B"),
                         ({"D": 0}, -1, "dimension"), ({"T": -1}, -1, "dimension"), ({"A": None}, -1, "required"),
                         ({"B": 70000, "S": 70000}, -2, "65535"),
                         ({"cu_seqlens": 16, "B": 2, "S": 2}, -1, "B == 1"),
                         ({"cu_seqlens": 16, "S": 0}, -1, "sequences"), ({"ht": 24}, -1, "16-byte"),
                         ({"states": 4}, -1, "16-byte"), ({"workspace": 8}, -1, "16-byte"),
                         ({"D": 70000, "G": 70000}, -2, "65535 groups")):
        _refused(C, "tops_gla_ssm_scan_fwd", _scan(C, **kw), st, text)
    _refused(C, "tops_gla_ssm_scan_step", _scan(C), -1, "T must be 1")
    _refused(C, "tops_gla_ssm_scan_step", _scan(C, T=1), -1, "required")
    b = C.ScanBwdArgs(f=_scan(C, states=16), dout=16, dx=16, ddt=16, dB=16, dC=16)
    assert C.lib().tops_gla_ssm_scan_bwd_workspace_size(ctypes.byref(b)) > 0
    _refused(C, "tops_gla_ssm_scan_bwd", b, -4, "workspace")
    _refused(C, "tops_gla_ssm_scan_bwd", C.ScanBwdArgs(f=_scan(C), dout=16, dx=16, ddt=16, dB=16, dC=16), -1, "states")


def _qk(C, **kw):
    a = C.QKNormArgs(B=1, T=4, H=2, HK=1, K=8, R=4, dtype=C.BF16, w_dtype=C.F32, table_rows=4, q=16, k=16, cos_table=16,
                     sin_table=16, q_out=16, k_out=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_qk_norm_refusals_without_a_device(C):
    for kw, st, text in (({"K": 257}, -2, "256"), ({"R": 3}, -1, "even"), ({"R": 10}, -1, "fit the head"),
                         ({"table_rows": 3}, -1, "more rows"), ({"cos_table": None}, -1, "tables"),
                         ({"w_dtype": C.F16}, -1, "w_dtype"), ({"q_out": None}, -1, "required"),
                         ({"T": -1}, -1, "dimension")):
        _refused(C, "tops_gla_qk_norm_rotary_fwd", _qk(C, **kw), st, text)
    b = C.QKNormBwdArgs(f=_qk(C), dq_out=16, dk_out=16, dq=16, dk=16, dq_weight=16)
    assert C.lib().tops_gla_qk_norm_rotary_bwd_workspace_size(ctypes.byref(b)) > 0
    _refused(C, "tops_gla_qk_norm_rotary_bwd", b, -4, "workspace")


def test_new_struct_layouts_match_ctypes(C, tmp_path):
    import subprocess
    from pathlib import Path
    header = Path(__file__).resolve().parents[1] / "include" / "tops_gla.h"
    structs = {"tops_gla_conv_args": C.ConvArgs, "tops_gla_conv_bwd_args": C.ConvBwdArgs,
               "tops_gla_scan_args": C.ScanArgs, "tops_gla_scan_bwd_args": C.ScanBwdArgs,
               "tops_gla_qk_norm_args": C.QKNormArgs, "tops_gla_qk_norm_bwd_args": C.QKNormBwdArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){"]
    for c, py in structs.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "probe"), str(src)], check=True)
    for line in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.splitlines():
        c, f, n = line.split()
        py = structs[c]
        assert int(n) == (ctypes.sizeof(py) if f == "size" else getattr(py, f).offset), (c, f)


def test_new_ops_refuse_cpu_tensors():
    from tops.modules import causal_conv1d, causal_conv1d_step, qk_norm_rotary
    from tops.ops.ssm import selective_scan, selective_scan_step
    t = torch.randn
    for f in (lambda: causal_conv1d(t(1, 4, 8), t(8, 4)), lambda: causal_conv1d_step(t(1, 8), t(1, 8, 3), t(8, 4)),
              lambda: selective_scan(t(1, 4, 8), t(1, 4, 8), t(8, 4), t(1, 4, 4), t(1, 4, 4)),
              lambda: selective_scan_step(t(1, 8), t(1, 8), t(8, 4), t(1, 4), t(1, 4), t(1, 8, 4)),
              lambda: qk_norm_rotary(t(1, 4, 2, 8), t(1, 4, 2, 8))):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()


def test_rotary_tables_far_positions():
    from tops.modules import rotary_tables
    import math
    cos, sin = rotary_tables(200001, 8)
    assert cos.shape == (200001, 4) and cos.dtype == torch.float32
    want = math.cos(200000.0 * 10000.0 ** (-2 / 8))
    assert abs(cos[200000, 1].item() - want) <= 2.0 ** -24
    with pytest.raises(AssertionError):
        rotary_tables(4, 3)
