"""The row operators' C entry points at sizes of zero and past their types, without a device."""
from __future__ import annotations

import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

PKG = Path(__file__).resolve().parents[1] / "pallas-kernel_b200"


@pytest.fixture(scope="module")
def C():
    import build as B  # pallas-kernel_b200/build.py (incremental)
    B.build()
    from tops import _C
    return _C


def test_scan_of_no_batch_rows_has_a_plan(C):
    """Long rows, none of them: the plan divided by the number of blocks (in a process of its own, which that ended)."""
    code = """
import ctypes
from tops import _C as C
a = C.ScanArgs(B=0, T=4096, D=8, N=16, G=1, S=0, dtype=C.BF16)
b = C.ScanBwdArgs(f=a)
L = C.lib()
print(L.tops_gla_ssm_scan_states_size(ctypes.byref(a)), L.tops_gla_ssm_scan_fwd_workspace_size(ctypes.byref(a)),
      L.tops_gla_ssm_scan_bwd_workspace_size(ctypes.byref(b)))
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=PKG, capture_output=True, text=True)
    assert r.returncode == 0, f"exit {r.returncode}: {r.stderr[-300:]}"
    assert r.stdout.split() == ["0", "0", "0"]


def test_scan_without_rows_needs_its_matrix(C):
    """Without rows the kernels still carry states from h0 to ht and read A for it."""
    a = C.ScanArgs(B=1, T=0, D=8, N=16, G=1, S=1, dtype=C.BF16, ht=16)
    assert C.lib().tops_gla_ssm_scan_fwd(ctypes.byref(a), None) == -1
    assert "A" in C.lib().tops_gla_last_error().decode()
    a.ht = None  # nothing to do
    assert C.lib().tops_gla_ssm_scan_fwd(ctypes.byref(a), None) == 0
    n = C.lib().tops_gla_ssm_scan_bwd_workspace_size(ctypes.byref(C.ScanBwdArgs(f=a)))
    assert n > 0
    b = C.ScanBwdArgs(f=a, workspace=256, workspace_bytes=n)
    assert C.lib().tops_gla_ssm_scan_bwd(ctypes.byref(b), None) == -1
    assert "A" in C.lib().tops_gla_last_error().decode()


def test_scan_states_at_any_place(C):
    """Only the forward stores four states at once, and only where N is a multiple of 4 above 8."""
    at = lambda T, N, ht, **kw: C.ScanArgs(B=1, T=T, D=8, N=N, G=1, S=1, dtype=C.BF16, ht=ht, **kw)  # noqa: E731
    L = C.lib()
    for N, ht, ok in ((16, 24, False), (16, 32, True), (8, 24, True), (11, 4, True), (12, 8, False)):
        # the arguments are looked at in order: an unaligned state is refused before what is missing
        assert L.tops_gla_ssm_scan_fwd(ctypes.byref(at(0, N, ht)), None) == -1
        assert ("aligned" not in L.tops_gla_last_error().decode()) == ok
        assert L.tops_gla_ssm_scan_step(ctypes.byref(at(1, N, ht)), None) == -1
        assert "required" in L.tops_gla_last_error().decode()


def test_sizes_past_32_bits_are_refused(C):
    """A row count that wraps would leave most of the output unwritten."""
    from tops.modules import causal_conv1d, causal_conv1d_step, qk_norm_rotary
    from tops.ops.ssm import selective_scan, selective_scan_step
    z = lambda *s: torch.zeros([1] * len(s)).expand(*s)  # noqa: E731
    n, A, D = 2 ** 32 + 8, z(1, 4), 2 ** 32 + 8
    for f in (lambda: causal_conv1d(z(1, n, 1), z(1, 4)), lambda: causal_conv1d(z(n, 1, 1), z(1, 4)),
              lambda: causal_conv1d_step(z(n, 1), z(n, 1, 3), z(1, 4)),
              lambda: selective_scan(z(1, n, 1), z(1, n, 1), A, z(1, n, 4), z(1, n, 4)),
              lambda: selective_scan(z(1, 1, D), z(1, 1, D), z(D, 4), z(1, 1, 4), z(1, 1, 4)),
              lambda: selective_scan_step(z(n, 1), z(n, 1), A, z(n, 4), z(n, 4), z(n, 1, 4)),
              lambda: qk_norm_rotary(z(1, n, 1, 2), z(1, n, 1, 2)), lambda: qk_norm_rotary(z(1, 1, n, 2), z(1, 1, 1, 2))):
        with pytest.raises(ValueError, match="at most"):
            f()
    big = 2 ** 31 - 1
    for name, a in (("tops_gla_causal_conv_fwd", C.ConvArgs(B=1, T=big, D=8, W=4, N=1, dtype=C.BF16, w_dtype=C.BF16)),
                    ("tops_gla_causal_conv_fwd", C.ConvArgs(B=1, T=1, D=big, W=4, N=1, dtype=C.BF16, w_dtype=C.BF16)),
                    ("tops_gla_ssm_scan_fwd", C.ScanArgs(B=1, T=big, D=8, N=4, G=1, S=1, dtype=C.BF16)),
                    ("tops_gla_qk_norm_rotary_fwd", C.QKNormArgs(B=1, T=big, H=1, HK=1, K=8, dtype=C.BF16, w_dtype=C.BF16))):
        assert getattr(C.lib(), name)(ctypes.byref(a), None) == -2, name
        assert "too many" in C.lib().tops_gla_last_error().decode()


def test_launches_go_to_the_tensors_device(monkeypatch):
    from contextlib import contextmanager
    from types import SimpleNamespace
    from tops import _rows
    at, calls = [0], []

    @contextmanager
    def device(d):
        keep, at[0] = at[0], d
        yield
        at[0] = keep

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: at[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_rows._C, "stream_of", lambda t: 100 + t.device)
    monkeypatch.setattr(_rows._C, "call", lambda name, args, stream: calls.append((name, args, stream, at[0])))
    for d in (0, 1):
        _rows.launch("f", "args", SimpleNamespace(device=d, get_device=lambda d=d: d))
    assert calls == [("f", "args", 100, 0), ("f", "args", 101, 1)] and at == [0]
