"""Which calls the row operators' kernels may take, decided without a device."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD


def test_plain_calls():
    from torch.fx.experimental.proxy_tensor import make_fx
    from tops import _rows
    x = torch.randn(3, 4)
    seen = []

    def see(t):
        seen.append(_rows.plain(None, t))
        return t * 2

    see(x)
    see(torch.nn.Parameter(x))
    assert seen == [True, True]
    torch.jit.trace(see, x, check_trace=False)
    torch.vmap(see)(x)
    torch.func.grad(lambda t: see(t).sum())(x)
    make_fx(see)(x)
    with torch._subclasses.FakeTensorMode() as mode:
        fake = mode.from_tensor(x)
        see(fake)
    see(fake)
    with fwAD.dual_level():
        see(x)
        see(fwAD.make_dual(x, x))
    assert seen[2:] == [False] * 6 + [True, False]


def test_short_convolution_of_fake_cuda_tensors():
    """Shapes go through the module where no memory is behind them (and no kernel is launched on it)."""
    from tops.modules import ShortConvolution
    with torch._subclasses.FakeTensorMode(), torch.device("cuda"):
        m = ShortConvolution(24, 4, bias=True)
        y, cache = m(torch.empty(2, 13, 24, device="cuda"), None, True)
    assert y.shape == (2, 13, 24) and cache.shape == (2, 24, 3) and y.device.type == "cuda"


def test_operators_say_what_they_cannot_follow():
    from torch.fx.experimental.proxy_tensor import make_fx
    from tops.modules import causal_conv1d, causal_conv1d_step, qk_norm_rotary
    from tops.ops.ssm import selective_scan, selective_scan_step
    t = torch.randn
    w, st, A, B, h, k = t(8, 4), t(2, 8, 3), t(8, 4), t(2, 4, 4), t(2, 8, 4), t(2, 4, 2, 8)
    for name, f, x in (("causal_conv1d", lambda v: causal_conv1d(v, w)[0], t(2, 4, 8)),
                       ("causal_conv1d_step", lambda v: causal_conv1d_step(v, st, w)[0], t(2, 8)),
                       ("selective_scan", lambda v: selective_scan(v, v, A, B, B)[0], t(2, 4, 8)),
                       ("selective_scan_step", lambda v: selective_scan_step(v, v, A, B[:, 0], B[:, 0], h)[0], t(2, 8)),
                       ("qk_norm_rotary", lambda v: qk_norm_rotary(v, k)[0], t(2, 4, 2, 8))):
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            torch.jit.trace(f, x, check_trace=False)
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            make_fx(f)(x)
        with pytest.raises(RuntimeError, match=f"{name} .*torch.func"):
            torch.vmap(f)(x[None])
        with torch._subclasses.FakeTensorMode(allow_non_fake_inputs=True) as mode:
            with pytest.raises(RuntimeError, match=f"{name} cannot run on fake"):
                f(mode.from_tensor(x))
        with fwAD.dual_level():
            with pytest.raises(RuntimeError, match=f"{name} has no forward-mode"):
                f(fwAD.make_dual(x, x))


def test_a_state_written_in_place_counts_as_changed():
    from tops import _rows
    h = torch.randn(2, 3, 4)
    x = torch.randn(2, 3, 4, requires_grad=True)
    y = (x * h).sum()  # keeps h for the backward
    assert _rows.state_target("step", h, h)[1] is h
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    out = torch.zeros(2, 3, 4, requires_grad=True)
    with pytest.raises(RuntimeError, match="state_out requires a gradient"):
        _rows.state_target("step", h, out)
    with torch.no_grad():
        assert _rows.state_target("step", h, out)[1] is out
    with torch.inference_mode():
        t = torch.zeros(2, 3, 4)
        assert _rows.state_target("step", t, t)[1] is t
