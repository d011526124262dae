"""Which calls the row operators' kernels may take, decided without a device."""
from __future__ import annotations

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
