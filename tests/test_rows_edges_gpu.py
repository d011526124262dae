"""The row operators on the GPU where sizes, offsets, scales and places in memory leave the usual ones."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [0, 5, 300])
def test_no_batch_rows(T):
    """A batch of no rows gives outputs of no rows and parameter gradients of zero."""
    from tops.modules import causal_conv1d, causal_conv1d_step, qk_norm_rotary
    from tops.ops.ssm import selective_scan, selective_scan_step
    D, N = 16, 4
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    x, w, A = z(0, T, D).requires_grad_(), torch.ones(D, 4, device="cuda").requires_grad_(), -torch.ones(D, N, device="cuda")
    A.requires_grad_()
    y, fin = causal_conv1d(x, w, output_final_state=True)
    assert y.shape == (0, T, D) and fin.shape == (0, D, 3)
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert dx.shape == x.shape and not dw.any()
    y, ht = selective_scan(x, x, A, z(0, T, N), z(0, T, N), output_final_state=True)
    assert y.shape == (0, T, D) and ht.shape == (0, D, N)
    dx, dA = torch.autograd.grad(y.sum(), [x, A])
    assert dx.shape == x.shape and not dA.any()
    qw = torch.ones(8, device="cuda").requires_grad_()
    q, _ = qk_norm_rotary(z(0, T, 2, 8), z(0, T, 1, 8), qw)
    assert q.shape == (0, T, 2, 8) and not torch.autograd.grad(q.sum(), qw)[0].any()
    with torch.no_grad():
        assert causal_conv1d_step(z(0, D), z(0, D, 3), w)[0].shape == (0, D)
        assert selective_scan_step(z(0, D), z(0, D), A, z(0, N), z(0, N), z(0, D, N))[0].shape == (0, D)
