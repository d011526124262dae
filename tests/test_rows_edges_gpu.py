"""The row operators on the GPU where sizes, offsets, scales and places in memory leave the usual ones."""
from __future__ import annotations

import pytest
import torch

from _rows_ref import close, scan_ref
from test_ssm_scan_gpu import NAMES, _dbl, _mk, _roundings

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


@pytest.mark.parametrize("ch,N,off", [(30, 11, 0), (30, 11, 330), (6, 3, 18), (32, 16, 2), (5, 8, 41)])
def test_scan_step_in_place_on_a_slice_of_a_cache(ch, N, off):
    """A layer's state inside a larger buffer, wherever it begins."""
    from tops.ops.ssm import selective_scan_step
    t, _, _ = _mk(31, 2, 1, ch, N, 1, torch.bfloat16, 2)
    c = {k: v.cuda() for k, v in t.items()}
    cache = torch.full((3 * 2 * ch * N + off,), 7.0, device="cuda")
    s = cache[off:off + 2 * ch * N].view(2, ch, N)
    s.copy_(c["h0"])
    a = (c["x"][:, 0], c["dt"][:, 0], c["A"], c["B"][:, 0], c["C"][:, 0])
    y, s2 = selective_scan_step(*a, s, c["D"], c["z"][:, 0], c["bias"], True, state_out=s)
    assert s2 is s
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), True, None)
    n = _roundings(1, N, ch, 1)
    close("y", y, r["out"][0][:, 0], r["out"][1][:, 0], n)
    close("state", s, *r["ht"], n)
    rest = torch.cat([cache[:off], cache[off + 2 * ch * N:]])
    assert torch.equal(rest, torch.full_like(rest, 7.0))
