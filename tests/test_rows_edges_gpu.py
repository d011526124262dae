"""The row operators on the GPU where sizes, offsets, scales and places in memory leave the usual ones."""
from __future__ import annotations

import pytest
import torch

from _rows_ref import close, qk_ref, scan_ref
from test_ssm_scan_gpu import NAMES, _call, _dbl, _mk, _roundings

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


def _used_memory(*shapes):
    """Leaves NaN in the blocks that the next tensors of these shapes are given."""
    held = [torch.full(s, float("nan"), device="cuda") for s in shapes for _ in range(4)]
    del held


@pytest.mark.parametrize("cu,lost,lost_back", [([0, 30, 12, 40], [1], [1, 2]), ([0, 40, 12, 20], [1, 2], [1, 2]),
                                               ([25, 3, 40, 40], [0, 2], [0, 2])])
def test_scan_falling_offsets_leave_nothing_unwritten(cu, lost, lost_back):
    """Wrong rows, but every state and gradient is written: a sequence whose last (first) row another one has keeps its
    initial state (the gradient of its final one)."""
    T, S, ch, N = 40, 3, 64, 16
    t, dout, dht = _mk(32, 1, T, ch, N, 1, torch.float32, S)
    c = {k: v.cuda().requires_grad_() for k, v in t.items()}
    off = torch.tensor(cu, dtype=torch.int32, device="cuda")
    _used_memory((S, ch, N))
    y, ht = _call(c, True, off)
    dht = dht.cuda()
    _used_memory((S, ch, N))
    g = dict(zip(NAMES, torch.autograd.grad([y, ht], [c[k] for k in NAMES], [dout.cuda(), dht])))
    assert all(torch.isfinite(v).all() for v in (y, ht, *g.values()))
    for n in lost:
        assert torch.equal(ht[n], c["h0"][n])
    for n in lost_back:
        assert torch.equal(g["h0"][n], dht[n])


@pytest.mark.parametrize("cu", [[0, 30, 12, 40], [0, 40, 12, 20], [25, 3, 40, 40]])
@pytest.mark.parametrize("D", [64, 37])
def test_conv_falling_offsets_leave_nothing_unwritten(cu, D):
    from tops.modules import causal_conv1d
    r = lambda *s: torch.randn(*s, device="cuda").requires_grad_()  # noqa: E731
    x, w, b, st = r(1, 40, D), r(D, 4), r(D), r(3, D, 3)
    off = torch.tensor(cu, dtype=torch.int32, device="cuda")
    _used_memory((1, 40, D), (3, D, 3), (D, 4))
    y, fin = causal_conv1d(x, w, b, "silu", st, True, off)
    _used_memory((1, 40, D), (3, D, 3), (D, 4))
    g = torch.autograd.grad([y, fin], [x, w, b, st], [torch.ones_like(y), torch.ones_like(fin)])
    assert all(torch.isfinite(v).all() for v in (y, fin, *g))


def _growing(T, ch, N):
    """A > 0: the state grows by exp(A dt) a row; all inputs zero."""
    t, _, _ = _mk(33, 1, T, ch, N, 1, torch.float32, 1, z=False, skip=False, bias=False)
    t["A"], t["dt"] = torch.full((ch, N), 0.7), torch.full((1, T, ch), 0.01)
    t["x"], t["h0"] = torch.zeros(1, T, ch), torch.zeros(1, ch, N)
    return t


def test_scan_growth_of_nothing_over_long_segments():
    """Rows in which the decay's product passes fp32 while the state (the gradient) is zero: as row by row."""
    T, ch, N = 512, 8, 4
    g = torch.Generator().manual_seed(33)
    t = _growing(T, ch, N)
    t["dt"][:, :400] = 4.0  # exp(2.8) a row
    t["x"][:, 400:] = torch.randn(1, 112, ch, generator=g)
    y, ht = _call({k: None if v is None else v.cuda() for k, v in t.items()}, False, None)
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), False, None)
    close("out", y, *r["out"], _roundings(112, N, ch, T))
    close("ht", ht, *r["ht"], _roundings(112, N, ch, T))
    t = _growing(T, ch, N)
    t["dt"][:, 100:] = 4.0
    dout = torch.zeros(1, T, ch)
    dout[:, :100] = torch.randn(1, 100, ch, generator=g)
    c = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    y, _ = _call(c, False, None)
    got = torch.autograd.grad(y, [c[k] for k in ("x", "dt", "A", "B", "C", "h0")], dout.cuda())
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), False, None, _dbl(dout), None)
    for k, v in zip(("x", "dt", "A", "B", "C", "h0"), got):
        close("d" + k, v, *r["d" + k], _roundings(100, N, ch, T))


def test_scan_growth_of_a_small_state():
    """exp(100) over one segment, from 1e-30: the product is in range though its factor is not."""
    T, ch, N = 512, 8, 4
    t = _growing(T, ch, N)
    t["h0"] += 1e-30
    t["dt"][:, :] = 1e-3
    t["dt"][:, 64:128] = 100 / 64 / 0.7
    _, ht = _call({k: None if v is None else v.cuda() for k, v in t.items()}, False, None)
    want = scan_ref(*(_dbl(t[k]) for k in NAMES), False, None)["ht"][0]
    # the exponent, about 100, is a sum of 64 rounded terms, and four roundings more
    assert ((ht.double().cpu() - want).abs() <= 100 * 68 * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("scale,eps", [(1e-14, 0.0), (1e-14, 1e-30), (1e14, 1e-6), (1e-3, 1e-6)])
@pytest.mark.parametrize("K", [64, 33])
def test_qk_norm_backward_of_far_scales(scale, eps, K):
    """1 / rms to the third power is out of fp32's range there, dx is not."""
    from tops.modules import qk_norm_rotary
    g = torch.Generator().manual_seed(34)
    q, dq = torch.randn(1, 7, 2, K, generator=g) * scale, torch.randn(1, 7, 2, K, generator=g)
    Q = q.cuda().requires_grad_()
    y, _ = qk_norm_rotary(Q, q[:, :, :1].cuda(), eps=eps)
    (dx,) = torch.autograd.grad(y, Q, dq.cuda())
    ref = qk_ref(q.double(), None, None, None, None, eps, False, dq.double())
    close("y", y, ref[0], ref[1], 2 * K + 24)
    close("dx", dx, ref[2], ref[3], 2 * K + 24)


def test_a_step_in_place_is_seen_by_the_backward():
    """A prompt's state that a gradient still needs, then a step into it: the backward says so."""
    from tops.modules import causal_conv1d, causal_conv1d_step
    from tops.ops.ssm import selective_scan, selective_scan_step
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    x, w, st = r(2, 9, 16).requires_grad_(), r(16, 4), r(2, 16, 3)
    y, _ = causal_conv1d(x, w, None, None, st)
    with torch.no_grad():
        causal_conv1d_step(x[:, 0], st, w, state_out=st)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    A, B, h = -torch.rand(16, 4, device="cuda"), r(2, 9, 4), r(2, 16, 4)
    y, _ = selective_scan(x, x, A, B, B, initial_state=h)
    with torch.no_grad():
        selective_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], h, state_out=h)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
