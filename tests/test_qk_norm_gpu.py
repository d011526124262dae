"""qk_norm_rotary on the GPU against its formula in 64 bits, and the operators around the recurrences in a run
together, as a token mixer uses them."""
from __future__ import annotations

import pytest
import torch

from _rows_ref import close, qk_ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _roundings(K):
    return 2 * K + 24  # the mean of K squares, its root, the weight, two products and a sum of the rotation


def _mk(seed, B, T, H, HK, K, dt, wdt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [rn(B, T, H, K).to(dt), rn(B, T, HK, K).to(dt), (1 + rn(K) / 4).to(wdt), (1 + rn(K) / 4).to(wdt),
            rn(B, T, H, K).to(dt), rn(B, T, HK, K).to(dt)]


def _dbl(t):
    return None if t is None else t.double().cpu()


def _check(q, k, qw, kw, dq, dk, R, pairs, pos, eps=1e-6, call_q=None, call_k=None):
    from tops.modules import qk_norm_rotary, rotary_tables
    B, T = q.shape[:2]
    cos = sin = None
    if R:
        cos, sin = rotary_tables(4096, R, device="cuda")
    leaf = lambda t: None if t is None else t.cuda().requires_grad_()  # noqa: E731
    Q, K_ = leaf(q) if call_q is None else call_q, leaf(k) if call_k is None else call_k
    QW, KW = leaf(qw), leaf(kw)
    yq, yk = qk_norm_rotary(Q, K_, QW, KW, cos, sin, None if pos is None else pos.cuda(), eps, pairs)
    leaves = [t for t in (Q, K_, QW, KW) if t is not None]
    got = iter(torch.autograd.grad([yq, yk], leaves, [dq.cuda(), dk.cuda()]))
    n = _roundings(q.shape[-1])
    at = torch.arange(T).expand(B, T) if pos is None else pos.long().expand(B, T)
    for name, x, w, y, d in (("q", q, qw, yq, dq), ("k", k, kw, yk, dk)):
        ref = qk_ref(_dbl(x), _dbl(w), _dbl(cos), _dbl(sin), at, eps, pairs, _dbl(d))
        close(name, y, ref[0], ref[1], n)
        close("d" + name, next(got), ref[2], ref[3], n)
        if name == "q":
            rq = ref
        else:
            rk = ref
    for name, w, ref in (("dqw", qw, rq), ("dkw", kw, rk)):
        if w is not None:
            close(name, next(got), ref[4], ref[5], n + B * T * max(q.shape[2], k.shape[2]))
    return yq, yk


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B,T,H,HK,K,R", [(1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (1, 37, 16, 4, 128, 64),
                                          (2, 5, 3, 3, 96, 48), (1, 7, 2, 1, 256, 256), (2, 9, 5, 2, 33, 20),
                                          (1, 4, 2, 2, 128, 0), (3, 11, 1, 1, 80, 32), (1, 3, 2, 1, 255, 254)])
@pytest.mark.parametrize("pairs", [False, True])
def test_qk_norm(dt, B, T, H, HK, K, R, pairs):
    _check(*_mk(1, B, T, H, HK, K, DT[dt]), R, pairs, None)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_qk_norm_positions(dt, wide):
    a = _mk(2, 3, 5, 4, 2, 64, DT[dt], DT[dt])
    pos = torch.randint(0, 4096, (3, 5), generator=torch.Generator().manual_seed(1)).to(wide)
    _check(*a, 64, False, pos)
    _check(*a, 32, True, pos[0].contiguous())


def test_qk_norm_without_weights_and_a_row_of_zeros():
    a = _mk(3, 2, 6, 2, 2, 64, torch.float32)
    a[0][0, 0] = 0
    a[2] = a[3] = None
    _check(*a, 64, False, None, eps=1e-5)
    b = _mk(3, 2, 6, 2, 2, 64, torch.bfloat16)
    b[2] = None
    _check(*b, 64, False, None)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("off", [0, 3])
def test_qk_norm_slices_of_one_projection(dt, off):
    q, k, qw, kw, dq, dk = _mk(4, 2, 13, 4, 2, 64, DT[dt])
    wide = torch.zeros(2, 13, 8 * 64 + 8, dtype=DT[dt], device="cuda")
    wide[..., off:off + 256] = q.flatten(2).cuda()
    wide[..., off + 256:off + 384] = k.flatten(2).cuda()
    Q = wide[..., off:off + 256].unflatten(-1, (4, 64)).detach().requires_grad_()
    K = wide[..., off + 256:off + 384].unflatten(-1, (2, 64)).detach().requires_grad_()
    _check(q, k, qw, kw, dq, dk, 64, False, None, call_q=Q, call_k=K)
    # heads before rows
    Q = q.cuda().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    _check(q, k, qw, kw, dq, dk, 64, False, None, call_q=Q, call_k=K)


def test_qk_norm_position_outside_the_tables():
    from tops.modules import qk_norm_rotary, rotary_tables
    q, k, qw, kw, dq, dk = (t.cuda() for t in _mk(5, 1, 4, 2, 1, 64, torch.float32))
    cos, sin = rotary_tables(8, 32, device="cuda")
    pos = torch.tensor([[0, 8, -1, 7]], device="cuda")
    Q = q.clone().requires_grad_()
    y, yk = qk_norm_rotary(Q, k, qw, kw, cos, sin, pos)
    (g,) = torch.autograd.grad(y, Q, dq)
    bad, good = y[:, 1:3], y[:, ::3]
    assert torch.isnan(bad[..., :32]).all() and torch.isfinite(bad[..., 32:]).all()
    assert torch.isfinite(good).all() and torch.isfinite(g[:, ::3]).all() and torch.isnan(yk[:, 1, :, :32]).all()


def test_qk_norm_many_tokens_and_one():
    """Units of several heads (many tokens) and of one (few) give the same bits."""
    from tops.modules import qk_norm_rotary, rotary_tables
    q, k, qw, kw, _, _ = (t.cuda() for t in _mk(6, 4, 1200, 16, 4, 64, torch.bfloat16))
    cos, sin = rotary_tables(1200, 64, device="cuda")
    y, yk = qk_norm_rotary(q, k, qw, kw, cos, sin)
    for t in (0, 7, 1199):
        pos = torch.full((4, 1), t, dtype=torch.int32, device="cuda")
        a, b = qk_norm_rotary(q[:, t:t + 1], k[:, t:t + 1], qw, kw, cos, sin, pos)
        assert torch.equal(a, y[:, t:t + 1]) and torch.equal(b, yk[:, t:t + 1])


def test_qk_norm_empty_and_refusals():
    from tops.modules import qk_norm_rotary, rotary_tables
    q, k, qw, kw, _, _ = (t.cuda() for t in _mk(7, 1, 4, 2, 1, 64, torch.float32))
    cos, sin = rotary_tables(8, 32, device="cuda")
    a, b = qk_norm_rotary(q[:, :0].requires_grad_(), k[:, :0], qw.requires_grad_(), kw, cos, sin)
    assert a.shape == (1, 0, 2, 64)
    assert not torch.autograd.grad(a.sum(), qw)[0].any()
    q, qw = q.detach(), qw.detach()
    for err, f in ((TypeError, lambda: qk_norm_rotary(q, k.half(), qw, kw)),
                   (TypeError, lambda: qk_norm_rotary(q, k, qw.half(), kw)),
                   (TypeError, lambda: qk_norm_rotary(q.double(), k.double())),
                   (AssertionError, lambda: qk_norm_rotary(q, k[:, :2], qw, kw)),
                   (AssertionError, lambda: qk_norm_rotary(q, k, qw[:3], kw)),
                   (AssertionError, lambda: qk_norm_rotary(q, k, qw, kw, cos)),
                   (AssertionError, lambda: qk_norm_rotary(q, k, qw, kw, cos[:3], sin[:3])),
                   (AssertionError, lambda: qk_norm_rotary(q[..., :8], k[..., :8], None, None, cos, sin)),
                   (AssertionError, lambda: qk_norm_rotary(q, k, qw, kw, cos, sin, torch.zeros(3, dtype=torch.int32, device="cuda"))),
                   (TypeError, lambda: qk_norm_rotary(q, k, qw, kw, cos, sin, torch.zeros(4, device="cuda"))),
                   (TypeError, lambda: qk_norm_rotary(q, k, qw, kw, cos.half(), sin.half())),
                   (RuntimeError, lambda: qk_norm_rotary(q, k, qw, kw, cos.cpu(), sin.cpu())),
                   (ValueError, lambda: qk_norm_rotary(q.new_zeros(1, 4, 2, 257), k.new_zeros(1, 4, 1, 257)))):
        with pytest.raises(err):
            f()


def test_mixers_prompt_then_steps():
    """projection -> short convolution -> norm and rotation -> chunk GLA, and projection -> short convolution ->
    selective scan: a packed batch of prompts with its gradients runs, and a prompt continued token by token
    from its states gives what the whole prompt gives."""
    from tops.modules import causal_conv1d, causal_conv1d_step, qk_norm_rotary, rotary_tables
    from tops.ops.gla import fused_recurrent_gla
    from tops.ops.simple_gla import chunk_simple_gla
    from tops.ops.ssm import selective_scan, selective_scan_step
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    B, T, H, K, N = 2, 70, 2, 64, 16
    Dm = H * K
    x = rn(B, T, 3 * Dm)
    w, b = rn(3 * Dm, 4) / 2, rn(3 * Dm) / 4
    qw, kw = 1 + rn(K) / 8, 1 + rn(K) / 8
    cos, sin = rotary_tables(T, K // 2, device="cuda")
    gamma = torch.tensor([-0.1, -0.02], device="cuda")

    def gla(c, pos, h0, chunk):
        q, k, v = (t.unflatten(-1, (H, K)) for t in c.split(Dm, -1))
        q, k = qk_norm_rotary(q, k, qw, kw, cos, sin, pos)
        if chunk:
            return chunk_simple_gla(q, k, v, g_gamma=gamma, initial_state=h0, output_final_state=True)
        gk = gamma.view(1, 1, H, 1).expand_as(q).contiguous()
        return fused_recurrent_gla(q, k, v, gk=gk, initial_state=h0, output_final_state=True)

    A, skip, bias = -torch.rand(3 * Dm, N, generator=g, device="cuda") - 0.1, rn(3 * Dm), rn(3 * Dm) - 3
    dt, Bm, Cm, z = rn(B, T, 3 * Dm), rn(B, T, N), rn(B, T, N), rn(B, T, 3 * Dm)

    def ssm(c, sl, h0):
        return selective_scan(c, dt[:, sl], A, Bm[:, sl], Cm[:, sl], skip, z[:, sl], bias, True, h0, True)

    whole, _ = causal_conv1d(x, w, b, "silu")
    want, _ = gla(whole, None, None, True)
    want2, _ = ssm(whole, slice(None), None)
    cut = 61
    c, cs = causal_conv1d(x[:, :cut], w, b, "silu", None, True)
    o, hs = gla(c, torch.arange(cut, device="cuda"), None, True)
    o2, ss = ssm(c, slice(0, cut), None)
    rel = lambda a, r: ((a - r).norm() / r.norm()).item()  # noqa: E731
    assert rel(o, want[:, :cut]) < 1e-5 and rel(o2, want2[:, :cut]) < 1e-5
    for t in range(cut, T):
        c, cs = causal_conv1d_step(x[:, t], cs, w, b, "silu", state_out=cs)
        o, hs = gla(c[:, None], torch.full((B, 1), t, device="cuda"), hs, False)
        assert rel(o[:, 0], want[:, t]) < 1e-5
        y, ss = selective_scan_step(c, dt[:, t], A, Bm[:, t], Cm[:, t], ss, skip, z[:, t], bias, True, state_out=ss)
        assert rel(y, want2[:, t]) < 1e-5
    # packed: the two rows as sequences of one axis, gradients of the whole run
    leaf = x.reshape(1, B * T, -1).clone().requires_grad_()
    cu = torch.tensor([0, T, 2 * T], dtype=torch.int32, device="cuda")
    c, _ = causal_conv1d(leaf, w, b, "silu", cu_seqlens=cu)
    y, _ = selective_scan(c, dt.reshape(1, B * T, -1), A, Bm.reshape(1, B * T, N), Cm.reshape(1, B * T, N), skip,
                          z.reshape(1, B * T, -1), bias, True, cu_seqlens=cu)
    assert rel(y.view_as(want2), want2) < 1e-5
    (dx,) = torch.autograd.grad(y.sum(), leaf)
    leaf2 = x.clone().requires_grad_()
    c, _ = causal_conv1d(leaf2, w, b, "silu")
    y2, _ = ssm(c, slice(None), None)
    (dx2,) = torch.autograd.grad(y2.sum(), leaf2)
    assert rel(dx.view_as(dx2), dx2) < 1e-5
