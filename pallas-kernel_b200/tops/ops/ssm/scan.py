"""Selective state space scan.  Per channel d of a group and state n,

    delta = softplus(dt + dt_bias)  (or dt + dt_bias)
    h_t = exp(delta_t A[d, n]) h_{t-1} + delta_t x_t B_t[n]
    y_t = sum_n C_t[n] h_t + D x_t,    out = y silu(z)

The forward and the single-token step run in ``ssm_scan.cu``, the backward in ``ssm_scan_bwd.cu``
(``tops_gla_ssm_scan_*``): fp32 arithmetic and states on fp32, bf16 or fp16 tensors.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ... import _C
from ... import _rows

__all__ = ["selective_scan", "selective_scan_step"]

MAX_STATES = 64


def _f32(t):
    return t if t is None or t.dtype == torch.float32 else t.float()


def _args(x, dt, A, Bm, Cm, D, z, bias, h0, softplus, S, cu):
    B, T, ch = x.shape
    G, N = Bm.shape[2:]
    zb, zt = (0, 0) if z is None else z.stride()[:2]
    return _C.ScanArgs(B, T, ch, N, G, S, _C.dtype_code(x.dtype), softplus, _C.ptr(cu), x.data_ptr(), dt.data_ptr(),
                       _C.ptr(z), Bm.data_ptr(), Cm.data_ptr(), *x.stride()[:2], *dt.stride()[:2], zb, zt,
                       *Bm.stride()[:2], *Cm.stride()[:2], A.data_ptr(), _C.ptr(D), _C.ptr(bias), _C.ptr(h0))


def _dense(x, dt, A, Bm, Cm, D, z, bias, h0):
    r, r2 = _rows.rows, _rows.rows2
    c = [None if t is None else t.contiguous() for t in (A, D, bias, h0)]
    return r(x), r(dt), c[0], r2(Bm), r2(Cm), c[1], r(z), c[2], c[3]


def _forward(x, dt, A, Bm, Cm, D, z, bias, h0, softplus, want_final, S, cu, save):
    x, dt, A, Bm, Cm, D, z, bias, h0 = _dense(x, dt, A, Bm, Cm, D, z, bias, h0)
    a = _args(x, dt, A, Bm, Cm, D, z, bias, h0, softplus, S, cu)
    L = _C.lib()
    y = x.new_empty(x.shape)
    ht = torch.empty(S, x.shape[2], Bm.shape[3], dtype=torch.float32, device=x.device) if want_final else None
    states = None
    if save:
        states = torch.empty(L.tops_gla_ssm_scan_states_size(a) // 4, dtype=torch.float32, device=x.device)
    a.y, a.ht, a.states = y.data_ptr(), _C.ptr(ht), _C.ptr(states)
    ws = _rows.workspace(L.tops_gla_ssm_scan_fwd_workspace_size(a), x)
    a.workspace, a.workspace_bytes = _C.ptr(ws), 0 if ws is None else ws.numel()
    _rows.launch("tops_gla_ssm_scan_fwd", a, x)
    return y, ht, states


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, Bm, Cm, D, z, bias, h0, softplus, want_final, S, cu):
        y, ht, states = _forward(x, dt, A, Bm, Cm, D, z, bias, h0, softplus, want_final, S, cu, True)
        ctx.save_for_backward(x, dt, A, Bm, Cm, D, z, bias, h0, cu, states)
        ctx.softplus, ctx.S = softplus, S
        ctx.set_materialize_grads(False)
        return (y, ht) if want_final else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dht=None):
        *inputs, cu, states = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dout is None and dht is None:
            return (None,) * 13
        _rows.eager_grads("selective_scan", dout, dht)
        x, dt, A, Bm, Cm, D, z, bias, h0 = _dense(*inputs)
        new = lambda like: like.new_empty(like.shape)  # noqa: E731
        dout = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dout is None else _rows.rows(dout.to(x.dtype))
        dht = None if dht is None else dht.float().contiguous()
        dx, ddt, dB, dC = new(x), new(dt), new(Bm), new(Cm)
        dz = None if z is None else new(z)
        dA = new(A) if need[2] else None
        dD = new(D) if D is not None and need[5] else None
        dbias = new(bias) if bias is not None and need[7] else None
        dh0 = new(h0) if h0 is not None and need[8] else None
        f = _args(x, dt, A, Bm, Cm, D, z, bias, h0, ctx.softplus, ctx.S, cu)
        f.states = states.data_ptr()
        a = _C.ScanBwdArgs(f, dout.data_ptr(), *dout.stride()[:2], _C.ptr(dht), dx.data_ptr(), ddt.data_ptr(), _C.ptr(dz),
                           dB.data_ptr(), dC.data_ptr(), _C.ptr(dA), _C.ptr(dD), _C.ptr(dbias), _C.ptr(dh0))
        ws = _rows.workspace(_C.lib().tops_gla_ssm_scan_bwd_workspace_size(a), x)
        a.workspace, a.workspace_bytes = _C.ptr(ws), 0 if ws is None else ws.numel()
        _rows.launch("tops_gla_ssm_scan_bwd", a, x)
        return dx, ddt, dA, dB, dC, dD, dz, dbias, dh0, None, None, None, None


def _check(op, lead, x, dt, A, Bm, Cm, D, z, dt_bias, state, S):
    """-> (Bm, Cm) as [*lead, G, N], with every shape and type checked (``lead`` = x's leading dims)."""
    shape, ch, n = x.shape, x.shape[-1], len(lead)
    if Bm.dim() == n + 1:
        Bm = Bm.unsqueeze(n)
    if Cm.dim() == n + 1:
        Cm = Cm.unsqueeze(n)
    if Bm.dim() == n + 2 and A.dim() == 2:  # quick: all in one expression, explained below where it fails
        N, G, dev, dtype = A.shape[1], Bm.shape[n], x.get_device(), x.dtype
        like, bc = _rows.like, (*lead, Bm.shape[n], A.shape[1])
        if (dev >= 0 and dtype in _C._DTYPE and 1 <= N <= MAX_STATES and G >= 1 and ch % G == 0 and like(dt, shape, dtype, dev)
                and like(z, shape, dtype, dev) and like(Bm, bc, dtype, dev) and like(Cm, bc, dtype, dev)
                and A.shape[0] == ch and A.get_device() == dev
                and (D is None or (D.shape == (ch,) and D.get_device() == dev))
                and (dt_bias is None or (dt_bias.shape == (ch,) and dt_bias.get_device() == dev))
                and (state is None or (state.shape == (S, ch, N) and state.get_device() == dev))):
            return Bm, Cm
    _rows.check_cuda(op, x, dt=dt, A=A, B=Bm, C=Cm, D=D, z=z, dt_bias=dt_bias, state=state)
    assert A.dim() == 2 and A.shape[0] == ch, f"{op}: expected A shape ({ch}, N), got {tuple(A.shape)}"
    N = A.shape[1]
    if not 1 <= N <= MAX_STATES:
        raise ValueError(f"{op}: a channel must have 1 to {MAX_STATES} states, got {N}")
    assert Bm.dim() == n + 2, f"{op}: expected B {tuple(lead) + (N,)} or with groups before N, got {tuple(Bm.shape)}"
    G = Bm.shape[n]
    assert G >= 1 and ch % G == 0, f"{op}: {ch} channels cannot be shared by {G} groups"
    for name, t, want in (("dt", dt, shape), ("z", z, shape), ("B", Bm, (*lead, G, N)), ("C", Cm, (*lead, G, N))):
        _rows.check_like(op, name, t, want, x.dtype)
    for name, t, want in (("A", A, (ch, N)), ("D", D, (ch,)), ("dt_bias", dt_bias, (ch,)), ("state", state, (S, ch, N))):
        assert t is None or tuple(t.shape) == want, f"{op}: expected {name} shape {want}, got {tuple(t.shape)}"
    return Bm, Cm


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: torch.Tensor | None = None, z: torch.Tensor | None = None, dt_bias: torch.Tensor | None = None,
                   dt_softplus: bool = False, initial_state: torch.Tensor | None = None,
                   output_final_state: bool = False, cu_seqlens=None):
    """Selective state space scan over time -> ``(out, final_state or None)``.

    Args:
        x, dt: [B, T, D] fp32, bf16 or fp16; z: [B, T, D] output gate (optional); dt, z, B and C in x's dtype
        A: [D, N], N up to 64; B, C: [B, T, N], or [B, T, G, N] shared by the D / G channels of a group
        D: [D] skip weight; dt_bias: [D]; dt_softplus: delta = softplus(dt + dt_bias)
        initial_state: [S, D, N]; output_final_state: return the final state [S, D, N], fp32
        cu_seqlens: [S + 1] offsets of S sequences packed along T (batch size 1).  Offsets on the GPU are
            not read by the host (capturable); rows behind the last sequence give zeros.
    x, dt, z, B and C may be slices of wider tensors (dense channels).  A, D, dt_bias and states are
    used in fp32.  Gradients flow to every tensor, also from the final state; for them the call keeps a state of
    every eighth row, N / 2 bytes a row and channel.  Eager calls only: tracing, ``torch.func`` and forward mode
    are refused.
    """
    op = "selective_scan"
    if _rows.watched():
        _rows.eager_only(op, x, dt, A, B, C, D, z, dt_bias, initial_state)
    assert x.dim() == 3, f"{op}: expected x [B, T, D], got {tuple(x.shape)}"
    if x.numel() > _rows.MAX_CHANNELS:
        _rows.check_sizes(op, *x.shape)
    S, cu = _rows.sequences(op, cu_seqlens, x.shape[0], x.shape[1], x.device)
    B, C = _check(op, x.shape[:2], x, dt, A, B, C, D, z, dt_bias, initial_state, S)
    A, D, dt_bias, h0 = _f32(A), _f32(D), _f32(dt_bias), _f32(initial_state)
    tensors = (x, dt, A, B, C, D, z, dt_bias, h0)
    if not _rows.wants_grad(*tensors):
        y, ht, _ = _forward(*tensors, int(dt_softplus), bool(output_final_state), S, cu, False)
        return y, ht
    out = _SelectiveScan.apply(*tensors, int(dt_softplus), bool(output_final_state), S, cu)
    return out if output_final_state else (out, None)


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        state: torch.Tensor, D: torch.Tensor | None = None, z: torch.Tensor | None = None,
                        dt_bias: torch.Tensor | None = None, dt_softplus: bool = False,
                        state_out: torch.Tensor | None = None):
    """One token of each row -> ``(out [B, D], new state [B, D, N])``.

    x, dt, z [B, D]; B, C [B, N] or [B, G, N]; state [B, D, N] fp32 as ``selective_scan`` returns it.
    The new state goes to ``state_out`` where given, which may be ``state`` itself (updated in
    place).  No gradient.
    """
    op = "selective_scan_step"
    if _rows.watched():
        _rows.eager_only(op, x, dt, A, B, C, state, D, z, dt_bias)
    assert x.dim() == 2, f"{op}: expected x [B, D], got {tuple(x.shape)}"
    Bsz, ch = x.shape
    if x.numel() > _rows.MAX_CHANNELS:
        _rows.check_sizes(op, Bsz, 1, ch)
    B, C = _check(op, x.shape[:1], x, dt, A, B, C, D, z, dt_bias, state, Bsz)
    if state.dtype != torch.float32:
        raise TypeError(f"{op}: state must be float32, got {state.dtype}")
    _rows.no_grad_only(op, "selective_scan", x, dt, A, B, C, state, D, z, dt_bias)
    r, r2 = _rows.rows, _rows.rows2
    x, dt, z, B, C = r(x), r(dt), r(z), r2(B), r2(C)
    A = _f32(A).contiguous()
    D, dt_bias = (None if t is None else _f32(t).contiguous() for t in (D, dt_bias))
    state, out = _rows.state_target(op, state, state_out, x, dt, A, B, C, D, z, dt_bias)
    y = x.new_empty(x.shape)
    G, N = B.shape[1:]
    a = _C.ScanArgs(Bsz, 1, ch, N, G, Bsz, _C.dtype_code(x.dtype), int(dt_softplus), None, x.data_ptr(), dt.data_ptr(),
                    _C.ptr(z), B.data_ptr(), C.data_ptr(), x.stride(0), 0, dt.stride(0), 0, 0 if z is None else z.stride(0),
                    0, B.stride(0), 0, C.stride(0), 0, A.data_ptr(), _C.ptr(D), _C.ptr(dt_bias), state.data_ptr(),
                    y.data_ptr(), out.data_ptr())
    _rows.launch("tops_gla_ssm_scan_step", a, x)
    return y, out
