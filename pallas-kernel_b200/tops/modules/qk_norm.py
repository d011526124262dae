"""RMS norm of every query and key head with the position rotation in the same pass, for the
recurrences' q and k (between the projections or short convolutions and ``chunk_gla`` /
``chunk_simple_gla``).  Forward and backward run in ``qk_norm.cu`` (``tops_gla_qk_norm_rotary_*``),
fp32 arithmetic on fp32, bf16 or fp16 tensors.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _C
from .. import _rows

__all__ = ["qk_norm_rotary", "rotary_tables"]

MAX_HEAD = 256


def rotary_tables(max_positions: int, rotary_dim: int, base: float = 10000.0, device=None):
    """``(cos, sin)`` [max_positions, rotary_dim / 2] fp32 of the angles pos * base^(-2 i / rotary_dim).
    The angles are taken in 64 bits: in 32 a far position loses its fraction of a turn."""
    assert rotary_dim > 0 and rotary_dim % 2 == 0, f"rotary_dim must be even and positive, got {rotary_dim}"
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    pos = torch.arange(max_positions, dtype=torch.float64, device=device)
    angle = pos[:, None] * (base ** (-i / rotary_dim))
    return angle.cos().float(), angle.sin().float()


_S3 = _C.C.c_int64 * 3


def _strides(t):
    return _S3(*t.stride()[:3])


def _args(q, k, qw, kw, cos, sin, positions, eps, interleaved):
    B, T, H, K = q.shape
    w = qw if qw is not None else kw
    return _C.QKNormArgs(B, T, H, k.shape[2], K, 0 if cos is None else 2 * cos.shape[1], _C.dtype_code(q.dtype),
                         _C.dtype_code(q.dtype if w is None else w.dtype), int(interleaved),
                         int(positions is not None and positions.dtype == torch.int64),
                         0 if cos is None else cos.shape[0], eps, q.data_ptr(), k.data_ptr(), _strides(q), _strides(k),
                         _C.ptr(qw), _C.ptr(kw), _C.ptr(cos), _C.ptr(sin), _C.ptr(positions),
                         positions.stride(0) if positions is not None and positions.dim() == 2 else 0, None, None)


def _forward(q, k, qw, kw, cos, sin, positions, eps, interleaved):
    q, k = _rows.rows(q), _rows.rows(k)
    qw, kw = (None if w is None else w.contiguous() for w in (qw, kw))
    qo, ko = q.new_empty(q.shape), k.new_empty(k.shape)
    a = _args(q, k, qw, kw, cos, sin, positions, eps, interleaved)
    a.q_out, a.k_out = qo.data_ptr(), ko.data_ptr()
    _rows.launch("tops_gla_qk_norm_rotary_fwd", a, q)
    return qo, ko


class _QKNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, cos, sin, positions, eps, interleaved):
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        return _forward(q, k, qw, kw, cos, sin, positions, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dqo, dko):
        _rows.eager_grads("qk_norm_rotary", dqo, dko)
        q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
        q, k = _rows.rows(q), _rows.rows(k)
        qw, kw = (None if w is None else w.contiguous() for w in (qw, kw))
        dqo, dko = _rows.rows(dqo.to(q.dtype)), _rows.rows(dko.to(q.dtype))
        dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
        dqw, dkw = (torch.empty_like(w) if w is not None and need else None
                    for w, need in zip((qw, kw), ctx.needs_input_grad[2:4]))
        f = _args(q, k, qw, kw, cos, sin, positions, ctx.eps, ctx.interleaved)
        a = _C.QKNormBwdArgs(f, dqo.data_ptr(), dko.data_ptr(), _strides(dqo), _strides(dko), dq.data_ptr(),
                             dk.data_ptr(), _C.ptr(dqw), _C.ptr(dkw), None, 0)
        ws = _rows.workspace(_C.lib().tops_gla_qk_norm_rotary_bwd_workspace_size(a), q)
        a.workspace, a.workspace_bytes = _C.ptr(ws), 0 if ws is None else ws.numel()
        _rows.launch("tops_gla_qk_norm_rotary_bwd", a, q)
        return dq, dk, dqw, dkw, None, None, None, None, None


def _check(op, q, k, q_weight, k_weight, cos, sin, positions):
    """-> the weights in one dtype, the tables and positions as the kernel takes them."""
    B, T, _, K = q.shape
    dev, dt = q.get_device(), q.dtype
    wd = dt if q_weight is None else q_weight.dtype
    if not (dev >= 0 and dt in _C._DTYPE and _rows.like(k, (B, T, k.shape[2], K), dt, dev) and (wd == dt or wd == torch.float32)
            and _rows.like(q_weight, (K,), wd, dev) and _rows.like(k_weight, (K,), wd, dev)):
        _rows.check_cuda(op, q, k=k, q_weight=q_weight, k_weight=k_weight)
        _rows.check_like(op, "k", k, (B, T, k.shape[2], K), dt)
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is not None:
                assert tuple(w.shape) == (K,), f"{op}: expected {name} shape {(K,)}, got {tuple(w.shape)}"
                if w.dtype not in (dt, torch.float32):
                    raise TypeError(f"{op}: {name} must be {dt} or float32, got {w.dtype}")
        if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
            q_weight, k_weight = q_weight.float(), k_weight.float()
    assert (cos is None) == (sin is None), f"{op}: cos and sin come together"
    if cos is None:
        return q_weight, k_weight, None, None, None
    if cos.shape[0] > _rows.MAX_ROWS:
        raise ValueError(f"{op}: at most {_rows.MAX_ROWS} positions in the tables, got {cos.shape[0]}")
    if cos.get_device() != dev or sin.get_device() != dev or (positions is not None and positions.get_device() != dev):
        _rows.check_cuda(op, q, cos=cos, sin=sin, positions=positions)
    R = 2 * cos.shape[-1]
    assert cos.dim() == 2 and cos.shape[0] > 0 and 0 < R <= K, \
        f"{op}: expected cos [P, R / 2] with R in 2..{K}, got {tuple(cos.shape)}"
    for name, t in (("cos", cos), ("sin", sin)):
        if t.shape != cos.shape or t.dtype != torch.float32:
            _rows.check_like(op, name, t, cos.shape, torch.float32)
        if t.requires_grad:
            raise RuntimeError(f"{op}: {name} has no gradient")
    if positions is None:
        assert T <= cos.shape[0], f"{op}: {T} rows, but the tables have {cos.shape[0]}"
    else:
        assert positions.shape == (B, T) or positions.shape == (T,), \
            f"{op}: expected positions [T] or [B, T], got {tuple(positions.shape)}"
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{op}: positions must be int32 or int64, got {positions.dtype}")
        positions = _rows.rows(positions)
    return q_weight, k_weight, cos.contiguous(), sin.contiguous(), positions


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                   sin: torch.Tensor | None = None, positions: torch.Tensor | None = None, eps: float = 1e-6,
                   interleaved: bool = False):
    """RMS norm of each head of q and k, then the rotation of its first R elements by the row's position
    -> ``(q, k)`` of the same shapes.

    Args:
        q: [B, T, H, K], k: [B, T, HK, K] fp32, bf16 or fp16, K up to 256; may be slices of a wider
            projection (dense heads)
        q_weight, k_weight: [K] or None, in q's dtype or fp32
        cos, sin: [P, R / 2] fp32 of positions 0..P-1 (``rotary_tables``), or None for the norm alone
        positions: [T] or [B, T] int32 or int64; default 0..T-1.  A position outside 0..P-1 gives NaN in
            the rotated elements (the host does not read the positions).
        interleaved: the pairs are (2i, 2i + 1) instead of (i, i + R / 2)
    Gradients flow to q, k and the weights.  Eager calls only: tracing, ``torch.func`` and forward mode are refused.
    """
    op = "qk_norm_rotary"
    if _rows.watched():
        _rows.eager_only(op, q, k, q_weight, k_weight, cos, sin)
    assert q.dim() == 4 and k.dim() == 4, f"{op}: expected q [B, T, H, K] and k [B, T, HK, K]"
    B, T, H, K = q.shape
    if q.numel() > _rows.MAX_CHANNELS or k.numel() > _rows.MAX_CHANNELS:
        _rows.check_sizes(op, B, T, max(H, k.shape[2]))
    if not 1 <= K <= MAX_HEAD:
        raise ValueError(f"{op}: heads must have 1 to {MAX_HEAD} elements, got {K}")
    q_weight, k_weight, cos, sin, positions = _check(op, q, k, q_weight, k_weight, cos, sin, positions)
    a = (q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved))
    return _QKNormRotary.apply(*a) if _rows.wants_grad(q, k, q_weight, k_weight) else _forward(*a)
