"""Causal depthwise short convolution (reference tops/modules/convolution.py:6).

``causal_conv1d`` (prompts and training) and ``causal_conv1d_step`` (one token a row) run in
``conv.cu`` (``tops_gla_causal_conv_*``), fp32 arithmetic on fp32, bf16 or fp16 tensors.
``ShortConvolution`` calls them for CUDA tensors.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import _C
from .. import _rows

__all__ = ["ShortConvolution", "causal_conv1d", "causal_conv1d_step"]

_ACT = {None: 0, "silu": 1, "swish": 1}
KERNEL_WIDTHS = (2, 3, 4)


def _args(x, w, bias, state, y, final, act, N, cu):
    B, T, D = x.shape
    return _C.ConvArgs(B, T, D, w.shape[1], N, _C.dtype_code(x.dtype), _C.dtype_code(w.dtype), act, _C.ptr(cu),
                       x.data_ptr(), x.stride(0), x.stride(1), w.data_ptr(), _C.ptr(bias), _C.ptr(state), _C.ptr(y),
                       _C.ptr(final))


def _forward(x, w, bias, state, act, want_final, N, cu):
    x = _rows.rows(x)
    w, bias, state = (t if t is None else t.contiguous() for t in (w, bias, state))
    y = x.new_empty(x.shape)
    final = x.new_empty((N, x.shape[2], w.shape[1] - 1)) if want_final else None
    _rows.launch("tops_gla_causal_conv_fwd", _args(x, w, bias, state, y, final, act, N, cu), x)
    return y, final


def _backward(x, w, bias, state, dy, dfinal, act, N, cu, need):
    """Gradients of x, w, bias and state from the kernel (None where not needed)."""
    x = _rows.rows(x)
    w, bias, state = (t if t is None else t.contiguous() for t in (w, bias, state))
    dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else _rows.rows(dy.to(x.dtype))
    dfinal = None if dfinal is None else dfinal.to(x.dtype).contiguous()
    dx = x.new_empty(x.shape)
    dw = torch.empty_like(w) if need[1] else None
    db = torch.empty_like(bias) if bias is not None and need[2] else None
    ds = torch.empty_like(state) if state is not None and need[3] else None
    a = _C.ConvBwdArgs(_args(x, w, bias, state, None, None, act, N, cu), dy.data_ptr(), dy.stride(0), dy.stride(1),
                       _C.ptr(dfinal), dx.data_ptr(), _C.ptr(dw), _C.ptr(db), _C.ptr(ds), None, 0)
    ws = _rows.workspace(_C.lib().tops_gla_causal_conv_bwd_workspace_size(a), x)
    a.workspace, a.workspace_bytes = _C.ptr(ws), 0 if ws is None else ws.numel()
    _rows.launch("tops_gla_causal_conv_bwd", a, x)
    return dx if need[0] else None, dw, db, ds


def _gradient_form(x, w, bias, state, dy, dfinal, act, need):
    """The same in elementary torch operations in 32 bits: what the gradients' own derivatives are taken through."""
    B, T, D = x.shape
    W = w.shape[1]
    prev = x.new_zeros(B, W - 1, D) if state is None else state.transpose(1, 2)
    rows, wf = torch.cat([prev, x], 1).float(), w.float()
    d = x.new_zeros(B, T, D, dtype=torch.float32) if dy is None else dy.float()
    if act:
        p = sum(rows[:, j:j + T] * wf[:, j] for j in range(W)) + (0.0 if bias is None else bias.float())
        s = torch.sigmoid(p)
        d = d * s * (1 + p * (1 - s))
    drows = dw = db = None
    if need[0] or need[3]:
        drows = sum(F.pad(d * wf[:, j], (0, 0, j, W - 1 - j)) for j in range(W))
        if dfinal is not None:
            drows = drows + F.pad(dfinal.float().transpose(1, 2), (0, 0, T, 0))
    if need[1]:
        dw = torch.stack([(d * rows[:, j:j + T]).sum((0, 1)) for j in range(W)], -1).to(w.dtype)
    if bias is not None and need[2]:
        db = d.sum((0, 1)).to(bias.dtype)
    return (drows[:, W - 1:].to(x.dtype) if need[0] else None, dw, db,
            drows[:, :W - 1].transpose(1, 2).to(x.dtype) if state is not None and need[3] else None)


class _CausalConvGradient(torch.autograd.Function):
    """The backward as an operation of its own (create_graph): the kernel's gradients, differentiated by their formula."""

    @staticmethod
    def forward(ctx, x, w, bias, state, dy, dfinal, act, N, cu, need):
        ctx.save_for_backward(x, w, bias, state, dy, dfinal)
        ctx.act, ctx.packed, ctx.need = act, cu is not None, need
        ctx.set_materialize_grads(False)
        return _backward(x, w, bias, state, dy, dfinal, act, N, cu, need)

    @staticmethod
    def backward(ctx, *grads):
        if ctx.packed:
            raise RuntimeError("causal_conv1d: packed sequences have no second derivative")
        again = torch.is_grad_enabled()
        with torch.enable_grad():
            # a view each: one tensor given in two places is two variables here
            given = [None if t is None else t.view_as(t) for t in ctx.saved_tensors]
            first = _gradient_form(*given, ctx.act, ctx.need)
            pairs = [(f, g) for f, g in zip(first, grads) if g is not None and f.requires_grad]
            wanted = [t for t, n in zip(given, ctx.needs_input_grad) if n]
            if pairs and wanted:
                got = iter(torch.autograd.grad([f for f, _ in pairs], wanted, [g for _, g in pairs], create_graph=again,
                                               allow_unused=True))
            else:
                got = iter([None] * len(wanted))
        return tuple(next(got) if n else None for n in ctx.needs_input_grad[:6]) + (None,) * 4


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, state, act, want_final, N, cu):
        ctx.save_for_backward(x, w, bias, state, cu)
        ctx.act, ctx.N = act, N
        ctx.set_materialize_grads(False)
        y, final = _forward(x, w, bias, state, act, want_final, N, cu)
        return (y, final) if want_final else y

    @staticmethod
    def backward(ctx, dy, dfinal=None):
        *inputs, cu = ctx.saved_tensors
        need = ctx.needs_input_grad[:4]
        if dy is None and dfinal is None:
            return (None,) * 8
        if not _rows.plain_grads(dy, dfinal):  # a batch of gradients, a tangent, a mode: the formula carries them
            if cu is None:
                return *_gradient_form(*inputs, dy, dfinal, ctx.act, need), None, None, None, None
            _rows.eager_grads("causal_conv1d of packed sequences", dy, dfinal)
        a = (*inputs, dy, dfinal, ctx.act, ctx.N, cu, need)
        got = _CausalConvGradient.apply(*a) if torch.is_grad_enabled() else _backward(*a)
        return *got, None, None, None, None


def _check(op, x, weight, bias, activation, D, state, state_shape):
    if activation not in _ACT:
        raise ValueError(f"{op}: activation must be None, 'silu' or 'swish', got {activation!r}")
    W, dev, wd = weight.shape[1], x.get_device(), weight.dtype
    if (dev >= 0 and x.dtype in _C._DTYPE and W in KERNEL_WIDTHS and weight.shape[0] == D and weight.get_device() == dev
            and (wd == x.dtype or wd == torch.float32) and (bias is None or _rows.like(bias, (D,), wd, dev))
            and (state is None or _rows.like(state, (*state_shape, D, W - 1), x.dtype, dev))):
        return
    _rows.check_cuda(op, x, weight=weight, bias=bias, state=state)
    if W not in KERNEL_WIDTHS:
        raise ValueError(f"{op}: the kernel width must be one of {KERNEL_WIDTHS}, got {W}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{op}: weight must be {x.dtype} or float32, got {weight.dtype}")
    assert weight.shape[0] == D, f"{op}: expected weight shape {(D, W)}, got {tuple(weight.shape)}"
    _rows.check_like(op, "bias", bias, (D,), weight.dtype)
    _rows.check_like(op, "state", state, state_shape + (D, W - 1), x.dtype)


def _weight2d(op, weight):
    if weight.dim() == 3 and weight.shape[1] == 1:
        weight = weight.squeeze(1)
    assert weight.dim() == 2, f"{op}: expected weight [D, W] or [D, 1, W], got {tuple(weight.shape)}"
    return weight


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                  activation: str | None = None, initial_state: torch.Tensor | None = None,
                  output_final_state: bool = False, cu_seqlens=None):
    """Causal depthwise convolution over time -> ``(y, final_state or None)``.

    Args:
        x: [B, T, D] fp32, bf16 or fp16; rows may be strided (a slice of a wider projection)
        weight: [D, W] or [D, 1, W], W in 2..4; bias: [D] (both in x's dtype or both fp32)
        activation: None, "silu" or "swish"
        initial_state: [N, D, W - 1], the inputs before each sequence (last column = newest)
        output_final_state: return [N, D, W - 1] of the same kind, the state after each sequence
        cu_seqlens: [N + 1] offsets of N sequences packed along T (B must be 1).  Offsets on the GPU are
            not read by the host (capturable); rows behind the last sequence give zeros.
    Gradients flow to x, weight, bias and initial_state, also from the final state; where sequences
    are not packed they can be differentiated again (the first gradients stay the kernel's, the rest is taken in
    fp32 torch operations).  Eager calls only: tracing, ``torch.func`` and forward mode
    are refused (``ShortConvolution`` goes through torch's conv1d there).
    """
    op = "causal_conv1d"
    if _rows.watched():
        _rows.eager_only(op, x, weight, bias, initial_state)
    assert x.dim() == 3, f"{op}: expected x [B, T, D], got {tuple(x.shape)}"
    if x.numel() > _rows.MAX_CHANNELS:
        _rows.check_sizes(op, *x.shape)
    weight = _weight2d(op, weight)
    N, cu = _rows.sequences(op, cu_seqlens, x.shape[0], x.shape[1], x.device)
    _check(op, x, weight, bias, activation, x.shape[2], initial_state, (N,))
    a = (x, weight, bias, initial_state, _ACT[activation], bool(output_final_state), N, cu)
    if not _rows.wants_grad(x, weight, bias, initial_state):
        return _forward(*a)
    out = _CausalConv.apply(*a)
    return out if output_final_state else (out, None)


def causal_conv1d_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                       activation: str | None = None, state_out: torch.Tensor | None = None):
    """One token of each row -> ``(y [B, D], new state [B, D, W - 1])``.

    x [B, D]; ``state`` as ``causal_conv1d`` returns it.  The new state goes to ``state_out`` where
    given, which may be ``state`` itself (updated in place).  No gradient.
    """
    op = "causal_conv1d_step"
    if _rows.watched():
        _rows.eager_only(op, x, state, weight, bias)
    assert x.dim() == 2, f"{op}: expected x [B, D], got {tuple(x.shape)}"
    weight = _weight2d(op, weight)
    B, D = x.shape
    if x.numel() > _rows.MAX_CHANNELS:
        _rows.check_sizes(op, B, 1, D)
    _check(op, x, weight, bias, activation, D, state, (B,))
    _rows.no_grad_only(op, "causal_conv1d", x, state, weight, bias)
    x = _rows.rows(x)
    weight, bias = weight.contiguous(), None if bias is None else bias.contiguous()
    state, out = _rows.state_target(op, state, state_out, x, weight, bias)
    y = x.new_empty((B, D))
    a = _C.ConvArgs(B, 1, D, weight.shape[1], B, _C.dtype_code(x.dtype), _C.dtype_code(weight.dtype), _ACT[activation],
                    None, x.data_ptr(), x.stride(0), 0, weight.data_ptr(), _C.ptr(bias), state.data_ptr(), y.data_ptr(),
                    out.data_ptr())
    _rows.launch("tops_gla_causal_conv_step", a, x)
    return y, out


class ShortConvolution(nn.Module):
    """Causal depthwise conv1d over time with an optional activation (reference
    tops/modules/convolution.py; torch gold tests/src/modules/convolution.py); the decode cache holds the
    last ``kernel_size - 1`` inputs of each sequence.  CUDA tensors of a kernel's dtype and width
    (``kernel_size`` 2 to 4) run on ``causal_conv1d``, packed sequences (``cu_seqlens``) there only;
    the rest (CPU tensors, other widths, an autocast dtype other than x's; without packing also tracing and
    compiling, ``torch.func``, forward mode, dispatch modes, tensor subclasses) is torch's conv1d."""

    def __init__(self, hidden_size: int, kernel_size: int = 4, bias: bool = False, activation: str | None = "silu"):
        super().__init__()
        self.hidden_size, self.kernel_size = hidden_size, kernel_size
        self.weight = nn.Parameter(torch.empty(hidden_size, 1, kernel_size))
        self.bias = nn.Parameter(torch.zeros(hidden_size)) if bias else None
        nn.init.kaiming_uniform_(self.weight, a=5 ** 0.5)
        self.activation = activation

    def _on_kernel(self, x, cache, packed):
        if not x.is_cuda or x.dtype not in _C._DTYPE or self.kernel_size not in KERNEL_WIDTHS:
            return False
        # packed rows have no other form: causal_conv1d says what it cannot follow
        if not packed and (torch.compiler.is_compiling() or not _rows.plain(x, self.weight, self.bias, cache)):
            return False
        return not torch.is_autocast_enabled("cuda") or x.dtype == torch.get_autocast_dtype("cuda")

    def forward(self, x, cache=None, output_final_state=False, cu_seqlens=None):
        if self._on_kernel(x, cache, cu_seqlens is not None):
            act = self.activation if self.activation in ("silu", "swish") else None
            bias = None if self.bias is None else self.bias.to(x.dtype)
            y, state = causal_conv1d(x, self.weight.to(x.dtype), bias, act, None if cache is None else cache.to(x.dtype),
                                     output_final_state, cu_seqlens)
            return y, None if state is None else state.detach()
        if cu_seqlens is not None:
            raise NotImplementedError("ShortConvolution: packed (cu_seqlens) inputs need the kernel: a CUDA tensor in "
                                      "float32, bfloat16 or float16 and a kernel_size of 2 to 4")
        B, T, D = x.shape
        xt = x.transpose(1, 2)  # [B, D, T]
        prev = cache if cache is not None else x.new_zeros(B, D, self.kernel_size - 1)
        xin = torch.cat([prev.to(x.dtype), xt], -1)
        y = F.conv1d(xin, self.weight.to(x.dtype), None if self.bias is None else self.bias.to(x.dtype),
                     groups=D)
        if self.activation in ("silu", "swish"):
            y = F.silu(y)
        new_cache = xin[..., -(self.kernel_size - 1):].detach() if output_final_state else None
        return y.transpose(1, 2), new_cache
