"""Argument handling shared by the operators that take strided rows and packed sequences
(``causal_conv1d``, ``selective_scan``, ``qk_norm_rotary`` and their single-token forms)."""
from __future__ import annotations

import torch
from torch._C import (_get_dispatch_mode, _has_storage, _increment_version, _is_tracing, _len_torch_dispatch_stack,
                      _TorchDispatchModeKey)
from torch._C._functorch import peek_interpreter_stack
from torch.autograd import forward_ad

from . import _C


def watched() -> bool:
    """Whether a trace, a transform, a dispatch mode or a forward-mode level is there to look at a call at all (the quick
    form of the checks below, 0.2 us)."""
    return (forward_ad._current_level >= 0 or _len_torch_dispatch_stack() != 0 or peek_interpreter_stack() is not None
            or _is_tracing())


def has_tangent(*tensors) -> bool:
    """Whether forward-mode differentiation goes through one of the tensors."""
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def plain(*tensors) -> bool:
    """Whether the call is eager and on tensors of its own memory.  A kernel reads and writes through addresses:
    ``torch.jit.trace``, ``torch.func``, forward mode, dispatch modes (``make_fx``, fake tensors, FLOP counts) and
    tensor subclasses see none of it, so a module whose torch form they followed goes that way there."""
    if watched() and (_is_tracing() or _len_torch_dispatch_stack() or peek_interpreter_stack() is not None
                      or has_tangent(*tensors)):
        return False
    return all(t is None or type(t) is torch.Tensor or type(t) is torch.nn.Parameter for t in tensors)


def eager_only(op: str, *tensors) -> None:
    """Refuses what a kernel's launch would silently fall out of: a recording would hold an empty output, a tangent
    would be dropped, a batch dimension or a fake tensor has no memory of its own."""
    if _is_tracing() or (_len_torch_dispatch_stack() and _get_dispatch_mode(_TorchDispatchModeKey.PROXY) is not None):
        raise RuntimeError(f"{op} cannot be traced (its kernel writes through addresses, which a trace does not record)")
    if peek_interpreter_stack() is not None:
        raise RuntimeError(f"{op} cannot be transformed by torch.func (vmap, grad, jvp)")
    if _len_torch_dispatch_stack() and _get_dispatch_mode(_TorchDispatchModeKey.FAKE) is not None:
        raise RuntimeError(f"{op} cannot run on fake tensors: there is no memory behind them")
    if has_tangent(*tensors):
        raise RuntimeError(f"{op} has no forward-mode derivative: a tensor carries a tangent")


def plain_grads(*grads) -> bool:
    """``plain`` for the gradients that a backward is given (it may run on another thread than a transform)."""
    return plain(*grads) and all(g is None or _has_storage(g) for g in grads)


def eager_grads(op: str, *grads) -> None:
    """``eager_only`` for the gradients that a backward is given."""
    if watched():
        eager_only(op, *grads)
    for g in grads:
        if g is not None and not _has_storage(g):
            raise RuntimeError(f"{op} has no gradient for a batch of them (is_grads_batched, torch.func)")


# The kernels count rows and channels in 32 bits (offsets in 64); a tile may step past the last row.
MAX_ROWS, MAX_CHANNELS = 2 ** 31 - 2 ** 16, 2 ** 28


def check_sizes(op: str, batch: int, rows: int, channels: int) -> None:
    """Called where a tensor has more elements than the smaller limit."""
    if batch > MAX_ROWS or rows > MAX_ROWS or channels > MAX_CHANNELS:
        raise ValueError(f"{op}: at most {MAX_ROWS} batch entries and rows and {MAX_CHANNELS} channels or heads, "
                         f"got {batch}, {rows} and {channels}")


def check_cuda(op: str, first: torch.Tensor, **others) -> None:
    """``first`` and every other given tensor lie on one CUDA device."""
    if not first.is_cuda:
        raise RuntimeError(f"{op} needs CUDA tensors (the kernels are the only implementation)")
    if first.dtype not in _C._DTYPE:
        raise TypeError(f"{op}: unsupported dtype {first.dtype} (float32, bfloat16 or float16)")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{op}: {name} is on {t.device}, expected {first.device}")


def check_like(op: str, name: str, t: torch.Tensor | None, shape: tuple, dtype: torch.dtype) -> None:
    if t is None:
        return
    assert tuple(t.shape) == tuple(shape), f"{op}: expected {name} shape {tuple(shape)}, got {tuple(t.shape)}"
    if t.dtype != dtype:
        raise TypeError(f"{op}: {name} must be {dtype}, got {t.dtype}")


def no_grad_only(op: str, other: str, *tensors) -> None:
    if wants_grad(*tensors):
        raise RuntimeError(f"{op} has no gradient: call {other}, or this under torch.no_grad()")


def wants_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def like(t: torch.Tensor | None, shape, dtype: torch.dtype, device: int) -> bool:
    """Whether ``t`` is absent or has that shape, dtype and device (the quick form of the checks below)."""
    return t is None or (t.shape == shape and t.dtype == dtype and t.get_device() == device)


def rows(t: torch.Tensor | None) -> torch.Tensor | None:
    """``t`` itself where its last dim is dense, else a contiguous copy."""
    return t if t is None or t.stride(-1) == 1 or t.is_contiguous() else t.contiguous()


def rows2(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself where its last two dims are dense, else a contiguous copy."""
    if t.stride(-1) == 1 and (t.shape[-2] == 1 or t.stride(-2) == t.shape[-1]):
        return t
    return t.contiguous()


def sequences(op: str, cu_seqlens, B: int, T: int, device) -> tuple[int, torch.Tensor | None]:
    """(number of sequences, device int32 offsets or None).

    Host offsets (list or CPU tensor) are checked and copied to the device.  Offsets that lie on the
    device are used as they are, without a read on the host: such a call can be captured into a CUDA
    graph and replayed with other offsets.  The kernels clamp them to [0, T]; rows behind the last
    sequence give zeros."""
    if cu_seqlens is None:
        return B, None
    assert B == 1, f"{op}: batch size must be 1 when using cu_seqlens, got {B}"
    if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.is_cuda:
        assert cu_seqlens.dim() == 1 and cu_seqlens.numel() >= 2, f"{op}: cu_seqlens must be [N + 1] with N >= 1"
        if cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{op}: cu_seqlens must be int32 or int64, got {cu_seqlens.dtype}")
        if cu_seqlens.device != device:
            raise RuntimeError(f"{op}: cu_seqlens is on {cu_seqlens.device}, expected {device}")
        return cu_seqlens.numel() - 1, cu_seqlens.to(torch.int32).contiguous()
    cu = [int(c) for c in (cu_seqlens.tolist() if isinstance(cu_seqlens, torch.Tensor) else cu_seqlens)]
    assert len(cu) >= 2 and cu[0] == 0 and cu[-1] == T, f"{op}: cu_seqlens must run from 0 to T={T}, got {cu}"
    assert all(b >= a for a, b in zip(cu, cu[1:])), f"{op}: cu_seqlens must be non-decreasing"
    return len(cu) - 1, torch.tensor(cu, dtype=torch.int32, device=device)


def state_target(op: str, state: torch.Tensor, out: torch.Tensor | None, *reads) -> tuple:
    """(state to read, tensor to write): ``out`` may be ``state`` itself; any other overlap with
    what the call reads is refused.  ``out`` counts as changed in place, so that a backward which still
    needs what it held says so."""
    if out is None:
        state = state.contiguous()
        return state, torch.empty_like(state)
    check_like(op, "state_out", out, state.shape, state.dtype)
    if out.device != state.device:
        raise RuntimeError(f"{op}: state_out is on {out.device}, expected {state.device}")
    assert out.is_contiguous(), f"{op}: state_out must be contiguous"
    if out.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{op}: state_out requires a gradient, which the step does not have")
    a, n = out.data_ptr(), out.numel() * out.element_size()
    same = state.data_ptr() == a and state.is_contiguous()
    for t in reads if same else (state, *reads):
        if t is not None and t.numel() and n:
            last = sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
            if t.data_ptr() < a + n and a < t.data_ptr() + (last + 1) * t.element_size():
                raise ValueError(f"{op}: state_out overlaps a tensor that the call reads")
    state = state if same else state.contiguous()
    _increment_version((out,))
    return state, out


def launch(name: str, args, t: torch.Tensor) -> None:
    """One C call on the current stream of ``t``'s device, whatever the current device is."""
    if t.get_device() == torch._C._cuda_getDevice():  # t is a CUDA tensor: the runtime is up
        _C.call(name, args, _C.stream_of(t))
    else:
        with torch.cuda.device(t.device):
            _C.call(name, args, _C.stream_of(t))


def workspace(nbytes: int, t: torch.Tensor) -> torch.Tensor | None:
    return torch.empty(int(nbytes), dtype=torch.uint8, device=t.device) if nbytes else None
