"""causal_conv1d, causal_conv1d_step and ShortConvolution on the GPU against the formulas in 64 bits."""
from __future__ import annotations

import pytest
import torch

from _rows_ref import close, conv_ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# roundings of one output: W products and sums, the bias, and the sigmoid's exponential and quotient
# (__expf: 2 + |p| / 8 steps, quotient 2), taken twice in the derivative
ONE, GRAD = 24, 48


def _mk(seed, B, T, D, W, dt, N, bias, state, wdt=None):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    wdt = wdt or dt
    x, dy = rn(B, T, D).to(dt), rn(B, T, D).to(dt)
    w, b = (rn(D, W) / 2).to(wdt), (rn(D) / 4).to(wdt) if bias else None
    st, df = (rn(N, D, W - 1).to(dt) if state else None), rn(N, D, W - 1).to(dt)
    return x, w, b, st, dy, df


def _dbl(*ts):
    return [None if t is None else t.double().cpu() for t in ts]


def _run(x, w, b, st, dy, df, act, cu, cu_arg=None, want_final=True, name=""):
    from tops.modules import causal_conv1d
    leaf = lambda t: None if t is None else t.cuda().requires_grad_()  # noqa: E731
    X, W_, Bb, S = leaf(x), leaf(w), leaf(b), leaf(st)
    y, fin = causal_conv1d(X, W_, Bb, "silu" if act else None, S, want_final, cu if cu_arg is None else cu_arg)
    outs, gs = [y], [dy.cuda()]
    if want_final:
        outs.append(fin)
        gs.append(df.cuda())
    else:
        assert fin is None
    leaves = [t for t in (X, W_, Bb, S) if t is not None]
    grads = dict(zip([n for n, t in (("dx", X), ("dw", W_), ("db", Bb), ("dstate", S)) if t is not None],
                     torch.autograd.grad(outs, leaves, gs)))
    r = conv_ref(*_dbl(x, w, b, st), act, cu, *_dbl(dy, df if want_final else None))
    rows = x.shape[0] * x.shape[1]
    close(name + "y", y, *r["y"], ONE)
    if want_final:
        assert torch.equal(fin.detach().double().cpu(), r["final"][0]), "final state is not the inputs"
    for k, v in grads.items():
        assert v.dtype == {"dx": x, "dw": w, "db": b, "dstate": st}[k].dtype
        close(name + k, v, *r[k], GRAD + (rows if k in ("dw", "db") else 0))
    return y, fin, grads


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B,T,D,W", [(1, 1, 1, 4), (2, 2, 7, 4), (3, 3, 64, 3), (1, 5, 72, 2), (2, 64, 40, 4),
                                     (2, 257, 64, 4), (1, 300, 1000, 4), (2, 33, 129, 3)])
@pytest.mark.parametrize("act,bias,state", [(1, False, False), (0, True, True), (1, True, True)])
def test_conv_fixed(dt, B, T, D, W, act, bias, state):
    _run(*_mk(1, B, T, D, W, DT[dt], B, bias, state), act, None)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("D", [64, 37])
@pytest.mark.parametrize("W", [2, 4])
@pytest.mark.parametrize("cu", [[0, 1], [0, 0, 9, 9, 10, 12, 15, 200], [0, 70, 70], [0, 3, 5, 8, 8, 8, 40]])
def test_conv_packed(dt, D, W, cu):
    T, N = cu[-1], len(cu) - 1
    args = _mk(2, 1, T, D, W, DT[dt], N, True, True)
    y, fin, g = _run(*args, 1, cu)
    # offsets on the GPU give the same bits
    y2, fin2, g2 = _run(*args, 1, cu, cu_arg=torch.tensor(cu, dtype=torch.int32, device="cuda"))
    assert torch.equal(y, y2) and torch.equal(fin, fin2) and all(torch.equal(g[k], g2[k]) for k in g)
    _run(*_mk(3, 1, T, D, W, DT[dt], N, False, False), 1, cu)


def test_conv_rows_behind_the_last_sequence():
    """GPU offsets may leave rows over: zeros, no gradient, whatever they hold."""
    from tops.modules import causal_conv1d
    x, w, b, st, dy, df = _mk(4, 1, 90, 64, 4, torch.bfloat16, 3, True, True)
    cu = [0, 20, 20, 61]
    x[:, 61:] = float("nan")
    X, W_ = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y, fin = causal_conv1d(X, W_, b.cuda(), "silu", st.cuda(), True, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    dx, dw = torch.autograd.grad([y, fin], [X, W_], [dy.cuda(), df.cuda()])
    r = conv_ref(*_dbl(x[:, :61], w, b, st), 1, cu, *_dbl(dy[:, :61], df))
    close("y", y[:, :61], *r["y"], ONE)
    close("dx", dx[:, :61], *r["dx"], GRAD)
    close("dw", dw, *r["dw"], GRAD + 61)
    assert torch.equal(y[:, 61:], torch.zeros_like(y[:, 61:])) and torch.equal(dx[:, 61:], torch.zeros_like(dx[:, 61:]))
    assert torch.equal(fin.detach().double().cpu(), r["final"][0])


def test_conv_nan_stays_in_its_sequence():
    from tops.modules import causal_conv1d
    x, w, b, st, dy, _ = _mk(5, 1, 60, 64, 4, torch.float32, 3, True, True)
    x[0, 20:40:7] = float("nan")
    x[0, 39] = float("inf")
    st[1, :, 1] = float("nan")
    X = x.cuda().requires_grad_()
    y, _ = causal_conv1d(X, w.cuda(), b.cuda(), "silu", st.cuda(), False, [0, 20, 40, 60])
    (dx,) = torch.autograd.grad(y, X, dy.cuda())
    for t in (y, dx):
        assert torch.isfinite(t[:, :20]).all() and torch.isfinite(t[:, 40:]).all()


@pytest.mark.parametrize("dt", DT)
def test_conv_strided_mixed_and_expanded(dt):
    """Slices of a wider projection (aligned, and at an odd offset), fp32 weights, an expanded gradient."""
    from tops.modules import causal_conv1d
    d = DT[dt]
    x, w, b, _, _, _ = _mk(6, 2, 50, 64, 4, d, 2, True, False, torch.float32)
    for off in (0, 16, 3):
        wide = torch.zeros(2, 50, 192, dtype=d, device="cuda")
        wide[..., off:off + 64] = x.cuda()
        X, W_ = wide[..., off:off + 64].detach().requires_grad_(), w.cuda().requires_grad_()
        assert not X.is_contiguous()
        y, _ = causal_conv1d(X, W_.unsqueeze(1), b.cuda(), "silu")
        dx, dw = torch.autograd.grad(y.sum(), [X, W_])
        r = conv_ref(*_dbl(x, w, b), None, 1, None, torch.ones(2, 50, 64, dtype=torch.float64))
        close("y", y, *r["y"], ONE)
        close("dx", dx, *r["dx"], GRAD)
        close("dw", dw, *r["dw"], GRAD + 100)
    t = x.cuda().transpose(0, 1)  # rows of a [T, B, D] tensor
    y, _ = causal_conv1d(t.contiguous().transpose(0, 1), w.cuda(), b.cuda(), "silu")
    close("y", y, *r["y"], ONE)


def test_conv_zero_rows_and_only_the_final_state():
    from tops.modules import causal_conv1d
    x, w, b, st, _, df = _mk(7, 2, 2, 16, 4, torch.float32, 2, True, True)
    st_ = st.cuda().requires_grad_()
    y, fin = causal_conv1d(x[:, :0].cuda(), w.cuda(), b.cuda(), None, st_, True)
    assert y.shape == (2, 0, 16) and torch.equal(fin, st.cuda())
    assert torch.equal(torch.autograd.grad(fin, st_, df.cuda())[0], df.cuda())
    X, st_ = x.cuda().requires_grad_(), st.cuda().requires_grad_()  # shorter than the state
    _, fin = causal_conv1d(X, w.cuda(), b.cuda(), None, st_, True)
    dx, ds = torch.autograd.grad(fin, [X, st_], df.cuda())
    assert torch.equal(dx.transpose(1, 2).cpu(), df[..., 1:])
    assert torch.equal(ds.cpu(), torch.cat([torch.zeros(2, 16, 2), df[..., :1]], -1))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B,D,W", [(1, 1, 4), (3, 64, 4), (5, 37, 3), (33, 128, 2), (2, 8, 3)])
def test_conv_steps_continue_a_prompt(dt, B, D, W):
    """Prompt, then tokens one at a time, equals the whole; in place too."""
    from tops.modules import causal_conv1d, causal_conv1d_step
    x, w, b, st, _, _ = _mk(8, B, 9, D, W, DT[dt], B, True, True)
    X, W_, Bb = x.cuda(), w.cuda(), b.cuda()
    r = conv_ref(*_dbl(x, w, b, st), 1, None)
    _, s = causal_conv1d(X[:, :4], W_, Bb, "silu", st.cuda(), True)
    keep = s.clone()
    for t in range(4, 9):
        y, s2 = causal_conv1d_step(X[:, t], s, W_, Bb, "silu")
        assert t > 4 or torch.equal(s, keep)
        y3, s3 = causal_conv1d_step(X[:, t], s, W_, Bb, "silu", state_out=s)
        assert s3 is s and torch.equal(s, s2) and torch.equal(y, y3)
        close(f"y{t}", y, r["y"][0][:, t], r["y"][1][:, t], ONE)
    assert torch.equal(s.double().cpu(), x[:, 9 - (W - 1):].transpose(1, 2).double())


def test_conv_second_derivative():
    from tops.modules import causal_conv1d
    x, w, b, st, dy, _ = _mk(9, 2, 11, 8, 4, torch.float32, 2, True, True)
    X, W_ = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y, _ = causal_conv1d(X, W_, b.cuda(), "silu", st.cuda())
    (dx,) = torch.autograd.grad(y, X, dy.cuda(), create_graph=True)
    got = torch.autograd.grad(dx.square().sum(), [X, W_])
    X2, W2 = x.double().requires_grad_(), w.double().requires_grad_()
    rows = torch.cat([st.double().transpose(1, 2), X2], 1)
    p = sum(rows[:, j:j + 11] * W2[:, j] for j in range(4)) + b.double()
    (dx2,) = torch.autograd.grad(torch.nn.functional.silu(p), X2, dy.double(), create_graph=True)
    for g, want in zip(got, torch.autograd.grad(dx2.square().sum(), [X2, W2])):
        # torch's conv1d may run in TF32 (11 bits) here: three chained products
        assert (g.double().cpu() - want).norm() <= 6 * 2.0 ** -11 * want.norm()


def test_conv_replayed_with_other_offsets_and_on_another_stream():
    from tops.modules import causal_conv1d
    x, w, b, st, _, _ = _mk(10, 1, 64, 64, 4, torch.float16, 4, True, True)
    X, W_, Bb, S = x.cuda(), w.cuda(), b.cuda(), st.cuda()
    cu = torch.tensor([0, 10, 20, 30, 64], dtype=torch.int32, device="cuda")
    causal_conv1d(X, W_, Bb, "silu", S, True, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, fin = causal_conv1d(X, W_, Bb, "silu", S, True, cu)
    for cuts in ([0, 10, 20, 30, 64], [0, 0, 1, 60, 61], [0, 64, 64, 64, 64]):
        cu.copy_(torch.tensor(cuts, dtype=torch.int32))
        graph.replay()
        e, f = causal_conv1d(X, W_, Bb, "silu", S, True, cu)
        assert torch.equal(y, e) and torch.equal(fin, f)
        r = conv_ref(*_dbl(x[:, :cuts[-1]], w, b, st), 1, cuts)
        close("y", y[:, :cuts[-1]], *r["y"], ONE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, _ = causal_conv1d(X, W_, Bb, "silu", S, True, cu)
    side.synchronize()
    assert torch.equal(y2, e)


def test_conv_wrong_gpu_offsets_stay_in_range():
    """Offsets below 0, past T or falling: wrong rows, but no access outside the tensors (they are
    clamped); the sequences with good offsets keep their values."""
    from tops.modules import causal_conv1d
    x, w, b, st, _, _ = _mk(11, 1, 40, 64, 4, torch.float32, 3, True, True)
    X = x.cuda().requires_grad_()
    cu = torch.tensor([-7, 12, 30, 10 ** 9], dtype=torch.int32, device="cuda")
    y, fin = causal_conv1d(X, w.cuda(), b.cuda(), "silu", st.cuda(), True, cu)
    torch.autograd.grad([y, fin], X, [torch.ones_like(y), torch.ones_like(fin)])
    r = conv_ref(*_dbl(x, w, b, st), 1, [0, 12, 30, 40])
    close("y", y, *r["y"], ONE)


def test_short_convolution_on_the_kernel():
    """ShortConvolution: the same values as torch's conv1d on the CPU, packed rows as single ones, and
    the cases that stay with torch."""
    from tops.layers import ShortConvolution
    torch.manual_seed(1)
    m = ShortConvolution(24, 4, bias=True)
    m.bias.data.normal_()
    x = torch.randn(2, 13, 24)
    want, cache = m(x, None, True)
    g = ShortConvolution(24, 4, bias=True).cuda()
    g.load_state_dict(m.state_dict())
    got, c2 = g(x.cuda(), None, True)
    r = conv_ref(*_dbl(x, m.weight.detach().squeeze(1), m.bias.detach(), None), 1, None)
    close("y", got, *r["y"], ONE)
    assert torch.equal(c2.cpu(), cache) and not c2.requires_grad
    packed, c3 = g(x.cuda().reshape(1, 26, 24), None, True, torch.tensor([0, 13, 26], device="cuda"))
    assert torch.equal(packed.view(2, 13, 24), got) and torch.equal(c3, c2)
    assert torch.equal(g(x.cuda()[:, :1], c2)[0], g(torch.cat([x, x[:, :1]], 1).cuda())[0][:, -1:])
    wide = ShortConvolution(24, 6).cuda()
    assert wide(x.cuda())[0].shape == x.shape
    with pytest.raises(NotImplementedError, match="kernel_size"):
        wide(x.cuda().reshape(1, 26, 24), None, False, [0, 13, 26])
    with torch.autocast("cuda", torch.bfloat16):
        assert g(x.cuda())[0].dtype == torch.bfloat16


def test_gla_layer_packs_its_short_convolutions():
    """A padded batch through the layer with short convolutions equals its rows one by one, and so does
    a step after it from the cache."""
    from tops.layers import GatedLinearAttention, GLACache
    torch.manual_seed(2)
    layer = GatedLinearAttention(hidden_size=64, num_heads=2, use_short_conv=True, layer_idx=0).cuda()
    x = torch.randn(3, 20, 64, device="cuda")
    lens = [20, 7, 1]
    mask = torch.zeros(3, 20, dtype=torch.long, device="cuda")
    for i, n in enumerate(lens):
        mask[i, 20 - n:] = 1
    cache = GLACache()
    o, _, cache = layer(x, mask, cache, use_cache=True)
    nxt = torch.randn(3, 1, 64, device="cuda")
    o2, _, _ = layer(nxt, None, cache, use_cache=True)
    # fp32 all the way; the projections may run in TF32 on both sides with other tilings
    tol = 8 * 2.0 ** -11
    for i, n in enumerate(lens):
        own = GLACache()
        p, _, own = layer(x[i:i + 1, 20 - n:], None, own, use_cache=True)
        assert (o[i, 20 - n:] - p[0]).abs().max() <= tol * p.abs().max()
        assert not o[i, :20 - n].any()
        p2, _, _ = layer(nxt[i:i + 1], None, own, use_cache=True)
        assert (o2[i] - p2[0]).abs().max() <= tol * p2.abs().max()


def test_conv_refusals():
    from tops.modules import causal_conv1d, causal_conv1d_step
    x, w, b, st, _, _ = (None if t is None else t.cuda() for t in _mk(12, 2, 8, 16, 4, torch.float32, 2, True, True))
    big = torch.zeros(100, device="cuda")
    for err, f in (
            (ValueError, lambda: causal_conv1d(x, w, activation="relu")),
            (ValueError, lambda: causal_conv1d(x, torch.randn(16, 5, device="cuda"))),
            (TypeError, lambda: causal_conv1d(x, w.half())),
            (TypeError, lambda: causal_conv1d(x.double(), w.double())),
            (TypeError, lambda: causal_conv1d(x, w, b.half())),
            (TypeError, lambda: causal_conv1d(x, w, b, None, st.half())),
            (AssertionError, lambda: causal_conv1d(x, w[:8])),
            (AssertionError, lambda: causal_conv1d(x[0], w)),
            (AssertionError, lambda: causal_conv1d(x, w, b, None, st[:1])),
            (AssertionError, lambda: causal_conv1d(x, w, cu_seqlens=[0, 8])),
            (AssertionError, lambda: causal_conv1d(x[:1], w, cu_seqlens=[0, 5])),
            (AssertionError, lambda: causal_conv1d(x[:1], w, cu_seqlens=[0, 6, 5, 8])),
            (TypeError, lambda: causal_conv1d(x[:1], w, cu_seqlens=torch.tensor([0., 8.], device="cuda"))),
            (RuntimeError, lambda: causal_conv1d(x, w.cpu())),
            (RuntimeError, lambda: causal_conv1d_step(x[:, 0].requires_grad_(), st, w)),
            (ValueError, lambda: causal_conv1d_step(x[:, 0], big[:96].view(2, 16, 3), w,
                                                    state_out=big[4:100].view(2, 16, 3))),
            (AssertionError, lambda: causal_conv1d_step(x[:, 0], st, w, state_out=st[:1])),
            (TypeError, lambda: causal_conv1d_step(x[:, 0], st, w, state_out=st.half()))):
        with pytest.raises(err):
            f()
