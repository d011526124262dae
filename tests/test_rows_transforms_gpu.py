"""ShortConvolution, causal_conv1d, selective_scan and qk_norm_rotary where something else than plain eager autograd
looks at the call: tracing, forward mode, torch.func, batched and second gradients, fake tensors, dispatch modes."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.func import functional_call

from _rows_ref import U32, close, conv_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_tf32():
    """torch's conv1d in full fp32, so that one bound holds for both ways."""
    with torch.backends.cudnn.flags(enabled=True, benchmark=False, deterministic=True, allow_tf32=False):
        yield


def _pair(bias=True, seed=1, D=24):
    """The module on the GPU and the same in 64 bits on the CPU (torch's conv1d)."""
    from tops.modules import ShortConvolution
    torch.manual_seed(seed)
    g = ShortConvolution(D, 4, bias=bias)
    if bias:
        g.bias.data.normal_()
    c = ShortConvolution(D, 4, bias=bias).double()
    c.load_state_dict(g.state_dict())
    return g.cuda(), c


def _near(name, got, want, size=1.0, roundings=64):
    """|got - want| <= roundings * 2^-24 * (largest |want| + size): W products and sums, the activation and its first
    derivatives are at most 48 roundings of terms no larger than `size` (here W |w| |x| |dy|, below)."""
    g, w = got.detach().double().cpu(), want.detach().double().cpu()
    assert g.shape == w.shape, f"{name}: {tuple(g.shape)} {tuple(w.shape)}"
    assert torch.isfinite(g).all(), f"{name}: non-finite values"
    err = (g - w).abs().max().item()
    assert err <= roundings * U32 * (w.abs().max().item() + size), f"{name}: {err:.2e}"


SIZE = 4 * 0.5 * 5.0 * 5.0  # taps, |w| <= 1/2, normal inputs and tangents below 5


def test_traced_short_convolution():
    class Whole(torch.nn.Module):
        def __init__(self, m):
            super().__init__()
            self.m = m

        def forward(self, t):
            return self.m(t, None, True)

    g, c = _pair()
    x, x2 = torch.randn(2, 13, 24), torch.randn(2, 13, 24)
    with torch.no_grad():
        tr = torch.jit.trace(Whole(g), x.cuda(), check_trace=False)
        y, cache = tr(x2.cuda())
    want, wc = c(x2.double(), None, True)
    _near("y", y, want, SIZE)
    assert torch.equal(cache.double().cpu(), wc)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_short_convolution(grad):
    g, c = _pair()
    x, t, tw, cache, tc = (torch.randn(*s) for s in ((2, 13, 24), (2, 13, 24), (24, 1, 4), (2, 24, 3), (2, 24, 3)))

    def go(m, cast):
        with torch.set_grad_enabled(grad), fwAD.dual_level():
            dual = lambda p, q: fwAD.make_dual(cast(p), cast(q))  # noqa: E731
            w = fwAD.make_dual(m.weight.detach(), cast(tw))
            y, _ = functional_call(m, {"weight": w, "bias": m.bias.detach()}, (dual(x, t), dual(cache, tc)))
            only_w, _ = functional_call(m, {"weight": w, "bias": m.bias.detach()}, (cast(x),))
            return [v for r in (y, only_w) for v in fwAD.unpack_dual(r)]

    for i, (a, b) in enumerate(zip(go(g, lambda v: v.cuda()), go(c, lambda v: v.double()))):
        assert a is not None, f"output {i}: no tangent"
        _near(str(i), a, b, 4 * SIZE)


def test_short_convolution_under_torch_func():
    g, c = _pair()
    x, t = torch.randn(3, 2, 9, 24), torch.randn(2, 9, 24)

    def run(m, cast):
        ps = {k: v.detach() for k, v in m.named_parameters()}
        f = lambda p, v: functional_call(m, p, (v,))[0]  # noqa: E731
        loss = lambda p, v: f(p, v).square().sum()  # noqa: E731
        X = cast(x)
        return {"grad": torch.func.grad(loss)(ps, X[0])["weight"], "vmap": torch.vmap(lambda v: f(ps, v))(X),
                "per sample": torch.vmap(torch.func.grad(loss), (None, 0))(ps, X)["bias"],
                "jvp": torch.func.jvp(lambda v: f(ps, v), (X[0],), (cast(t),))[1],
                "hvp": torch.func.jvp(torch.func.grad(lambda v: loss(ps, v)), (X[0],), (cast(t),))[1]}

    got, want = run(g, lambda v: v.cuda()), run(c, lambda v: v.double())
    for k in want:
        _near(k, got[k], want[k], 20 * SIZE, 256)  # gradients of a square: one product more, sums of 18 rows


def test_batched_gradients_of_short_convolution():
    g, c = _pair()
    x, dy = torch.randn(2, 7, 24), torch.randn(3, 2, 7, 24)
    got, want = [], []
    for m, cast, out in ((g, lambda v: v.cuda(), got), (c, lambda v: v.double(), want)):
        X = cast(x).requires_grad_()
        y, _ = m(X)
        out.extend(torch.autograd.grad(y, [X, *m.parameters()], cast(dy), is_grads_batched=True))
    for i, (a, b) in enumerate(zip(got, want)):
        _near(str(i), a, b, SIZE, 256)


def test_tangent_of_the_gradient_reaches_the_input():
    """The gradient that goes in carries a tangent; dx is linear in it, so its tangent is the tangent's own gradient."""
    g, c = _pair()
    x, dy, t = (torch.randn(2, 7, 24) for _ in range(3))
    X, Xc = x.cuda().requires_grad_(), x.double().requires_grad_()
    y, _ = g(X)
    with fwAD.dual_level():
        (dx,) = torch.autograd.grad(y, X, fwAD.make_dual(dy.cuda(), t.cuda()))
        value, tangent = fwAD.unpack_dual(dx)
    assert tangent is not None
    yc, _ = c(Xc)
    for name, got, d in (("dx", value, dy), ("tangent", tangent, t)):
        _near(name, got, torch.autograd.grad(yc, Xc, d.double(), retain_graph=True)[0], SIZE)


def test_packed_gradients_refuse_batches_and_tangents():
    from tops.modules import causal_conv1d
    X, w = torch.randn(1, 12, 8, device="cuda").requires_grad_(), torch.randn(8, 4, device="cuda")
    y, _ = causal_conv1d(X, w, cu_seqlens=[0, 5, 12])
    dy = torch.randn(1, 12, 8, device="cuda")
    with pytest.raises(RuntimeError, match="batch"):
        torch.autograd.grad(y, X, dy[None], is_grads_batched=True)
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad(y, X, fwAD.make_dual(dy, dy), retain_graph=True)
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False):  # a mode that only looks on
        (a,) = torch.autograd.grad(y, X, dy, retain_graph=True)
    assert torch.equal(a, torch.autograd.grad(y, X, dy)[0])


def test_short_convolution_sees_modes_and_compilers():
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    g, c = _pair()
    x, x2 = torch.randn(2, 13, 24), torch.randn(2, 13, 24)
    with torch.no_grad():
        gm = make_fx(lambda t: g(t)[0])(x.cuda())
        _near("make_fx", gm(x2.cuda()), c(x2.double())[0], SIZE)
        with FlopCounterMode(display=False) as f:
            g(x.cuda())
        assert f.get_total_flops() > 0
        with torch._subclasses.FakeTensorMode(allow_non_fake_inputs=True) as mode:
            y, s = g(mode.from_tensor(x.cuda()), None, True)
        assert y.shape == (2, 13, 24) and s.shape == (2, 24, 3)
        _near("compiled", torch.compile(g, backend="eager")(x2.cuda())[0], c(x2.double())[0], SIZE)


def test_packed_short_convolution_under_modes_and_compilers():
    """Packed rows have the kernel alone: what only looks on does not keep them from it, what cannot follow it is told."""
    from torch.utils.flop_counter import FlopCounterMode
    g, _ = _pair()
    x = torch.randn(1, 20, 24, device="cuda")
    cu = torch.tensor([0, 7, 7, 20], dtype=torch.int32, device="cuda")
    want, state = g(x, None, True, cu)
    with FlopCounterMode(display=False):
        y, s = g(x, None, True, cu)
    assert torch.equal(y, want) and torch.equal(s, state)
    with torch.no_grad():
        y, s = torch.compile(g, backend="eager")(x, None, True, cu)
        assert torch.equal(y, want) and torch.equal(s, state)
        g.requires_grad_(False)  # a function's trace takes no parameter that does
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(lambda t: g(t, None, False, cu)[0], x, check_trace=False)
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.vmap(lambda t: g(t, None, False, cu)[0])(x[None])


def test_vmap_over_a_backward():
    """A batch of gradients by torch.vmap around autograd.grad, as by is_grads_batched."""
    g, c = _pair()
    x, dy = torch.randn(2, 7, 24), torch.randn(3, 2, 7, 24)
    got = []
    for m, cast in ((g, lambda v: v.cuda()), (c, lambda v: v.double())):
        X = cast(x).requires_grad_()
        y, _ = m(X)
        got.append(torch.vmap(lambda v, y=y, X=X: torch.autograd.grad(y, X, v, retain_graph=True)[0])(cast(dy)))
    _near("dx", *got, SIZE)


def _calls():
    """Every operator as a function of one tensor that requires nothing, with its argument."""
    from tops.modules import causal_conv1d, causal_conv1d_step, qk_norm_rotary
    from tops.ops.ssm import selective_scan, selective_scan_step
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    w, st, A, B, C, h = r(16, 4), r(2, 16, 3), -torch.rand(16, 4, device="cuda"), r(2, 8, 4), r(2, 8, 4), r(2, 16, 4)
    k = r(2, 8, 1, 16)
    return {"causal_conv1d": (lambda x: causal_conv1d(x, w)[0], r(2, 8, 16)),
            "causal_conv1d, weight": (lambda v: causal_conv1d(h.transpose(1, 2), v)[0], w),
            "causal_conv1d_step": (lambda x: causal_conv1d_step(x, st, w)[0], r(2, 16)),
            "selective_scan": (lambda x: selective_scan(x, x, A, B, C)[0], r(2, 8, 16)),
            "selective_scan, C": (lambda c: selective_scan(h.new_ones(2, 8, 16), h.new_ones(2, 8, 16), A, B, c)[0], C),
            "selective_scan_step": (lambda x: selective_scan_step(x, x, A, B[:, 0], C[:, 0], h)[0], r(2, 16)),
            "qk_norm_rotary": (lambda q: qk_norm_rotary(q, k)[0], r(2, 8, 2, 16))}


def test_operators_refuse_what_they_cannot_follow():
    """No tangent is dropped, no empty tensor recorded, nothing run on tensors without memory."""
    from torch.fx.experimental.proxy_tensor import make_fx
    for name, (f, x) in _calls().items():
        op = name.split(",")[0]
        f(x)
        with torch.no_grad():
            with pytest.raises(RuntimeError, match=f"{op}.*trac"):
                torch.jit.trace(f, x, check_trace=False)
            with fwAD.dual_level():
                with pytest.raises(RuntimeError, match=f"{op}.*tangent"):
                    f(fwAD.make_dual(x, torch.ones_like(x)))
                f(x)  # a level without a tangent is nothing to refuse
            with pytest.raises(RuntimeError, match=f"{op}.*trac"):
                make_fx(f)(x)
            with torch._subclasses.FakeTensorMode(allow_non_fake_inputs=True) as mode:
                with pytest.raises(RuntimeError, match=f"{op}.*(fake|trac)"):
                    f(mode.from_tensor(x))
        for t in (lambda: torch.vmap(f)(x[None]), lambda: torch.func.jvp(f, (x,), (x,)),
                  lambda: torch.func.grad(lambda v: f(v).sum())(x)):
            with pytest.raises(RuntimeError, match=f"{op}.*torch.func"):
                t()


def test_backwards_refuse_what_they_cannot_follow():
    for name, (f, x) in _calls().items():
        if "step" in name or name.startswith("causal"):
            continue
        X = x.clone().requires_grad_()
        y = f(X)
        dy = torch.ones_like(y)
        with fwAD.dual_level():
            with pytest.raises(RuntimeError, match="tangent"):
                torch.autograd.grad(y, X, fwAD.make_dual(dy, dy), retain_graph=True)
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.autograd.grad(y, X, dy[None], is_grads_batched=True)


def test_operators_inside_compiled_callers():
    """The graph breaks at the operator, which runs as it does alone."""
    for name, (f, x) in _calls().items():
        with torch.no_grad():
            want = f(x) * 2
            assert torch.equal(torch.compile(lambda t, f=f: f(t) * 2, backend="eager")(x), want), name


# -- second derivatives of the convolution ----------------------------------------------------------------------


def _second(dt, wdt, seed=5, B=2, T=11, D=8, W=4):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return {"x": rn(B, T, D).to(dt), "w": (rn(D, W) / 2).to(wdt), "b": (rn(D) / 4).to(wdt), "st": rn(B, D, W - 1).to(dt),
            "dy": rn(B, T, D).to(dt), "df": rn(B, D, W - 1).to(dt)}


def _form(x, w, b, st):
    T, W = x.shape[1], w.shape[1]
    rows = torch.cat([st.transpose(1, 2), x], 1)
    p = sum(rows[:, j:j + T] * w[:, j] for j in range(W)) + b
    return torch.nn.functional.silu(p), rows[:, T:].transpose(1, 2)


@pytest.mark.parametrize("dt,wdt", [(torch.float32,) * 2, (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_first_gradients_are_the_same_bits_with_create_graph(dt, wdt):
    from tops.modules import causal_conv1d
    s = {k: v.cuda().requires_grad_() for k, v in _second(dt, wdt).items()}
    leaves = [s[k] for k in ("x", "w", "b", "st")]
    got = []
    for create in (False, True):
        y, fin = causal_conv1d(s["x"], s["w"], s["b"], "silu", s["st"], True)
        got.append(torch.autograd.grad([y, fin], leaves, [s["dy"], s["df"]], create_graph=create))
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(*got))
    assert all(g.requires_grad for g in got[1])


def test_second_and_third_derivatives_in_full_precision():
    from tops.modules import causal_conv1d
    cpu = _second(torch.float32, torch.float32)
    names = ("x", "w", "b", "st", "dy", "df")
    res = []
    for f, s in ((lambda *a: causal_conv1d(a[0], a[1], a[2], "silu", a[3], True), {k: v.cuda() for k, v in cpu.items()}),
                 (_form, {k: v.double() for k, v in cpu.items()})):
        s = {k: v.requires_grad_() for k, v in s.items()}
        y, fin = f(*(s[k] for k in names[:4]))
        first = torch.autograd.grad([y, fin], [s[k] for k in names[:4]], [s["dy"], s["df"]], create_graph=True)
        second = torch.autograd.grad(sum(g.square().sum() for g in first), [s[k] for k in names], create_graph=True)
        third = torch.autograd.grad(sum(g.square().sum() for g in second), [s[k] for k in names[:4]])
        res.append((*first, *second, *third))
    # each derivative adds at most 64 roundings to terms whose sums do not cancel by more than 2^6 here
    for i, (a, b) in enumerate(zip(*res)):
        rel = ((a.double().cpu() - b).norm() / b.norm()).item()
        assert rel <= 64 * 2 ** 6 * U32, f"{i}: {rel:.2e}"


def test_create_graph_of_frozen_inputs():
    """Only the weight is trained, and the final state, which does not depend on it, has a gradient too."""
    from tops.modules import causal_conv1d
    s = {k: v.cuda() for k, v in _second(torch.float32, torch.float32).items()}
    w = s["w"].requires_grad_()
    y, fin = causal_conv1d(s["x"], w, s["b"], "silu", s["st"], True)
    (dw,) = torch.autograd.grad([y, fin], w, [s["dy"], s["df"]], create_graph=True)
    (ddw,) = torch.autograd.grad(dw.square().sum(), w)
    W2 = s["w"].detach().double().cpu().requires_grad_()
    y2, _ = _form(s["x"].double().cpu(), W2, s["b"].double().cpu(), s["st"].double().cpu())
    (want,) = torch.autograd.grad(y2, W2, s["dy"].double().cpu(), create_graph=True)
    (ddwant,) = torch.autograd.grad(want.square().sum(), W2)
    for a, b in ((dw, want), (ddw, ddwant)):
        assert ((a.double().cpu() - b).norm() / b.norm()).item() <= 64 * 2 ** 6 * U32
    # the final state alone
    _, fin = causal_conv1d(s["x"], w, s["b"], "silu", s["st"], True)
    (dw,) = torch.autograd.grad(fin, w, s["df"], create_graph=True, allow_unused=True)
    assert dw is None or not dw.any()


def test_create_graph_of_packed_rows():
    """First gradients as without it; the second is refused."""
    from tops.modules import causal_conv1d
    s = {k: v.cuda() for k, v in _second(torch.float32, torch.float32).items()}
    w = s["w"].requires_grad_()
    X = s["x"].reshape(1, 22, 8).requires_grad_()
    args = (X, w, s["b"], "silu", s["st"], False, [0, 11, 22])
    y, _ = causal_conv1d(*args)
    dy = s["dy"].reshape(1, 22, 8)
    (dx,) = torch.autograd.grad(y, X, dy, create_graph=True)
    (dx2,) = torch.autograd.grad(causal_conv1d(*args)[0], X, dy)
    assert torch.equal(dx, dx2)
    with pytest.raises(RuntimeError, match="packed sequences"):
        torch.autograd.grad(dx.sum(), X)


def test_one_tensor_in_two_places():
    """The gradient that goes in is the input itself: both ways count once."""
    from tops.modules import causal_conv1d
    s = {k: v.cuda() for k, v in _second(torch.float32, torch.float32).items()}
    X = s["x"].requires_grad_()
    y, _ = causal_conv1d(X, s["w"], s["b"], "silu", s["st"])
    (dx,) = torch.autograd.grad(y, X, X, create_graph=True)
    (got,) = torch.autograd.grad(dx.square().sum(), X)
    X2 = s["x"].detach().double().cpu().requires_grad_()
    y2, _ = _form(X2, *(s[k].double().cpu() for k in ("w", "b", "st")))
    (dx2,) = torch.autograd.grad(y2, X2, X2, create_graph=True)
    (want,) = torch.autograd.grad(dx2.square().sum(), X2)
    assert ((got.double().cpu() - want).norm() / want.norm()).item() <= 64 * 2 ** 6 * U32


def test_eager_short_convolution():
    """Eager calls stay on the kernel: its values within its own, tighter bound."""
    g, c = _pair(bias=False, D=40)
    x = torch.randn(2, 30, 40)
    r = conv_ref(x.double(), c.weight.detach().squeeze(1), None, None, 1, None)
    close("y", g(x.cuda())[0], *r["y"], 24)
