"""selective_scan and selective_scan_step on the GPU against the formulas in 64 bits."""
from __future__ import annotations

import pytest
import torch

from _rows_ref import close, scan_ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NAMES = ("x", "dt", "A", "B", "C", "D", "z", "bias", "h0")


def _roundings(T, N, ch, rows):
    """A state is a product of up to T decays, each off by the rounding of delta (softplus: 8 steps), of
    delta A log2(e) and of the exponential (2 steps; |delta A| stays below 3 here: 12 in all), and a sum
    of T terms; the rest are sums over N, the channels and the rows, and the gates (16)."""
    return 16 * T + N + ch + rows + 64


def _mk(seed, B, T, ch, N, G, dt, S, z=True, skip=True, bias=True, h0=True):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": rn(B, T, ch).to(dt), "dt": rn(B, T, ch).to(dt), "B": rn(B, T, G, N).to(dt), "C": rn(B, T, G, N).to(dt),
         "z": rn(B, T, ch).to(dt) if z else None, "A": -torch.rand(ch, N, generator=g) - 0.05,
         "D": rn(ch) if skip else None, "bias": rn(ch) - 2 if bias else None, "h0": rn(S, ch, N) if h0 else None}
    return t, rn(B, T, ch).to(dt), rn(S, ch, N)


def _dbl(t):
    return None if t is None else t.detach().double().cpu()


def _call(t, softplus, cu, final=True):
    from tops.ops.ssm import selective_scan
    return selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], t["D"], t["z"], t["bias"], softplus, t["h0"], final, cu)


def _check(t, dout, dht, softplus, cu, cu_arg=None, rows=None):
    dev = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    y, ht = _call(dev, softplus, cu if cu_arg is None else cu_arg)
    leaves = [k for k in NAMES if dev[k] is not None]
    grads = dict(zip(leaves, torch.autograd.grad([y, ht], [dev[k] for k in leaves], [dout.cuda(), dht.cuda()])))
    cut = lambda v: v if rows is None else v[:, :rows]  # noqa: E731
    r = scan_ref(*(_dbl(cut(t[k])) if k in ("x", "dt") else _dbl(t[k]) if k in ("A", "D", "bias", "h0") else
                   (None if t[k] is None else _dbl(cut(t[k]))) for k in ("x", "dt", "A", "B", "C", "D", "z", "bias", "h0")),
                 softplus, cu, _dbl(cut(dout)), _dbl(dht))
    B, T, ch = cut(t["x"]).shape
    n = _roundings(T, t["A"].shape[1], ch, B * T)
    close("out", cut(y), *r["out"], n)
    close("ht", ht, *r["ht"], n)
    for k, v in grads.items():
        assert v.dtype == t[k].dtype
        close("d" + k, cut(v) if k in ("x", "dt", "z", "B", "C") else v, *r["d" + k], n)
    with torch.no_grad():  # without a graph: the same bits
        y2, ht2 = _call(dev, softplus, cu if cu_arg is None else cu_arg)
    close("out, no grad", cut(y2), *r["out"], n)
    close("ht, no grad", ht2, *r["ht"], n)
    return y, ht, grads


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B,T,ch,N,G", [(1, 1, 1, 1, 1), (2, 2, 6, 16, 2), (1, 3, 64, 4, 1), (2, 15, 40, 16, 1),
                                        (1, 16, 33, 8, 3), (2, 17, 64, 11, 1), (1, 65, 130, 16, 2), (2, 200, 24, 3, 1),
                                        (1, 40, 20, 32, 1), (1, 33, 12, 64, 2), (3, 31, 8, 17, 1)])
def test_scan_fixed(dt, B, T, ch, N, G):
    _check(*_mk(1, B, T, ch, N, G, DT[dt], B), True, None)


@pytest.mark.parametrize("softplus,z,skip,bias,h0", [(False, False, False, False, False), (True, False, True, False, True),
                                                     (True, True, False, True, False)])
def test_scan_without_optional_parts(softplus, z, skip, bias, h0):
    t, dout, dht = _mk(2, 2, 37, 48, 16, 1, torch.float32, 2, z, skip, bias, h0)
    if not softplus:
        t["dt"] = t["dt"].abs() / 4
    _check(t, dout, dht, softplus, None)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("ch,N,G", [(64, 16, 1), (36, 5, 2)])
@pytest.mark.parametrize("cu", [[0, 1], [0, 0, 9, 9, 10, 12, 15, 130], [0, 70, 70], [0, 16, 32, 33, 64], [0, 3, 5, 8, 8, 8, 40]])
def test_scan_packed(dt, ch, N, G, cu):
    T, S = cu[-1], len(cu) - 1
    t, dout, dht = _mk(3, 1, T, ch, N, G, DT[dt], S)
    y, ht, g = _check(t, dout, dht, True, cu)
    y2, ht2, g2 = _check(t, dout, dht, True, cu, torch.tensor(cu, dtype=torch.int64, device="cuda"))
    assert torch.equal(y, y2) and torch.equal(ht, ht2) and all(torch.equal(g[k], g2[k]) for k in g)
    t["h0"] = None
    _check(t, dout, dht, True, cu)


@pytest.mark.parametrize("T,ch,B", [(1500, 16, 1), (1031, 40, 2)])
def test_scan_long_rows_of_few_channels(T, ch, B):
    """So few channels that the time axis is split."""
    _check(*_mk(4, B, T, ch, 16, 1, torch.float32, B), True, None)
    _check(*_mk(5, B, T, ch, 16, 1, torch.bfloat16, B), True, None)


def test_scan_long_packed_rows_of_few_channels():
    cu = [0, 700, 701, 701, 1100, 1400]
    t, dout, dht = _mk(6, 1, 1400, 24, 16, 1, torch.float32, 5)
    _check(t, dout, dht, True, cu)


def test_scan_rows_behind_the_last_sequence():
    t, dout, dht = _mk(7, 1, 150, 64, 16, 1, torch.bfloat16, 4)
    cu = [0, 20, 20, 61, 97]
    for k in ("x", "dt", "B", "C", "z"):
        t[k][:, 97:] = float("nan")
    y, ht, g = _check(t, dout, dht, True, cu, torch.tensor(cu, dtype=torch.int32, device="cuda"), rows=97)
    for v in (y, g["x"], g["dt"], g["z"], g["B"], g["C"]):
        assert torch.equal(v[:, 97:], torch.zeros_like(v[:, 97:]))


def test_scan_nan_stays_in_its_sequence():
    t, dout, dht = _mk(8, 1, 96, 64, 16, 1, torch.float32, 3)
    t["x"][0, 40] = float("nan")
    t["dt"][0, 50] = float("inf")
    t["B"][0, 33] = float("inf")
    t["h0"][1] = float("nan")
    dev = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    y, ht = _call(dev, True, [0, 32, 64, 96])
    g = torch.autograd.grad([y, ht], [dev["x"], dev["dt"], dev["B"], dev["C"], dev["h0"]], [dout.cuda(), dht.cuda()])
    assert torch.isfinite(ht[0]).all() and torch.isfinite(ht[2]).all() and torch.isnan(ht[1]).any()
    for v in (y, *g[:4]):
        assert torch.isfinite(v[:, :32]).all() and torch.isfinite(v[:, 64:]).all()
    assert torch.isfinite(g[4][0]).all() and torch.isfinite(g[4][2]).all()


@pytest.mark.parametrize("dt", DT)
def test_scan_slices_of_projections(dt):
    """x, z, B and C as slices (aligned, and at odd offsets), A in another type, a gradient that is expanded."""
    from tops.ops.ssm import selective_scan
    t, _, _ = _mk(9, 2, 37, 64, 16, 2, DT[dt], 2)
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), True, None, torch.ones(2, 37, 64, dtype=torch.float64), None)
    n = _roundings(37, 16, 64, 74)
    for off in (0, 8, 3):
        def part(v):
            flat = v.reshape(2, 37, -1).cuda()
            wide = torch.zeros(2, 37, flat.shape[-1] + 16, dtype=v.dtype, device="cuda")
            wide[..., off:off + flat.shape[-1]] = flat
            return wide[..., off:off + flat.shape[-1]].view(v.shape).detach().requires_grad_()
        x, z, d, Bm, Cm = (part(t[k]) for k in ("x", "z", "dt", "B", "C"))
        A = t["A"].cuda().double().requires_grad_()
        y, ht = selective_scan(x, d, A, Bm, Cm, t["D"].cuda(), z, t["bias"].cuda(), True, t["h0"].cuda())
        assert ht is None
        got = torch.autograd.grad(y.sum(), [x, d, Bm, Cm, z, A])
        close("out", y, *r["out"], n)
        for k, v in zip(("dx", "ddt", "dB", "dC", "dz", "dA"), got):
            close(k, v.float() if k == "dA" else v, *r[k], n)


def test_scan_shared_b_and_c_without_a_group_dim():
    from tops.ops.ssm import selective_scan
    t, _, _ = _mk(10, 2, 21, 32, 8, 1, torch.float32, 2)
    c = {k: None if v is None else v.cuda() for k, v in t.items()}
    a, _ = _call(c, True, None)
    b, _ = selective_scan(c["x"], c["dt"], c["A"], c["B"][:, :, 0], c["C"][:, :, 0], c["D"], c["z"], c["bias"], True,
                          c["h0"], True)
    assert torch.equal(a, b)


def test_scan_zero_rows():
    t, _, dht = _mk(11, 2, 1, 16, 4, 1, torch.float32, 2)
    c = {k: None if v is None else v.cuda() for k, v in t.items()}
    for k in ("x", "dt", "B", "C", "z"):
        c[k] = c[k][:, :0]
    c["h0"].requires_grad_()
    y, ht = _call(c, True, None)
    assert y.shape == (2, 0, 16) and torch.equal(ht, c["h0"])
    (g,) = torch.autograd.grad(ht, c["h0"], dht.cuda())
    assert torch.equal(g.cpu(), dht)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("B,ch,N,G", [(1, 1, 1, 1), (3, 64, 16, 1), (5, 30, 11, 2), (2, 40, 64, 4), (33, 128, 8, 1), (2, 24, 6, 1)])
def test_scan_steps_continue_a_prompt(dt, B, ch, N, G):
    from tops.ops.ssm import selective_scan_step
    t, _, _ = _mk(12, B, 9, ch, N, G, DT[dt], B)
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), True, None)
    c = {k: None if v is None else v.cuda() for k, v in t.items()}
    pre = dict(c, **{k: c[k][:, :4] for k in ("x", "dt", "B", "C", "z")})
    _, s = _call(pre, True, None)
    n = _roundings(9, N, ch, 9)
    for i in range(4, 9):
        a = (c["x"][:, i], c["dt"][:, i], c["A"], c["B"][:, i], c["C"][:, i])
        kw = dict(D=c["D"], z=c["z"][:, i], dt_bias=c["bias"], dt_softplus=True)
        y, s2 = selective_scan_step(*a, s, **kw)
        y3, s3 = selective_scan_step(*a, s, **kw, state_out=s)
        assert s3 is s and torch.equal(s, s2) and torch.equal(y, y3)
        close(f"y{i}", y, r["out"][0][:, i], r["out"][1][:, i], n)
    close("state", s, *r["ht"], n)


def test_scan_step_of_many_rows_is_its_parts():
    """So many rows that a thread takes eight of them: the same bits as from calls of few rows."""
    from tops.ops.ssm import selective_scan_step
    B, ch, N = 157, 2048, 16
    t, _, _ = _mk(19, B, 1, ch, N, 1, torch.bfloat16, B)
    c = {k: v.cuda() for k, v in t.items()}

    def step(a, b):
        return selective_scan_step(c["x"][a:b, 0], c["dt"][a:b, 0], c["A"], c["B"][a:b, 0], c["C"][a:b, 0], c["h0"][a:b],
                                   D=c["D"], z=c["z"][a:b, 0], dt_bias=c["bias"], dt_softplus=True)

    y, s = step(0, B)
    parts = [step(a, min(a + 40, B)) for a in range(0, B, 40)]
    assert torch.equal(y, torch.cat([p[0] for p in parts])) and torch.equal(s, torch.cat([p[1] for p in parts]))
    r = scan_ref(*(_dbl(t[k][-2:]) if k in ("x", "dt", "B", "C", "z", "h0") else _dbl(t[k]) for k in NAMES), True, None)
    close("y", y[-2:], r["out"][0][:, 0], r["out"][1][:, 0], _roundings(1, N, ch, 1))
    close("s", s[-2:], *r["ht"], _roundings(1, N, ch, 1))


def test_scan_step_without_optional_parts():
    from tops.ops.ssm import selective_scan_step
    t, _, _ = _mk(13, 4, 1, 32, 16, 1, torch.float32, 4, False, False, False)
    t["dt"] = t["dt"].abs()
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), False, None)
    c = {k: None if v is None else v.cuda() for k, v in t.items()}
    y, s = selective_scan_step(c["x"][:, 0], c["dt"][:, 0], c["A"], c["B"][:, 0, 0], c["C"][:, 0, 0], c["h0"])
    close("y", y, r["out"][0][:, 0], r["out"][1][:, 0], _roundings(1, 16, 32, 1))
    close("s", s, *r["ht"], _roundings(1, 16, 32, 1))


def test_scan_replayed_with_other_offsets_and_on_another_stream():
    t, _, _ = _mk(14, 1, 64, 64, 16, 1, torch.float16, 4)
    c = {k: None if v is None else v.cuda() for k, v in t.items()}
    cu = torch.tensor([0, 10, 20, 30, 64], dtype=torch.int32, device="cuda")
    _call(c, True, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, ht = _call(c, True, cu)
    for cuts in ([0, 10, 20, 30, 64], [0, 0, 1, 60, 61], [0, 64, 64, 64, 64]):
        cu.copy_(torch.tensor(cuts, dtype=torch.int32))
        graph.replay()
        e, f = _call(c, True, cu)
        assert torch.equal(y, e) and torch.equal(ht, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, _ = _call(c, True, cu)
    side.synchronize()
    assert torch.equal(y2, e)


def test_scan_wrong_gpu_offsets_stay_in_range():
    t, dout, _ = _mk(15, 1, 40, 64, 16, 1, torch.float32, 3)
    c = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    cu = torch.tensor([-7, 12, 30, 10 ** 9], dtype=torch.int32, device="cuda")
    y, ht = _call(c, True, cu)
    torch.autograd.grad([y, ht], [c["x"], c["h0"]], [dout.cuda(), torch.ones_like(ht)])
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), True, [0, 12, 30, 40])
    close("out", y, *r["out"], _roundings(40, 16, 64, 40))
    close("ht", ht, *r["ht"], _roundings(40, 16, 64, 40))


def test_scan_two_backwards_give_the_same_bits():
    """No sum depends on the order in which blocks finish."""
    t, dout, dht = _mk(16, 2, 300, 136, 16, 1, torch.float32, 2)
    c = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    runs = []
    for _ in range(3):
        y, ht = _call(c, True, None)
        runs.append((y, ht, *torch.autograd.grad([y, ht], list(c.values()), [dout.cuda(), dht.cuda()])))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_scan_far_states_keep_small_decays():
    """Step sizes as small as training starts from: the decay lies next to 1 and thousands of tokens add up."""
    g = torch.Generator().manual_seed(17)
    B, T, ch, N = 1, 4096, 32, 16
    t = {"x": torch.randn(B, T, ch, generator=g), "dt": torch.full((B, T, ch), -6.9), "B": torch.randn(B, T, 1, N, generator=g),
         "C": torch.randn(B, T, 1, N, generator=g), "z": None, "A": -torch.arange(1, N + 1.0).expand(ch, N).contiguous(),
         "D": None, "bias": None, "h0": None}
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), True, None)
    y, ht = _call({k: None if v is None else v.cuda() for k, v in t.items()}, True, None)
    for name, got in (("out", y), ("ht", ht)):
        want = r[name][0]
        rel = ((got.double().cpu() - want).norm() / want.norm()).item()
        # a decay is off by at most 3 * 2^-23 a step (rounding of the exponent and of the exponential); a
        # state remembers 1 / (delta n) ~ 1000 / n steps, and the error grows with that memory
        assert rel <= 3 * 2.0 ** -23 * 1000, f"{name}: {rel:.2e}"


def test_scan_refusals():
    from tops.ops.ssm import selective_scan, selective_scan_step
    t, _, _ = _mk(18, 2, 8, 16, 4, 1, torch.float32, 2)
    c = {k: v.cuda() for k, v in t.items()}
    base = [c["x"], c["dt"], c["A"], c["B"], c["C"]]
    def go(i=None, v=None, **kw):
        a = list(base)
        if i is not None:
            a[i] = v
        return lambda: selective_scan(*a, **kw)
    step = [c["x"][:, 0], c["dt"][:, 0], c["A"], c["B"][:, 0], c["C"][:, 0], c["h0"]]
    big = torch.zeros(2 * 16 * 4 + 8, device="cuda")
    for err, f in ((AssertionError, go(1, c["dt"][:, :4])), (TypeError, go(1, c["dt"].half())),
                   (AssertionError, go(2, c["A"][:8])), (ValueError, go(2, torch.zeros(16, 65, device="cuda"))),
                   (AssertionError, go(3, c["B"][..., :3])), (AssertionError, go(3, c["B"].expand(2, 8, 3, 4))),
                   (RuntimeError, go(2, c["A"].cpu())), (AssertionError, go(initial_state=c["h0"][:1])),
                   (AssertionError, go(D=c["D"][:3])), (AssertionError, go(dt_bias=c["D"][:3])),
                   (TypeError, go(z=c["z"].half())), (AssertionError, go(cu_seqlens=[0, 8])),
                   (AssertionError, go(0, c["x"][0])), (TypeError, go(0, c["x"].double())),
                   (TypeError, lambda: selective_scan_step(*step[:5], c["h0"].half())),
                   (AssertionError, lambda: selective_scan_step(*step[:5], c["h0"][:1])),
                   (RuntimeError, lambda: selective_scan_step(*step[:5], c["h0"].clone().requires_grad_())),
                   (ValueError, lambda: selective_scan_step(*step[:5], big[:128].view(2, 16, 4),
                                                            state_out=big[4:132].view(2, 16, 4)))):
        with pytest.raises(err):
            f()
    x = c["x"].clone().requires_grad_()
    y, _ = selective_scan(x, *base[1:])
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)
