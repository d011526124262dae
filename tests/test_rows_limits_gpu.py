"""The short convolution, the selective scan and the query/key norm where programs go beyond one call on one stream:
captured backwards, two graphs, two streams at once, offsets past 32 bits, thousands of sequences, shared inputs."""
from __future__ import annotations

import pytest
import torch

from _rows_ref import close, conv_ref, qk_ref, scan_ref
from test_ssm_scan_gpu import NAMES, _call, _dbl, _mk, _roundings

pytestmark = pytest.mark.gpu


def _captured(step):
    """`step` captured into a graph after a warm-up on a side stream; -> (graph, its outputs)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    return g, out


def test_scan_backward_captured_and_replayed_with_other_offsets_and_inputs():
    """Two graphs of the same call, replayed in turn, each with what lies in its inputs at the time."""
    cu = torch.tensor([0, 60, 60, 200], dtype=torch.int32, device="cuda")
    t, dout, dht = _mk(1, 1, 200, 64, 16, 1, torch.bfloat16, 3)
    dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
    go, gh = dout.cuda(), dht.cuda()

    def step():
        y, ht = _call(dev, True, cu)
        grads = torch.autograd.grad([y, ht], [dev[k] for k in NAMES], [go, gh])
        return (y.detach(), ht.detach(), *grads)  # no graph of the leaves outlives the step

    (g1, o1), (g2, o2) = _captured(step), _captured(step)
    for seed, cuts in ((2, [0, 60, 60, 200]), (3, [0, 1, 130, 199]), (4, [0, 200, 200, 200])):
        t, dout, dht = _mk(seed, 1, 200, 64, 16, 1, torch.bfloat16, 3)
        with torch.no_grad():
            for k in NAMES:
                dev[k].copy_(t[k])
            go.copy_(dout)
            gh.copy_(dht)
            cu.copy_(torch.tensor(cuts, dtype=torch.int32))
        g1.replay()
        g2.replay()
        T = cuts[-1]
        cut = {k: v[:, :T] if k in ("x", "dt", "B", "C", "z") else v for k, v in t.items()}
        r = scan_ref(*(_dbl(cut[k]) for k in NAMES), True, cuts, _dbl(dout[:, :T]), _dbl(dht))
        n = _roundings(200, 16, 64, 200)
        for o in (o1, o2):
            for name, got in zip(("out", "ht", *("d" + k for k in NAMES)), o):
                rows = name in ("out", "dx", "ddt", "dB", "dC", "dz")
                close(name, got[:, :T] if rows else got, *r[name], n)
        assert all(torch.equal(a, b) for a, b in zip(o1, o2))


def test_conv_and_norm_backward_captured():
    from tops.modules import causal_conv1d, qk_norm_rotary, rotary_tables
    gen = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, w, b, dy = (v.cuda() for v in (rn(2, 70, 64), rn(64, 4), rn(64), rn(2, 70, 64)))
    q, k, qw, kw, dq, dk = (v.cuda() for v in (rn(2, 9, 4, 64), rn(2, 9, 2, 64), rn(64), rn(64), rn(2, 9, 4, 64), rn(2, 9, 2, 64)))
    cos, sin = rotary_tables(16, 32, device="cuda")
    leaves = [t.requires_grad_() for t in (x, w, b, q, k, qw, kw)]

    def step():
        y, _ = causal_conv1d(x, w, b, "silu")
        a, c = qk_norm_rotary(q, k, qw, kw, cos, sin)
        return torch.autograd.grad([y, a, c], leaves, [dy, dq, dk])

    g, out = _captured(step)
    for seed in (6, 7):
        gen.manual_seed(seed)
        with torch.no_grad():
            for t in (x, q, k):
                t.copy_(rn(*t.shape))
        g.replay()
        torch.cuda.synchronize()
        r = conv_ref(*(_dbl(t) for t in (x, w, b)), None, 1, None, _dbl(dy))
        for name, got, extra in (("dx", out[0], 0), ("dw", out[1], 140), ("db", out[2], 140)):
            close(name, got, *r[name], 48 + extra)
        pos = torch.arange(9).expand(2, 9)
        for got, gw, t, wt, d in ((out[3], out[5], q, qw, dq), (out[4], out[6], k, kw, dk)):
            f = qk_ref(_dbl(t), _dbl(wt), _dbl(cos), _dbl(sin), pos, 1e-6, False, _dbl(d))
            close("dx", got, f[2], f[3], 2 * 64 + 24)
            close("dw", gw, f[4], f[5], 2 * 64 + 24 + 72)


def test_two_streams_at_once():
    """Calls on two streams share nothing: each gives what it gives alone."""
    a = [_mk(s, 1, 700, 40, 16, 1, torch.float32, 1) for s in (8, 9)]
    dev = [({k: v.cuda().requires_grad_() for k, v in t.items()}, d.cuda(), h.cuda()) for t, d, h in a]

    def step(c, d, h):
        y, ht = _call(c, True, None)
        return (y, ht, *torch.autograd.grad([y, ht], [c[k] for k in NAMES], [d, h]))

    alone = [step(*c) for c in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    for _ in range(5):
        got = []
        for s, c in zip(streams, dev):
            with torch.cuda.stream(s):
                got.append(step(*c))
        torch.cuda.synchronize()
        for g, w in zip(got, alone):
            assert all(torch.equal(x, y) for x, y in zip(g, w))


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows are what a short call from the state before them gives."""
    from tops.modules import causal_conv1d
    from tops.ops.ssm import selective_scan
    T, D, N, last = (1 << 20) + 4096, 2048, 4, 96
    assert T * D > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    x, w = rn(1, T, D), rn(D, 4)
    y, fin = causal_conv1d(x, w, None, "silu", None, True)
    e, fe = causal_conv1d(x[:, -last:], w, None, "silu", x[:, -last - 3:-last].transpose(1, 2).contiguous(), True)
    assert torch.equal(y[:, -last:], e) and torch.equal(fin, fe)
    leaf = x.requires_grad_()
    y, _ = causal_conv1d(leaf, w, None, "silu")
    (dx,) = torch.autograd.grad(y, leaf, x.detach())
    sl = x[:, -last:].detach().requires_grad_()
    e, _ = causal_conv1d(sl, w, None, "silu", x[:, -last - 3:-last].detach().transpose(1, 2).contiguous())
    (de,) = torch.autograd.grad(e, sl, sl.detach())
    assert torch.equal(dx[:, -last:], de)
    del y, dx, e, de, leaf
    x = x.detach()
    dt, A = rn(1, T, D), -torch.rand(D, N, generator=g, device="cuda") - 0.5
    Bm, Cm = rn(1, T, N), rn(1, T, N)
    y, ht = selective_scan(x, dt, A, Bm, Cm, dt_softplus=True, output_final_state=True)
    _, h0 = selective_scan(x[:, :-last], dt[:, :-last], A, Bm[:, :-last], Cm[:, :-last], dt_softplus=True, output_final_state=True)
    e, he = selective_scan(x[:, -last:], dt[:, -last:], A, Bm[:, -last:], Cm[:, -last:], dt_softplus=True, initial_state=h0,
                           output_final_state=True)
    # the decays are at most exp(-0.5 softplus(dt)): a state forgets within some 100 rows, its rounding with it
    close("ht", ht, he, he.abs() + 1, 16 * 200)
    close("y", y[:, -last:], e.double(), e.abs().double() + 1, 16 * 200)


def test_thousands_of_sequences():
    from tops.modules import causal_conv1d
    gen = torch.Generator().manual_seed(2)
    S, T = 3000, 2000
    cu = [0] + torch.randint(0, T + 1, (S - 1,), generator=gen).sort().values.tolist() + [T]
    t, dout, dht = _mk(10, 1, T, 8, 4, 1, torch.float32, S)
    dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
    y, ht = _call(dev, True, torch.tensor(cu, device="cuda"))
    got = torch.autograd.grad([y, ht], [dev[k] for k in NAMES], [dout.cuda(), dht.cuda()])
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), True, cu, _dbl(dout), _dbl(dht))
    n = _roundings(64, 4, 8, T)
    close("out", y, *r["out"], n)
    close("ht", ht, *r["ht"], n)
    for k, v in zip(NAMES, got):
        close("d" + k, v, *r["d" + k], n)
    w = torch.randn(8, 4, generator=gen)
    y, _ = causal_conv1d(t["x"].cuda(), w.cuda(), None, "silu", None, False, cu)
    close("conv", y, *conv_ref(_dbl(t["x"]), _dbl(w), None, None, 1, cu)["y"], 24)


def test_scan_shared_and_expanded_inputs():
    """dt shared by all channels, A by all of them, B and C by the batch: their gradients are sums."""
    from tops.ops.ssm import selective_scan
    gen = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    B, T, D, N = 2, 33, 24, 8
    x, dt, A, Bm, Cm, dy = rn(B, T, D), rn(B, T, 1), -torch.rand(1, N, generator=gen) - 0.1, rn(1, T, N), rn(1, T, N), rn(B, T, D)
    leaves = [t.cuda().requires_grad_() for t in (x, dt, A, Bm, Cm)]
    X, d, a, b, c = leaves
    y, _ = selective_scan(X, d.expand(B, T, D), a.expand(D, N), b.expand(B, T, N), c.expand(B, T, N), dt_softplus=True)
    got = torch.autograd.grad(y, leaves, dy.cuda())
    r = scan_ref(_dbl(x), _dbl(dt.expand(B, T, D)), _dbl(A.expand(D, N)), _dbl(Bm.expand(B, T, N)).unsqueeze(2),
                 _dbl(Cm.expand(B, T, N)).unsqueeze(2), None, None, None, None, True, None, _dbl(dy))
    n = _roundings(T, N, D, B * T)
    close("y", y, *r["out"], n)
    fold = {"dx": lambda v: v, "ddt": lambda v: v.sum(-1, keepdim=True), "dA": lambda v: v.sum(0, keepdim=True),
            "dB": lambda v: v[:, :, 0].sum(0, keepdim=True), "dC": lambda v: v[:, :, 0].sum(0, keepdim=True)}
    for (k, f), v in zip(fold.items(), got):
        close(k, v, f(r[k][0]), f(r[k][1]), n + D)


def test_scan_groups_of_one_channel_and_many_states():
    t, dout, dht = _mk(11, 1, 20, 6, 64, 6, torch.float32, 1)
    dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
    y, ht = _call(dev, True, None)
    got = torch.autograd.grad([y, ht], [dev[k] for k in NAMES], [dout.cuda(), dht.cuda()])
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), True, None, _dbl(dout), _dbl(dht))
    n = _roundings(20, 64, 6, 20)
    close("out", y, *r["out"], n)
    for k, v in zip(NAMES, got):
        close("d" + k, v, *r["d" + k], n)
