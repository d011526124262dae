"""64-bit references of the short convolution, the selective scan and the query/key norm, from their
formulas, and the tolerances that go with them.

Each reference returns (value, size) pairs: ``size`` is the same expression with every term replaced by
its absolute value, so rounding errors of a sum are at most (roundings per term) * 2^-24 * size however
much the terms cancel.  ``close`` allows that plus half a step of the stored type.
"""
from __future__ import annotations

import torch

U32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(name, got, want, size, roundings, floor=0.0):
    """|got - want| <= half a step of got's type * |want| + roundings * 2^-24 * size (+ floor)."""
    assert got.shape == want.shape, f"{name}: shape {tuple(got.shape)}, expected {tuple(want.shape)}"
    g, w = got.detach().double().cpu(), want.double().cpu()
    assert torch.isfinite(g).all(), f"{name}: non-finite values"
    # a stored value below the type's smallest normal is rounded to a fixed step
    tiny = torch.finfo(got.dtype).smallest_normal * half_step(got.dtype)
    extra = roundings * U32 * size.double().cpu()
    bound = half_step(got.dtype) * (w.abs() + extra) + extra + tiny + floor
    worst = ((g - w).abs() / bound.clamp(min=1e-300)).max().item() if g.numel() else 0.0
    assert worst <= 1.0, f"{name}: error / tolerance {worst:.2f}, largest error {(g - w).abs().max():.3e}"


def cuts_of(B, T, cu):
    """[(batch row, start, end)] of every sequence."""
    return [(b, 0, T) for b in range(B)] if cu is None else [(0, a, b) for a, b in zip(cu, cu[1:])]


def _silu(p):
    return p * torch.sigmoid(p)


def _dsilu(p):
    s = torch.sigmoid(p)
    return s * (1 + p * (1 - s))


def conv_ref(x, w, bias, state, act, cu, dy=None, dfinal=None):
    """All double CPU tensors.  -> dict name -> (value, size)."""
    B, T, D = x.shape
    W = w.shape[1]
    seqs = cuts_of(B, T, cu)
    st = torch.zeros(len(seqs), D, W - 1, dtype=x.dtype) if state is None else state
    y, ys = torch.zeros_like(x), torch.zeros_like(x)
    fin = torch.zeros_like(st)
    z = lambda t: torch.zeros_like(t)  # noqa: E731
    dx, dxs, dw, dws, ds, dss = z(x), z(x), z(w), z(w), z(st), z(st)
    db, dbs = torch.zeros(D, dtype=x.dtype), torch.zeros(D, dtype=x.dtype)
    for n, (b, s, e) in enumerate(seqs):
        rows = torch.cat([st[n].t(), x[b, s:e]])  # [W - 1 + len, D]
        L = e - s
        p = sum(rows[j:j + L] * w[:, j] for j in range(W)) + (0 if bias is None else bias)
        ps = sum(rows[j:j + L].abs() * w[:, j].abs() for j in range(W)) + (0 if bias is None else bias.abs())
        # |act'| <= 1.1: an error of p reaches y at most that much enlarged, and y itself is rounded
        y[b, s:e], ys[b, s:e] = (_silu(p) if act else p), 1.1 * ps
        fin[n] = rows[L:].t()
        if dy is None:
            continue
        d = dy[b, s:e] * (_dsilu(p) if act else 1)
        # |act''| <= 0.5: an error of p in act'
        dsz = dy[b, s:e].abs() * (1.1 + (0.5 * ps if act else 0))
        drows, drs = torch.zeros_like(rows), torch.zeros_like(rows)
        for j in range(W):
            drows[j:j + L] += d * w[:, j]
            drs[j:j + L] += dsz * w[:, j].abs()
            dw[:, j] += (d * rows[j:j + L]).sum(0)
            dws[:, j] += (dsz * rows[j:j + L].abs()).sum(0)
        if dfinal is not None:
            drows[L:] += dfinal[n].t()
            drs[L:] += dfinal[n].t().abs()
        db += d.sum(0)
        dbs += dsz.sum(0)
        ds[n], dss[n] = drows[:W - 1].t(), drs[:W - 1].t()
        dx[b, s:e], dxs[b, s:e] = drows[W - 1:], drs[W - 1:]
    return {"y": (y, ys), "final": (fin, fin.abs()), "dx": (dx, dxs), "dw": (dw, dws), "db": (db, dbs),
            "dstate": (ds, dss)}


def scan_ref(x, dt, A, Bm, Cm, D, z, bias, h0, softplus, cu, dout=None, dht=None):
    """All double CPU tensors; Bm, Cm [B, T, G, N].  -> dict name -> (value, size)."""
    rows, T, ch = x.shape
    G, N = Bm.shape[2:]
    rep = lambda t: t.repeat_interleave(ch // G, -2)  # noqa: E731
    seqs = cuts_of(rows, T, cu)
    v = dt + (0 if bias is None else bias)
    delta = torch.nn.functional.softplus(v) if softplus else v
    dv_dv = torch.sigmoid(v) if softplus else torch.ones_like(v)
    gate = torch.ones_like(x) if z is None else _silu(z)
    skip = torch.zeros(ch, dtype=x.dtype) if D is None else D
    st = torch.zeros(len(seqs), ch, N, dtype=x.dtype) if h0 is None else h0
    out = {}
    new = lambda name, like: out.setdefault(name, (torch.zeros_like(like), torch.zeros_like(like)))  # noqa: E731
    for name, like in (("out", x), ("ht", st), ("dx", x), ("ddt", x), ("dz", x), ("dA", A), ("dB", Bm), ("dC", Cm),
                       ("dD", skip), ("dbias", skip), ("dh0", st)):
        new(name, like)

    def both(fn):
        """(fn of the values, fn of the sizes): `m` marks an absolute value in the size."""
        return fn(lambda t: t), fn(torch.abs)

    for n, (b, s, e) in enumerate(seqs):
        hv, hs = [st[n]], [st[n].abs()]
        a = torch.exp(delta[b, s:e, :, None] * A)
        Bt, Ct = rep(Bm[b, s:e]), rep(Cm[b, s:e])
        ya, yb = [], []
        for i in range(e - s):
            u = (delta[b, s + i] * x[b, s + i])[:, None] * Bt[i]
            hv.append(a[i] * hv[-1] + u)
            hs.append(a[i] * hs[-1] + u.abs())
            ya.append((Ct[i] * hv[-1]).sum(-1) + skip * x[b, s + i])
            yb.append((Ct[i].abs() * hs[-1]).sum(-1) + (skip * x[b, s + i]).abs())
            out["out"][0][b, s + i], out["out"][1][b, s + i] = ya[-1] * gate[b, s + i], yb[-1] * gate[b, s + i].abs()
        out["ht"][0][n], out["ht"][1][n] = hv[-1], hs[-1]
        if dout is None:
            continue
        g = torch.zeros(ch, N, dtype=x.dtype) if dht is None else dht[n]
        gs = g.abs()
        for i in range(e - s - 1, -1, -1):
            t = s + i
            dy = dout[b, t] * gate[b, t]
            if z is not None:
                out["dz"][0][b, t] = dout[b, t] * ya[i] * _dsilu(z[b, t])
                out["dz"][1][b, t] = (dout[b, t] * _dsilu(z[b, t])).abs() * yb[i] + (dout[b, t] * ya[i]).abs()
            g, gs = Ct[i] * dy[:, None] + g, (Ct[i] * dy[:, None]).abs() + gs
            dx_, dl, xx = delta[b, t] * x[b, t], delta[b, t], x[b, t]
            for k, (gg, hh, hp, m) in enumerate(((g, hv[i + 1], hv[i], lambda q: q),
                                                (gs, hs[i + 1], hs[i], torch.abs))):
                fold = lambda q: q.view(G, ch // G, N).sum(1)  # noqa: E731
                out["dB"][k][b, t] += fold(gg * m(dx_)[:, None])
                out["dC"][k][b, t] += fold(m(dy)[:, None] * hh)
                gB = (gg * m(Bt[i])).sum(-1)
                r = a[i] * gg
                aw = (m(A) * r * hp).sum(-1)
                out["dx"][k][b, t] = m(dl) * gB + m(skip * dy)
                dv = (m(xx) * gB + aw) * dv_dv[b, t]
                out["ddt"][k][b, t] = dv
                out["dbias"][k].add_(dv)
                out["dD"][k].add_(m(dy * xx))
                out["dA"][k].add_(m(dl)[:, None] * r * hp)
                if k == 0:
                    g_next = r
                else:
                    gs = r
            g = g_next
        out["dh0"][0][n], out["dh0"][1][n] = g, gs
    return out


def qk_ref(x, w, cos, sin, pos, eps, pairs, dy=None):
    """One of q, k [B, T, H, K] (double CPU); cos, sin [P, R / 2]; pos [B, T].  -> y, size, dx, size, dw, size."""
    K = x.shape[-1]
    R = 0 if cos is None else 2 * cos.shape[1]
    rs = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    ww = torch.ones(K, dtype=x.dtype) if w is None else w

    def turn(t, c, s, absolute=False):
        lo, hi = (t[..., 0:R:2], t[..., 1:R:2]) if pairs else (t[..., :R // 2], t[..., R // 2:R])
        if absolute:
            a, b = lo * c.abs() + hi * s.abs(), lo * s.abs() + hi * c.abs()
        else:
            a, b = lo * c - hi * s, lo * s + hi * c
        r = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
        return torch.cat([r, t[..., R:]], -1)

    nrm = x * rs * ww
    if R:
        c, s = cos[pos][:, :, None], sin[pos][:, :, None]
        y, ys = turn(nrm, c, s), turn(nrm.abs(), c, s, True)
    else:
        y, ys = nrm, nrm.abs()
    if dy is None:
        return y, ys
    d, dsz = (turn(dy, c, -s), turn(dy.abs(), c, s, True)) if R else (dy, dy.abs())
    e, es = d * ww, dsz * ww.abs()
    dx = rs * (e - x * rs * rs * (e * x).mean(-1, keepdim=True))
    dxs = rs * (es + x.abs() * rs * rs * (es * x.abs()).mean(-1, keepdim=True))
    return y, ys, dx, dxs, (d * x * rs).sum((0, 1, 2)), (dsz * x.abs() * rs).sum((0, 1, 2))
