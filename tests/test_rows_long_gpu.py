"""The row operators where their inner loops run long: rings that wrap, units and strips of many rows, several passes of a
grid, time segments with every number of states, groups and boundaries."""
from __future__ import annotations

import pytest
import torch

from _rows_ref import close, conv_ref, qk_ref, scan_ref
from test_ssm_scan_gpu import NAMES, _call, _check, _dbl, _mk, _roundings

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# -- selective scan ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
@pytest.mark.parametrize("ch,N,G", [(20, 20, 1), (24, 32, 2), (12, 64, 1), (10, 17, 2)])
@pytest.mark.parametrize("cu", [[0, 0, 9, 9, 10, 12, 15, 130], [0, 5, 5, 300, 301, 333], [0, 16, 32, 33, 64]])
def test_scan_packed_with_many_states(dt, ch, N, G, cu):
    """Eight and sixteen lanes a channel over packed rows, in one segment and in several (from 128 rows)."""
    S = len(cu) - 1
    t, dout, dht = _mk(41, 1, cu[-1], ch, N, G, DT[dt], S)
    _check(t, dout, dht, True, cu)
    t["h0"] = None
    _check(t, dout, dht, True, cu, torch.tensor(cu, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
@pytest.mark.parametrize("T,ch,N,G,B", [(700, 12, 32, 1, 1), (331, 10, 64, 2, 2), (500, 24, 20, 3, 1), (613, 32, 16, 2, 2),
                                        (450, 14, 6, 2, 1)])
def test_scan_segments_with_every_number_of_states(dt, T, ch, N, G, B):
    """So few channels that the rows are split; the last segment ends inside a tile."""
    _check(*_mk(42, B, T, ch, N, G, DT[dt], B), True, None)


def test_scan_rows_behind_the_last_sequence_in_segments():
    """A sequence over several segments, then rows of none: what they hold reaches nothing."""
    cu, T = [0, 400, 400, 433], 700
    t, dout, dht = _mk(43, 1, T, 12, 32, 1, torch.float32, 3)
    for k in ("x", "dt", "B", "C", "z"):
        t[k][:, 433:] = float("nan")
    y, _, g = _check(t, dout, dht, True, cu, torch.tensor(cu, device="cuda"), rows=433)
    for v in (y, g["x"], g["dt"], g["z"], g["B"], g["C"]):
        assert not v[:, 433:].any()


def test_scan_far_states_of_varied_steps():
    """Small steps that differ from row to row, so that what the exponentials are off by on average adds up over a
    state's memory while their roundings do not."""
    g = torch.Generator().manual_seed(47)
    T, ch, N = 4096, 32, 16
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": rn(1, T, ch), "dt": -6.9 + rn(1, T, ch) / 2, "B": rn(1, T, 1, N), "C": rn(1, T, 1, N), "z": None,
         "A": -torch.arange(1, N + 1.0).expand(ch, N).contiguous(), "D": None, "bias": None, "h0": None}
    dout = rn(1, T, ch)
    r = scan_ref(*(_dbl(t[k]) for k in NAMES), True, None, _dbl(dout), None)
    c = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    y, ht = _call(c, True, None)
    names = ("x", "dt", "A", "B", "C")
    got = dict(zip(names, torch.autograd.grad(y, [c[k] for k in names], dout.cuda())))
    # A state that forgets within M rows weighs an error of k rows back by exp(-k / M): errors of one sign e a row come
    # to e M / sqrt(2), rounded ones of 2^-24 a row to 2^-24 sqrt(M / 2).  M = 1000 / n for A = -n; outputs mix all n
    # and their smallest M, 1000, bounds them: 2e-9 * 707 + 2^-24 * 22, and what the rounded steps add.
    for name, v, want in (("out", y, r["out"][0]), ("ht", ht, r["ht"][0]), *((f"d{k}", got[k], r[f"d{k}"][0]) for k in names)):
        rel = ((v.double().cpu() - want).norm() / want.norm()).item()
        assert rel <= 3e-6, f"{name}: {rel:.2e}"
    # A = -5 and below: M <= 200, 5e-9 * 141 + 2^-24 * 10 = 1.3e-6 and the sums' own roundings (an exponential that is
    # 2e-8 off on average, as the hardware's is there, would give 2.8e-6)
    err, size = (got["A"].double().cpu() - r["dA"][0])[:, 4:].norm(dim=0), r["dA"][0][:, 4:].norm(dim=0)
    assert (err <= 1.5e-6 * size).all(), f"dA: {(err / size).max():.2e}"


# -- norm and rotation ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dt,H,HK,K,R,tokens", [("bf16", 16, 4, 128, 64, 16384), ("fp32", 5, 2, 128, 128, 21003),
                                                ("fp16", 5, 2, 64, 32, 45001), ("bf16", 5, 2, 33, 20, 21003),
                                                ("bf16", 3, 0, 128, 64, 30011), ("fp32", 2, 5, 80, 32, 21003)])
@pytest.mark.parametrize("pairs", [False, True])
def test_qk_norm_long_units(dt, H, HK, K, R, tokens, pairs):
    """Units of more heads than the ring has slots, some with heads of q and of k, and more of them than one pass of the
    backward's grid: every row and both weights' gradients."""
    from tops.modules import qk_norm_rotary, rotary_tables
    g = torch.Generator(device="cuda").manual_seed(44)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    q, k = rn(1, tokens, H, K).to(DT[dt]), rn(1, tokens, HK, K).to(DT[dt])
    qw, kw = 1 + rn(K) / 4, 1 + rn(K) / 4
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    cos, sin = rotary_tables(4096, R, device="cuda")
    pos = torch.randint(0, 4096, (1, tokens), generator=g, device="cuda", dtype=torch.int32)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    y = qk_norm_rotary(*leaves, cos, sin, pos, 1e-6, pairs)
    got = torch.autograd.grad(y, leaves, [dq, dk])
    n = 2 * K + 24
    for x, w, out, d, gx, gw, name in ((q, qw, y[0], dq, got[0], got[2], "q"), (k, kw, y[1], dk, got[1], got[3], "k")):
        ref = qk_ref(x.detach().double(), w.detach().double(), cos.double(), sin.double(), pos.long(), 1e-6, pairs, d.double())
        close(name, out, ref[0], ref[1], n)
        close("d" + name, gx, ref[2], ref[3], n)
        # a thread adds up the heads of its units one by one (at most 119 in these cases), then come the groups of a
        # warp, four warps, and the blocks as 19 in a row and 32 of those
        close(f"d{name}w", gw, ref[4], ref[5], n + 256)


# -- short convolution ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dt,D,W", [("bf16", 2048, 4), ("fp16", 2048, 3), ("fp32", 2048, 4), ("bf16", 2047, 4), ("fp32", 1024, 2)])
@pytest.mark.parametrize("packed", [False, True])
def test_conv_long_strips(dt, D, W, packed):
    """Strips of 32 rows forward and more than 64 backward (256 without vectors): rings that wrap, sequences that begin
    and end inside strips, the parameters' gradients over all of them."""
    from tops.modules import causal_conv1d
    T = 20011 * 2048 // D
    g = torch.Generator(device="cuda").manual_seed(45)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    cu = None
    if packed:
        c = torch.randint(0, T + 1, (60,), generator=torch.Generator().manual_seed(46)).tolist()
        cu = sorted([0, 0, 1, 500, 501, 503, 503, T - 2, T - 1, T, *c])
    N = len(cu) - 1 if packed else 1
    x, w, b, st = rn(1, T, D).to(DT[dt]), (rn(D, W) / 2).to(DT[dt]), rn(D).to(DT[dt]), rn(N, D, W - 1).to(DT[dt])
    dy, df = rn(1, T, D).to(DT[dt]), rn(N, D, W - 1).to(DT[dt])
    leaves = [t.requires_grad_() for t in (x, w, b, st)]
    y, fin = causal_conv1d(x, w, b, "silu", st, True, cu)
    got = torch.autograd.grad([y, fin], leaves, [dy, df])
    with torch.device("cuda"):
        r = conv_ref(*(t.detach().double() for t in leaves), 1, cu, dy.double(), df.double())
    close("y", y, *r["y"], 24)
    assert torch.equal(fin.detach().double(), r["final"][0])
    for name, v in zip(("dx", "dw", "db", "dstate"), got):
        # a strip's rows (at most 256) in a row, then the strips as 32 sums of at most 80, and those 32
        rows = (256 if D % 4 else 96) + 80 + 32 if name in ("dw", "db") else 0
        close(name, v, *r[name], 48 + rows)
