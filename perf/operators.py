"""What is measured of the operators around the framework's recurrences: the causal short convolution, the selective
state space scan (both over prompts, in training and for single tokens) and the norm of queries and keys with the
position rotation.

``run`` computes them in elementary torch operations in 32 bits, or, where ``own`` is set, through ``tops``.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


def _tops():
    """The framework's package lies one folder below the root."""
    at = os.path.join(os.getcwd(), "pallas-kernel_b200")
    if at not in sys.path:
        sys.path.insert(1, at)
    import tops.modules
    import tops.ops.ssm
    return tops


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # a training step of the value path's convolution of the 2048-wide GLA language model
        {"name": "conv_train", "op": "conv_train", "B": 8, "T": 4096, "D": 2048, "W": 4, "bias": False, "act": "silu",
         "dtype": "bf16"},
        # 23 prompts of uneven length packed for serving, each continuing a carried state
        {"name": "conv_packed", "op": "conv_packed", "T": 9973, "N": 23, "D": 1024, "W": 4, "bias": True, "act": "silu",
         "dtype": "fp16"},
        # one token for each of 256 requests
        {"name": "conv_step", "op": "conv_step", "B": 256, "D": 2048, "W": 4, "bias": True, "act": "silu", "dtype": "bf16"},
        # one token of one request: latency
        {"name": "conv_step_one", "op": "conv_step", "B": 1, "D": 1024, "W": 4, "bias": False, "act": "silu",
         "dtype": "bf16"},
        # a training step of a scan layer twice as wide as the 2048-wide model
        {"name": "scan_train", "op": "scan_train", "B": 4, "T": 2048, "D": 4096, "N": 16, "G": 1, "z": True,
         "dtype": "bf16"},
        # training on short odd rows in full precision, channels in two groups
        {"name": "scan_train_odd", "op": "scan_train", "B": 2, "T": 517, "D": 1000, "N": 8, "G": 2, "z": False,
         "dtype": "fp32"},
        # one long prompt: few rows, the time axis has to be split
        {"name": "scan_prompt", "op": "scan_prompt", "B": 1, "T": 8191, "D": 4096, "N": 16, "G": 1, "z": True,
         "dtype": "bf16"},
        # 19 packed prompts (one empty, one of a single token), each continuing a carried state
        {"name": "scan_packed", "op": "scan_packed", "T": 6007, "N": 16, "S": 19, "D": 2048, "G": 1, "z": True,
         "dtype": "fp16"},
        # one token for each of 256 requests
        {"name": "scan_step", "op": "scan_step", "B": 256, "D": 4096, "N": 16, "G": 1, "z": True, "dtype": "bf16"},
        # one token for two requests: latency
        {"name": "scan_step_two", "op": "scan_step", "B": 2, "D": 2048, "N": 16, "G": 1, "z": True, "dtype": "bf16"},
        # a training step: 16 query heads over 4 key heads, half of each head rotated
        {"name": "qk_train", "op": "qk_train", "B": 8, "T": 4096, "H": 16, "HK": 4, "K": 128, "R": 64, "pairs": False,
         "dtype": "bf16"},
        # one token for each of 256 requests at positions up to 131071, whole heads rotated
        {"name": "qk_step", "op": "qk_step", "B": 256, "T": 1, "H": 16, "HK": 16, "K": 128, "R": 128, "pairs": False,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv_train", "conv_packed", "conv_step", "scan_train", "scan_prompt", "scan_packed", "scan_step",
                     "qk_train", "qk_step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    odd = rng.random() < 0.4
    wide = lambda hi: _log(rng, 64, hi) if odd else 64 * _log(rng, 1, hi // 64)  # noqa: E731
    if op.startswith("conv"):
        c = {"op": op, "D": wide(2048), "W": rng.choice([2, 3, 4, 4, 4]), "bias": rng.random() < 0.5,
             "act": rng.choice(["silu", "silu", "none"]), "dtype": dtype}
        if op == "conv_train":
            c |= {"B": rng.randint(1, 8), "T": _log(rng, 16, 4096)}
        elif op == "conv_packed":
            c |= {"N": _log(rng, 1, 48), "T": _log(rng, 64, 9973)}
        else:
            c |= {"B": _log(rng, 1, 256)}
    elif op.startswith("scan"):
        G = rng.choice([1, 1, 2])
        c = {"op": op, "D": G * (wide(4096) // G), "G": G, "N": rng.choice([4, 8, 11, 16, 16, 16, 32]), "z": rng.random() < 0.7,
             "dtype": dtype}
        most = 4 * 2048 * 4096 * 16 // (c["D"] * c["N"])  # rows, so that no case is larger than the largest listed one
        if op == "scan_train":
            B = rng.randint(1, 4)
            c |= {"B": B, "T": _log(rng, 16, max(17, min(2048, most // B)))}
        elif op == "scan_prompt":
            B = rng.randint(1, 3)
            c |= {"B": B, "T": _log(rng, 64, max(65, min(8191, most // B)))}
        elif op == "scan_packed":
            c |= {"S": _log(rng, 1, 32), "T": _log(rng, 64, max(65, min(6007, most)))}
        else:
            c |= {"B": _log(rng, 1, max(2, min(256, 256 * 4096 * 16 // (c["D"] * c["N"]))))}
    else:
        K = rng.choice([64, 96, 128, 128, 256])
        HK = rng.choice([1, 2, 4, 8])
        c = {"op": op, "K": K, "HK": HK, "H": HK * rng.choice([1, 2, 4]), "R": rng.choice([K, K // 2, 32]),
             "pairs": rng.random() < 0.3, "dtype": dtype}
        c["H"] = min(c["H"], 16)
        most = 8 * 4096 * 20 * 128 // ((c["H"] + HK) * K)
        if op == "qk_train":
            B = rng.randint(1, 8)
            c |= {"B": B, "T": _log(rng, 1, max(2, min(4096, most // B)))}
        else:
            c |= {"B": _log(rng, 1, 256), "T": 1}
    return c


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------


def _cuts(n, total, gen):
    """[n + 1] offsets of n sequences over `total` rows: uneven lengths, from three sequences on one of them empty and
    one of a single token."""
    at = torch.randint(0, total + 1, (n - 1,), generator=gen, device=DEV).sort().values
    cu = torch.cat([at.new_zeros(1), at, at.new_full((1,), total)])
    if n > 2:
        cu[2], cu[3 if n > 3 else 1] = cu[1], (cu[1] + 1 if n > 3 else cu[2])
        cu = cu.cummax(0).values.clamp(max=total)
        cu[-1] = total
    return cu.int()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt_ = DTYPES[case["dtype"]]
    rn = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    ru = lambda lo, hi, *s: torch.rand(*s, generator=gen, device=DEV) * (hi - lo) + lo  # noqa: E731
    op, s = case["op"], {"case": dict(case)}
    if op.startswith("conv"):
        D, W = case["D"], case["W"]
        s["w"] = ru(-W ** -0.5, W ** -0.5, D, W).to(dt_)
        s["b"] = (0.1 * rn(D)).to(dt_) if case["bias"] else None
        if op == "conv_train":
            s["x"], s["dy"] = rn(case["B"], case["T"], D).to(dt_), rn(case["B"], case["T"], D).to(dt_)
        elif op == "conv_packed":
            s["x"] = rn(1, case["T"], D).to(dt_)
            s["state"] = rn(case["N"], D, W - 1).to(dt_)
            s["cu"] = _cuts(case["N"], case["T"], gen)
        else:
            s["x"], s["state"] = rn(case["B"], D).to(dt_), rn(case["B"], D, W - 1).to(dt_)
    elif op.startswith("scan"):
        D, N, G, step = case["D"], case["N"], case["G"], op == "scan_step"
        rows = (case["B"],) if step else (1, case["T"]) if op == "scan_packed" else (case["B"], case["T"])
        # x and z are the halves of one projection, B and C the tails of another, as a layer makes them
        xz = rn(*rows, 2 * D if case["z"] else D).to(dt_)
        s["x"], s["z"] = xz[..., :D], xz[..., D:] if case["z"] else None
        bc = rn(*rows, 2 * G * N).to(dt_)
        s["Bm"], s["Cm"] = bc[..., :G * N].unflatten(-1, (G, N)), bc[..., G * N:].unflatten(-1, (G, N))
        s["dt"] = (0.5 * rn(*rows, D)).to(dt_)
        s["A"] = -torch.arange(1, N + 1, device=DEV, dtype=torch.float32).expand(D, N) * torch.exp(0.1 * rn(D, N))
        s["D"] = 1 + 0.1 * rn(D)
        want = torch.exp(ru(math.log(1e-3), math.log(1e-1), D))  # the step sizes that training starts from
        s["bias"] = want + torch.log(-torch.expm1(-want))
        if op == "scan_train":
            s["dy"] = rn(*rows, D).to(dt_)
        elif op == "scan_packed":
            s["cu"] = _cuts(case["S"], case["T"], gen)
            s["h0"] = 0.5 * rn(case["S"], D, N)
        elif step:
            s["h0"] = 0.5 * rn(case["B"], D, N)
    else:
        B, T, K = case["B"], case["T"], case["K"]
        s["q"], s["k"] = rn(B, T, case["H"], K).to(dt_), rn(B, T, case["HK"], K).to(dt_)
        s["qw"], s["kw"] = 1 + 0.1 * rn(K), 1 + 0.1 * rn(K)
        most = 131072 if op == "qk_step" else max(T, 1)
        angle = torch.arange(most, device=DEV, dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(0, case["R"], 2, device=DEV, dtype=torch.float64) / case["R"]))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["pos"] = None
        if op == "qk_step":
            s["pos"] = torch.randint(0, most, (B, T), generator=gen, device=DEV, dtype=torch.int32)
        else:
            s["dq"], s["dk"] = rn(B, T, case["H"], K).to(dt_), rn(B, T, case["HK"], K).to(dt_)
    leaf = {"conv_train": ("x", "w", "b"), "scan_train": ("x", "dt", "A", "Bm", "Cm", "D", "z", "bias"),
            "qk_train": ("q", "k", "qw", "kw")}.get(op, ())
    for n in leaf:
        if s[n] is not None:
            s[n] = s[n].detach().requires_grad_()
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------


def _silu(p):
    return p / (1 + torch.exp(-p))


def _taps(rows, W, cu, device):
    """For rows of packed sequences: [rows, W] indices of each row's window in cat(rows, N (W - 1) carried columns)."""
    t = torch.arange(rows, device=device)
    n = torch.searchsorted(cu[1:].contiguous(), t.int(), right=True)
    src = t[:, None] - (W - 1) + torch.arange(W, device=device)
    before = src - cu[n].long()[:, None]
    return torch.where(before >= 0, src, rows + (n * (W - 1))[:, None] + (W - 1) + before)


def _conv_plain(s):
    c = s["case"]
    W, dt_ = c["W"], DTYPES[c["dtype"]]
    w, b = s["w"].float(), 0.0 if s["b"] is None else s["b"].float()
    act = _silu if c["act"] == "silu" else (lambda p: p)
    if c["op"] == "conv_step":
        win = torch.cat([s["state"], s["x"][..., None]], -1)
        return act((win.float() * w).sum(-1) + b).to(dt_), win[..., 1:].contiguous()
    if c["op"] == "conv_packed":
        x, cu, N = s["x"][0], s["cu"], c["N"]
        every = torch.cat([x, s["state"].transpose(1, 2).reshape(N * (W - 1), -1)])
        win = every[_taps(x.shape[0], W, cu, x.device)].float()  # [T, W, D]
        y = act((win * w.t()).sum(1) + b).to(dt_)[None]
        back = cu[1:].long()[:, None] - (W - 1) + torch.arange(W - 1, device=x.device)
        before = back - cu[:-1].long()[:, None]
        n = torch.arange(N, device=x.device)[:, None]
        at = torch.where(before >= 0, back, x.shape[0] + n * (W - 1) + (W - 1) + before)
        return y, every[at].transpose(1, 2).contiguous()
    x, T = s["x"].detach(), c["T"]
    pad = torch.nn.functional.pad(x.float(), (0, 0, W - 1, 0))
    win = pad.unfold(1, W, 1)  # [B, T, D, W]
    p = (win * w.detach()).sum(-1) + (b if s["b"] is None else b.detach())
    y, dy = act(p), s["dy"].float()
    if c["act"] == "silu":
        g = 1 / (1 + torch.exp(-p))
        dp = dy * g * (1 + p * (1 - g))
    else:
        dp = dy
    dwin = torch.nn.functional.pad(dp, (0, 0, 0, W - 1)).unfold(1, W, 1)  # dp_{t .. t + W - 1}
    dx = (dwin * w.detach().flip(-1)).sum(-1)
    dw = (win * dp[..., None]).sum((0, 1))
    out = {"y": y.to(dt_), "dx": dx.to(dt_), "dw": dw.to(dt_)}
    if s["b"] is not None:
        out["db"] = dp.sum((0, 1)).to(dt_)
    return out


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _linear_scan(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 1, by doubling: log2(T) passes."""
    k, T = 1, u.shape[1]
    while k < T:
        u = torch.cat([u[:, :k], u[:, k:] + a[:, k:] * u[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return u


def _scan_plain(s):
    c = s["case"]
    dt_, G, N, D = DTYPES[c["dtype"]], c["G"], c["N"], c["D"]
    f = lambda n: None if s.get(n) is None else s[n].detach().float()  # noqa: E731
    x, z, A = f("x"), f("z"), f("A")
    Bm, Cm = (f(n).repeat_interleave(D // G, -2) for n in ("Bm", "Cm"))  # [..., D, N]
    v = f("dt") + f("bias")
    delta = _softplus(v)
    a = torch.exp(delta[..., None] * A)
    u = (delta * x)[..., None] * Bm
    gate = lambda y: y if z is None else y * _silu(z)  # noqa: E731
    if c["op"] == "scan_step":
        h = a * f("h0") + u
        return gate((h * Cm).sum(-1) + f("D") * x).to(dt_), h
    if c["op"] == "scan_packed":
        cu = s["cu"].long()
        used = cu[1:] > cu[:-1]
        first = torch.zeros(c["T"] + 1, device=x.device).index_fill(0, cu[:-1], 1.0)[:-1].bool()
        seq = torch.searchsorted(cu[1:].contiguous(), torch.arange(c["T"], device=x.device), right=True)
        u = u + torch.where(first[None, :, None, None], a * f("h0")[seq][None], 0.0)
        a = torch.where(first[None, :, None, None], 0.0, a)
    h = _linear_scan(a, u)
    y = (h * Cm).sum(-1) + f("D") * x
    if c["op"] == "scan_packed":
        ht = torch.where(used[:, None, None], h[0, (cu[1:] - 1).clamp(min=0)], f("h0"))
        return gate(y).to(dt_), ht
    if c["op"] == "scan_prompt":
        return gate(y).to(dt_), h[:, -1].clone()
    out = gate(y).to(dt_)
    dout = s["dy"].float()
    if z is not None:
        sg = 1 / (1 + torch.exp(-z))
        dz, dy = dout * y * sg * (1 + z * (1 - sg)), dout * z * sg
    else:
        dz, dy = None, dout
    # g_t = C_t dy_t + a_{t+1} g_{t+1}: the same scan from the end
    nxt = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _linear_scan(nxt.flip(1), (Cm * dy[..., None]).flip(1)).flip(1)
    del nxt
    dCm = (h * dy[..., None]).unflatten(2, (G, D // G)).sum(3)
    dBm = (g * (delta * x)[..., None]).unflatten(2, (G, D // G)).sum(3)
    gB = (g * Bm).sum(-1)
    r = a * g * torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    dA = (r * delta[..., None]).sum((0, 1))
    dv = (x * gB + (r * A).sum(-1)) / (1 + torch.exp(-v))
    res = {"out": out, "dx": (delta * gB + f("D") * dy).to(dt_), "ddt": dv.to(dt_), "dA": dA, "dB": dBm.to(dt_),
           "dC": dCm.to(dt_), "dD": (dy * x).sum((0, 1)), "dbias": dv.sum((0, 1))}
    if dz is not None:
        res["dz"] = dz.to(dt_)
    return res


def _rotate(x, cos, sin, pairs):
    a, b = (x[..., 0::2], x[..., 1::2]) if pairs else x.chunk(2, -1)
    u, v = a * cos - b * sin, a * sin + b * cos
    return torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1)


def _qk_plain(s):
    c = s["case"]
    dt_, R, eps = DTYPES[c["dtype"]], c["R"], 1e-6
    pos = s["pos"].long() if s["pos"] is not None else torch.arange(c["T"], device=DEV)[None].expand(c["B"], -1)
    cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    out = {}
    for n in ("q", "k"):
        x, w = s[n].detach().float(), s[n + "w"].detach()
        rs = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        y = x * rs * w
        out[n] = torch.cat([_rotate(y[..., :R], cos, sin, c["pairs"]), y[..., R:]], -1).to(dt_)
        if c["op"] == "qk_train":
            d = s["d" + n].float()
            d = torch.cat([_rotate(d[..., :R], cos, -sin, c["pairs"]), d[..., R:]], -1)
            out["d" + n + "w"] = (d * x * rs).sum((0, 1, 2))
            e = d * w
            out["d" + n] = (rs * (e - x * rs * rs * (e * x).mean(-1, keepdim=True))).to(dt_)
    return out


# ---------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------


def _run_own(s):
    c, t = s["case"], _tops()
    op = c["op"]
    act = None if c.get("act") == "none" else c.get("act")
    if op == "conv_step":
        return t.modules.causal_conv1d_step(s["x"], s["state"], s["w"], s["b"], act)
    if op == "conv_packed":
        return t.modules.causal_conv1d(s["x"], s["w"], s["b"], act, initial_state=s["state"], output_final_state=True,
                                       cu_seqlens=s["cu"])
    if op == "conv_train":
        y, _ = t.modules.causal_conv1d(s["x"], s["w"], s["b"], act)
        names = [n for n in ("x", "w", "b") if s[n] is not None]
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
        return {"y": y.detach(), **{"d" + n: g for n, g in zip(names, grads)}}
    if op == "scan_step":
        return t.ops.ssm.selective_scan_step(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], s["h0"], D=s["D"], z=s["z"],
                                             dt_bias=s["bias"], dt_softplus=True)
    if op.startswith("scan"):
        y, ht = t.ops.ssm.selective_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s["z"], dt_bias=s["bias"],
                                         dt_softplus=True, initial_state=s.get("h0"),
                                         output_final_state=op != "scan_train", cu_seqlens=s.get("cu"))
        if op != "scan_train":
            return y, ht
        names = [n for n in ("x", "dt", "A", "Bm", "Cm", "D", "z", "bias") if s[n] is not None]
        grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
        called = {"Bm": "dB", "Cm": "dC"}
        return {"out": y.detach(), **{called.get(n, "d" + n): g for n, g in zip(names, grads)}}
    q, k = t.modules.qk_norm_rotary(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], positions=s["pos"], eps=1e-6,
                                    interleaved=c["pairs"])
    if op == "qk_step":
        return {"q": q, "k": k}
    grads = torch.autograd.grad((q, k), [s[n] for n in ("q", "k", "qw", "kw")], (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), **dict(zip(("dq", "dk", "dqw", "dkw"), grads))}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    with torch.no_grad():
        return (_conv_plain if op.startswith("conv") else _scan_plain if op.startswith("scan") else _qk_plain)(state)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------


def work(case):
    e = DTYPES[case["dtype"]].itemsize
    op = case["op"]
    if op.startswith("conv"):
        D, W = case["D"], case["W"]
        if op == "conv_step":
            n = case["B"] * D
            return {"bytes": n * e * (2 + 2 * (W - 1)) + D * W * e, "flops": n * (2 * W + 4)}
        n = case["T"] * D * case.get("B", 1)
        if op == "conv_packed":
            return {"bytes": n * e * 2 + 2 * case["N"] * D * (W - 1) * e, "flops": n * (2 * W + 4)}
        return {"bytes": n * e * 4 + 2 * D * W * e, "flops": n * (6 * W + 12)}
    if op.startswith("scan"):
        D, N, G = case["D"], case["N"], case["G"]
        rows = case["B"] if op == "scan_step" else case["T"] * case.get("B", 1)
        n = rows * D
        wide = 3 + bool(case["z"])  # x, dt, out and z
        if op == "scan_step":
            return {"bytes": n * e * wide + 2 * rows * G * N * e + 8 * n * N + 4 * D * N, "flops": n * (7 * N + 12)}
        if op == "scan_train":
            return {"bytes": n * e * (wide + 3 + bool(case["z"])) + 4 * rows * G * N * e + 8 * D * N,
                    "flops": n * (22 * N + 30)}
        states = 4 * D * N * (2 * case["S"] if op == "scan_packed" else case["B"])
        return {"bytes": n * e * wide + 2 * rows * G * N * e + states, "flops": n * (7 * N + 12)}
    n = case["B"] * case["T"] * (case["H"] + case["HK"]) * case["K"]
    if op == "qk_step":
        return {"bytes": 2 * n * e + case["B"] * case["T"] * case["R"] * 4, "flops": 8 * n}
    return {"bytes": 4 * n * e, "flops": 24 * n}


# ---------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op, L = case["op"], {}
    for n, v in s.items():
        if torch.is_tensor(v) and v.is_floating_point():
            L[n] = v.detach().double().requires_grad_(v.requires_grad)
    cu = s["cu"].tolist() if "cu" in s else None
    if op.startswith("conv"):
        W, w = case["W"], L["w"]
        act = torch.nn.functional.silu if case["act"] == "silu" else (lambda p: p)

        def conv(x, old):  # x [B, T, D], old [B, D, W - 1]
            rows = torch.cat([old.transpose(1, 2), x], 1)
            p = sum(rows[:, j:j + x.shape[1]] * w[:, j] for j in range(W))
            return act(p + L["b"] if "b" in L else p), rows[:, rows.shape[1] - (W - 1):].transpose(1, 2)

        if op == "conv_step":
            y, new = conv(L["x"][:, None], L["state"])
            return y[:, 0], new
        if op == "conv_packed":
            got = [conv(L["x"][:, i:j], L["state"][n:n + 1]) for n, (i, j) in enumerate(zip(cu, cu[1:]))]
            return torch.cat([g[0] for g in got], 1), torch.cat([g[1] for g in got])
        y, _ = conv(L["x"], L["x"].new_zeros(case["B"], case["D"], W - 1))
        names = [n for n in ("x", "w", "b") if n in L]
        grads = torch.autograd.grad(y, [L[n] for n in names], L["dy"])
        return {"y": y.detach(), **{"d" + n: g for n, g in zip(names, grads)}}
    if op.startswith("scan"):
        rep = case["D"] // case["G"]
        delta = torch.nn.functional.softplus(L["dt"] + L["bias"])

        def step(h, x, d, Bt, Ct):  # one token of every row
            h = torch.exp(d[..., None] * L["A"]) * h + (d * x)[..., None] * Bt.repeat_interleave(rep, -2)
            return h, (h * Ct.repeat_interleave(rep, -2)).sum(-1) + L["D"] * x

        gate = lambda y, z: y * torch.nn.functional.silu(z)  # noqa: E731
        if op == "scan_step":
            h, y = step(L["h0"], L["x"], delta, L["Bm"], L["Cm"])
            return gate(y, L["z"]) if "z" in L else y, h

        def sweep(h, i, j):
            ys = []
            for t in range(i, j):
                h, y = step(h, L["x"][:, t], delta[:, t], L["Bm"][:, t], L["Cm"][:, t])
                ys.append(y)
            return (torch.stack(ys, 1) if ys else L["x"][:, :0]), h

        if op == "scan_packed":
            got = [sweep(L["h0"][n:n + 1], i, j) for n, (i, j) in enumerate(zip(cu, cu[1:]))]
            y, ht = torch.cat([g[0] for g in got], 1), torch.cat([g[1] for g in got])
        else:
            y, ht = sweep(L["x"].new_zeros(case["B"], case["D"], case["N"]), 0, case["T"])
        if "z" in L:
            y = gate(y, L["z"])
        if op != "scan_train":
            return y, ht
        names = [n for n in ("x", "dt", "A", "Bm", "Cm", "D", "z", "bias") if n in L]
        grads = torch.autograd.grad(y, [L[n] for n in names], L["dy"])
        return {"out": y.detach(), **{{"Bm": "dB", "Cm": "dC"}.get(n, "d" + n): g for n, g in zip(names, grads)}}
    R = case["R"]
    pos = s["pos"].double() if s["pos"] is not None else torch.arange(case["T"], device=DEV).double().expand(case["B"], -1)
    freq = torch.exp(-math.log(10000.0) * torch.arange(0, R, 2, device=DEV).double() / R)
    turn = torch.polar(torch.ones_like(pos[..., None] * freq), pos[..., None] * freq)[:, :, None]

    def one(x, w):
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        r = y[..., :R].unflatten(-1, (R // 2, 2) if case["pairs"] else (2, R // 2))
        r = r if case["pairs"] else r.transpose(-1, -2)
        r = torch.view_as_real(torch.view_as_complex(r.contiguous()) * turn)
        r = (r if case["pairs"] else r.transpose(-1, -2)).flatten(-2)
        return torch.cat([r, y[..., R:]], -1)

    q, k = one(L["q"], L["qw"]), one(L["k"], L["kw"])
    if op == "qk_step":
        return {"q": q, "k": k}
    grads = torch.autograd.grad((q, k), [L[n] for n in ("q", "k", "qw", "kw")], (L["dq"], L["dk"]))
    return {"q": q.detach(), "k": k.detach(), **dict(zip(("dq", "dk", "dqw", "dkw"), grads))}
