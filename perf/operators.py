"""The per-channel gated recurrence and the two norms of a recurrent layer, as measurable cases.

Three operators, each in its plain form (elementary torch operations in 32 bits) and through this
package's entry points (``own = True``):

``scan`` / ``scan_train`` / ``step``
    h_t = g_t h_{t-1} + beta_t x_t per channel, with the gates of the package's other recurrences:
    g = exp(-exp(A_log) softplus(a + dt_bias)), beta = sigmoid(b); packed sequences, one state row each.
``add_norm`` / ``add_norm_train``
    r = x + residual; y = r / sqrt(mean(r^2) + eps) * weight, in the inputs' type or in e4m3 with one
    scale per row or per 128 channels (scale = amax / 448).
``gated_norm`` / ``gated_norm_train``
    y = x / sqrt(mean(x^2) + eps) * weight * silu(z) over each head of a [tokens, heads, 128] output,
    in the inputs' type or in e4m3 with one scale per head.

The ``_train`` forms are a forward and a backward pass.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6
AMAX_MIN = 1e-12  # the least amax a scale is made from: an all-zero row keeps a finite scale
FP8_MAX = 448.0
GROUP = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases --
def _scan(op, seqs, lo, hi, channels, dtype="bf16", state=True, fused=False, lseed=0):
    return {"op": op, "seqs": seqs, "lo": lo, "hi": hi, "channels": channels, "dtype": dtype, "state": state,
            "fused": fused, "lseed": lseed}


def _norm(op, rows, width, dtype="bf16", quant="", heads=0):
    return {"op": op, "rows": rows, "width": width, "dtype": dtype, "quant": quant, "heads": heads}


def listed():
    return [
        # a short prompt appended to a conversation: one sequence, latency counts
        {"name": "scan_append_64", **_scan("scan", 1, 64, 64, 1024)},
        # a batch of ragged prompts; x, a and b are column blocks of one projection's output
        {"name": "scan_ragged_32", **_scan("scan", 32, 64, 2048, 2048, fused=True)},
        # one long document
        {"name": "scan_long_40000", **_scan("scan", 1, 40000, 40000, 1024)},
        # a training step on packed 4096-token sequences
        {"name": "scan_train_8x4096", **_scan("scan_train", 8, 4096, 4096, 1024, state=False)},
        # training in 32 bits on short and empty sequences, an odd channel count
        {"name": "scan_train_odd", **_scan("scan_train", 37, 0, 300, 1001, dtype="fp32")},
        # one decode step of a small and of a large batch
        {"name": "step_8", **_scan("step", 8, 1, 1, 1024)},
        {"name": "step_256", **_scan("step", 256, 1, 1, 4096)},
        # the norm before a layer's projections: a decode step with e4m3 in groups of 128
        {"name": "add_norm_8_group", **_norm("add_norm", 8, 2048, quant="group")},
        # the same over a large prefill, one scale per token
        {"name": "add_norm_65536_row", **_norm("add_norm", 65536, 4096, quant="row")},
        # a training step's norm, an odd number of rows, in fp16
        {"name": "add_norm_train_8191", **_norm("add_norm_train", 8191, 2048, dtype="fp16")},
        # the recurrence's output of a 256-sequence decode step, to e4m3 for the output projection
        {"name": "gated_norm_256_group", **_norm("gated_norm", 256, 128, quant="group", heads=8)},
        # the same norm in training, 32 heads
        {"name": "gated_norm_train_32768", **_norm("gated_norm_train", 32768, 128, heads=32)},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "scan_train", "step", "add_norm", "add_norm_train", "gated_norm", "gated_norm_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "step":
        return _scan(op, _log_int(rng, 1, 1024), 1, 1, rng.choice([8 * _log_int(rng, 32, 512), _log_int(rng, 250, 4100)]),
                     dtype, lseed=rng.randrange(1000))
    if op in ("scan", "scan_train"):
        channels = rng.choice([64 * _log_int(rng, 4, 64), 8 * _log_int(rng, 32, 512), _log_int(rng, 250, 4100)])
        most = min(40000, ((10 if op == "scan_train" else 20) << 20) // channels)  # packed tokens, twice that at most
        tokens = _log_int(rng, 32, most)
        seqs = _log_int(rng, 1, max(1, min(300, tokens // 4)))
        mean = max(1, tokens // seqs)
        lo = rng.choice([0, 1, mean // 2, mean])
        return _scan(op, seqs, lo, 2 * mean - lo, channels, dtype, state=rng.random() < 0.7,
                     fused=rng.random() < 0.4, lseed=rng.randrange(1000))
    if op in ("add_norm", "add_norm_train"):
        width = rng.choice([128 * _log_int(rng, 4, 64), 8 * _log_int(rng, 64, 1024), _log_int(rng, 500, 8200)])
        rows = _log_int(rng, 1, min(65536, (160 << 20) // width))
        quant = "" if op == "add_norm_train" else rng.choice(["", "row", "group" if width % GROUP == 0 else "row"])
        return _norm(op, rows, width, dtype, quant)
    heads = rng.choice([4, 8, 16, 32, rng.randrange(1, 33)])
    rows = _log_int(rng, 1, min(65536, (128 << 20) // (heads * 128)))
    return _norm(op, rows, 128, dtype, "" if op == "gated_norm_train" else rng.choice(["", "group"]), heads)


def _lengths(case):
    gen = torch.Generator().manual_seed(case["lseed"])
    return torch.randint(case["lo"], case["hi"] + 1, (case["seqs"],), generator=gen).tolist()


def work(case):
    es = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] in ("scan", "scan_train", "step"):
        C, N = case["channels"], case["seqs"]
        T = sum(_lengths(case)) if case["op"] != "step" else N
        states = (2 if case["state"] or case["op"] == "step" else 1) * N * C * 4
        if case["op"] == "scan_train":  # x, a, b, dy read; y, dx, da, db written; the state's gradients too
            return {"bytes": 8 * T * C * es + 2 * states + 16 * C, "flops": 60 * T * C}
        return {"bytes": 4 * T * C * es + states + 8 * C, "flops": 20 * T * C}
    n = case["rows"] * case["width"] * max(1, case["heads"])
    out = n if case["quant"] else n * es
    scales = 4 * (0 if not case["quant"] else case["rows"] if case["quant"] == "row" else n // GROUP)
    w = 4 * case["width"]
    return {
        "add_norm": {"bytes": 3 * n * es + out + scales + w, "flops": 6 * n},
        # x, residual, dy, dr read; r, y, dx written
        "add_norm_train": {"bytes": 7 * n * es + 2 * w, "flops": 18 * n},
        "gated_norm": {"bytes": 2 * n * es + out + scales + w, "flops": 12 * n},
        # x, z, dy read; y, dx, dz written
        "gated_norm_train": {"bytes": 6 * n * es + 2 * w, "flops": 36 * n},
    }[case["op"]]


# ----------------------------------------------------------------- inputs --
def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=dt, scale=1.0):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).mul_(scale).to(dtype)

    def uniform(n, lo, hi):
        return torch.rand(n, generator=gen, device=dev) * (hi - lo) + lo

    s = {"case": case}
    if case["op"] in ("scan", "scan_train", "step"):
        C, N = case["channels"], case["seqs"]
        lens = _lengths(case) if case["op"] != "step" else [1] * N
        T = sum(lens)
        if case["fused"]:  # column blocks of one [T, 3C] projection
            p = normal(T, 3 * C)
            s["x"], s["a"], s["b"] = p[:, :C], p[:, C:2 * C], p[:, 2 * C:]
        else:
            s["x"], s["a"], s["b"] = normal(T, C), normal(T, C), normal(T, C)
        # decay rates 1 .. 16 and time steps 1e-3 .. 1e-1, log-uniform: memories of one to a thousand tokens
        s["A_log"] = torch.log(uniform(C, 1.0, 16.0))
        step = torch.exp(uniform(C, math.log(1e-3), math.log(1e-1)))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))  # softplus(dt_bias) = step
        s["state"] = normal(N, C, dtype=torch.float32, scale=0.5) if case["state"] else None
        s["lens"], s["max_len"] = lens, max(lens, default=0)
        cu = np.concatenate([[0], np.cumsum(np.asarray(lens, dtype=np.int64))])
        s["cu"] = torch.from_numpy(cu).to(dev)
        if case["op"] == "scan_train":
            s["dy"] = normal(T, C)
            s["dns"] = normal(N, C, dtype=torch.float32) if case["state"] else None
        return s
    shape = (case["rows"], case["heads"], case["width"]) if case["heads"] else (case["rows"], case["width"])
    s["x"] = normal(*shape)
    s["weight"] = 1.0 + normal(case["width"], dtype=torch.float32, scale=0.1)
    if case["heads"]:
        s["z"] = normal(*shape)
    else:
        s["residual"] = normal(*shape, scale=2.0)  # the stream is larger than what a layer adds to it
    if case["op"].endswith("_train"):
        s["dy"] = normal(*shape)
        if not case["heads"]:
            s["dr"] = normal(*shape)
    return s


# ------------------------------------------------------------------- runs --
def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _gates32(s):
    z = s["a"].float() + s["dt_bias"]
    softplus = torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs()))
    log_g = -torch.exp(s["A_log"]) * softplus
    return z, log_g, torch.exp(log_g), 1 / (1 + torch.exp(-s["b"].float()))


def _doubling(A, H, most, back):
    """Every row t of H plus the rows it reaches through the decays A, in log2(most) steps."""
    A, H = A.clone(), H.clone()
    d = 1
    while d < most:
        if back:
            H[:-d] += A[:-d] * H[d:]
            A[:-d] = A[:-d] * A[d:]
        else:
            H[d:] += A[d:] * H[:-d]
            A[d:] = A[d:] * A[:-d]
        d *= 2
    return H


def _bounds(s):
    first, last = s["cu"][:-1], s["cu"][1:] - 1
    some = last >= first
    return first[some], last[some], some


def _plain_scan(s):
    first, last, some = _bounds(s)
    _, _, g, beta = _gates32(s)
    A, H = g.clone(), beta * s["x"].float()
    zero = torch.zeros(len(s["lens"]), H.shape[1], device=H.device)
    start = s["state"] if s["state"] is not None else zero
    H[first] += g[first] * start[some]
    A[first] = 0
    h = _doubling(A, H, s["max_len"], False)
    new_state = start.clone()
    new_state[some] = h[last]
    return h, new_state, start


def _plain_scan_forward(s):
    h, new_state, _ = _plain_scan(s)
    return {"y": h.to(s["x"].dtype), "new_state": new_state}


def _plain_scan_train(s):
    h, new_state, start = _plain_scan(s)
    first, last, some = _bounds(s)
    z, log_g, g, beta = _gates32(s)
    x, dt = s["x"].float(), s["x"].dtype
    A = torch.zeros_like(g)
    A[:-1] = g[1:]
    A[last] = 0
    G = s["dy"].float().clone()
    dns = s["dns"] if s["dns"] is not None else torch.zeros_like(new_state)
    G[last] += dns[some]
    G = _doubling(A, G, s["max_len"], True)
    before = torch.zeros_like(h)
    before[1:] = h[:-1]
    before[first] = start[some]
    d_log_g = G * before * g
    da = d_log_g * -torch.exp(s["A_log"]) / (1 + torch.exp(-z))
    out = {"y": h.to(dt), "new_state": new_state, "dx": (G * beta).to(dt), "da": da.to(dt),
           "db": (G * x * beta * (1 - beta)).to(dt),
           "dA_log": (d_log_g * log_g).double().sum(0).float(), "ddt_bias": da.double().sum(0).float()}
    if s["state"] is not None:
        out["dstate"] = dns.clone()
        out["dstate"][some] = g[first] * G[first]
    return out


def _plain_step(s):
    _, _, g, beta = _gates32(s)
    h = g * s["state"] + beta * s["x"].float()
    return {"y": h.to(s["x"].dtype), "new_state": h}


def _quantised(y, quant):
    if not quant:
        return None
    rows = y if quant == "row" else y.reshape(*y.shape[:-1], -1, GROUP)
    scale = rows.abs().amax(-1).clamp(min=AMAX_MIN) / FP8_MAX
    q = (rows / scale[..., None]).clamp(-FP8_MAX, FP8_MAX).reshape(y.shape).to(torch.float8_e4m3fn)
    return {"q": q, "scale": scale.reshape(scale.shape[0], -1)}


def _rstd32(r):
    return torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)


def _plain_add_norm(s):
    r = s["x"].float() + s["residual"].float()
    y = r * _rstd32(r) * s["weight"]
    return {"r": r.to(s["x"].dtype), **(_quantised(y, s["case"]["quant"]) or {"y": y.to(s["x"].dtype)})}


def _plain_add_norm_train(s):
    out = _plain_add_norm(s)
    r, dy = out["r"].float(), s["dy"].float()
    rstd = _rstd32(r)
    n = r * rstd
    wdy = dy * s["weight"]
    dr = s["dr"].float() + rstd * (wdy - n * (wdy * n).mean(-1, keepdim=True))
    return {**out, "dx": dr.to(s["x"].dtype), "dweight": (dy * n).double().sum(0).float()}


def _plain_gated_norm(s):
    x, z = s["x"].float(), s["z"].float()
    y = x * _rstd32(x) * s["weight"] * (z / (1 + torch.exp(-z)))
    return _quantised(y, s["case"]["quant"]) or {"y": y.to(s["x"].dtype)}


def _plain_gated_norm_train(s):
    x, z, dy = s["x"].float(), s["z"].float(), s["dy"].float()
    sig = 1 / (1 + torch.exp(-z))
    rstd = _rstd32(x)
    n = x * rstd
    wdy = dy * s["weight"] * (z * sig)
    dx = rstd * (wdy - n * (wdy * n).mean(-1, keepdim=True))
    dz = dy * n * s["weight"] * (sig * (1 + z * (1 - sig)))
    return {**_plain_gated_norm(s), "dx": dx.to(s["x"].dtype), "dz": dz.to(s["x"].dtype),
            "dweight": (dy * n * (z * sig)).double().sum((0, 1)).float()}


_plain = {"scan": _plain_scan_forward, "scan_train": _plain_scan_train, "step": _plain_step, "add_norm": _plain_add_norm,
          "add_norm_train": _plain_add_norm_train, "gated_norm": _plain_gated_norm, "gated_norm_train": _plain_gated_norm_train}


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _own_scan(s):
    y, ns = _package().recurrence.launch_scan(s["x"], s["A_log"], s["a"], s["dt_bias"], s["b"], s["cu"], s["state"])
    return {"y": y, "new_state": ns}


def _own_scan_train(s):
    rec = _package().recurrence
    gates = (s["x"], s["A_log"], s["a"], s["dt_bias"], s["b"], s["cu"])
    ckpt = rec.empty_checkpoints(s["x"])
    y, ns = rec.launch_scan(*gates, s["state"], checkpoints=ckpt)
    dx, da, db, dA_log, ddt_bias, dstate = rec.launch_scan_backward(s["dy"], *gates, s["state"], ckpt, d_new_state=s["dns"])
    out = {"y": y, "new_state": ns, "dx": dx, "da": da, "db": db, "dA_log": dA_log, "ddt_bias": ddt_bias}
    if s["state"] is not None:
        out["dstate"] = dstate
    return out


def _own_step(s):
    y, ns = _package().recurrence.launch_step(s["x"], s["A_log"], s["a"], s["dt_bias"], s["b"], s["state"])
    return {"y": y, "new_state": ns}


def _own_add_norm(s):
    quant = s["case"]["quant"] or None
    got = _package().norm.launch_add_norm(s["x"], s["residual"], s["weight"], EPS, quant=quant)
    return {"r": got[1], "q": got[0], "scale": got[2]} if quant else {"r": got[1], "y": got[0]}


def _own_add_norm_train(s):
    norm = _package().norm
    y, r = norm.launch_add_norm(s["x"], s["residual"], s["weight"], EPS)
    dx, dw = norm.launch_add_norm_backward(s["dy"], r, s["weight"], EPS, d_new_residual=s["dr"])
    return {"r": r, "y": y, "dx": dx, "dweight": dw}


def _own_gated_norm(s):
    got = _package().norm.launch_gated_norm(s["x"], s["z"], s["weight"], EPS, quant=bool(s["case"]["quant"]))
    return {"q": got[0], "scale": got[1]} if s["case"]["quant"] else {"y": got}


def _own_gated_norm_train(s):
    norm = _package().norm
    y = norm.launch_gated_norm(s["x"], s["z"], s["weight"], EPS)
    dx, dz, dw = norm.launch_gated_norm_backward(s["dy"], s["x"], s["z"], s["weight"], EPS)
    return {"y": y, "dx": dx, "dz": dz, "dweight": dw}


_own = {"scan": _own_scan, "scan_train": _own_scan_train, "step": _own_step, "add_norm": _own_add_norm,
        "add_norm_train": _own_add_norm_train, "gated_norm": _own_gated_norm, "gated_norm_train": _own_gated_norm_train}


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_scan(s) if "A_log" in s else _exact_norm(s)


def _exact_scan(s):
    """Token by token over the sequences side by side, in 64 bits."""
    op, lens = s["case"]["op"], s["lens"]
    x, a, b = (s[k].double() for k in ("x", "a", "b"))
    dev, (T, C), N, L = x.device, x.shape, len(lens), s["max_len"]
    rate = torch.exp(s["A_log"].double())
    zpre = a + s["dt_bias"].double()
    soft = torch.logaddexp(zpre, torch.zeros_like(zpre))
    g, beta = torch.exp(-rate * soft), torch.sigmoid(b)
    n_of = torch.repeat_interleave(torch.arange(N, device=dev), torch.tensor(lens, device=dev))
    t_of = torch.arange(T, device=dev) - s["cu"][:-1][n_of]
    decay, drive = (torch.zeros(L, N, C, dtype=torch.float64, device=dev) for _ in range(2))
    decay += 1  # past a sequence's end the state stays
    decay[t_of, n_of], drive[t_of, n_of] = g, beta * x
    h0 = s["state"].double() if s["state"] is not None else torch.zeros(N, C, dtype=torch.float64, device=dev)
    h, h_before, h_after = h0.clone(), torch.empty_like(drive), torch.empty_like(drive)
    for t in range(L):
        h_before[t] = h
        h = torch.addcmul(drive[t], decay[t], h)
        h_after[t] = h
    y = h_after[t_of, n_of]
    if op != "scan_train":
        return {"y": y, "new_state": h}
    incoming = torch.zeros_like(drive)
    incoming[t_of, n_of] = s["dy"].double()
    e = s["dns"].double() if s["dns"] is not None else torch.zeros_like(h0)
    total = torch.empty_like(drive)
    for t in reversed(range(L)):
        total[t] = incoming[t] + e
        e = decay[t] * total[t]
    # past a sequence's end `incoming` is zero and `decay` one, so e passes through unchanged
    G, prev = total[t_of, n_of], h_before[t_of, n_of]
    dlog = G * prev * g
    da = -dlog * rate * torch.sigmoid(zpre)
    out = {"y": y, "new_state": h, "dx": G * beta, "da": da, "db": G * x * torch.sigmoid(b) * torch.sigmoid(-b),
           "dA_log": (-dlog * rate * soft).sum(0), "ddt_bias": da.sum(0)}
    if s["state"] is not None:
        out["dstate"] = e
    return out


def _exact_norm(s):
    case, w = s["case"], s["weight"].double()
    x = s["x"].double()
    if case["heads"]:
        r, gate = x, s["z"].double() * torch.sigmoid(s["z"].double())
    else:
        r, gate = x + s["residual"].double(), None
    rms = torch.sqrt((r ** 2).mean(-1, keepdim=True) + EPS)
    y = r / rms * w if gate is None else r / rms * w * gate
    out = {} if gate is not None else {"r": r}
    if case["quant"]:
        # the e4m3 codes go with a scale that is itself rounded: what they are held to is y over the exact scale
        per = y if case["quant"] == "row" else y.unflatten(-1, (-1, GROUP))
        scale = per.abs().amax(-1).clamp(min=AMAX_MIN) / FP8_MAX
        out["q"] = (per / scale.unsqueeze(-1)).reshape(y.shape)
        out["scale"] = scale.reshape(scale.shape[0], -1)
    else:
        out["y"] = y
    if not case["op"].endswith("_train"):
        return out
    dy = s["dy"].double()
    if gate is None:  # the backward pass starts from the stored, rounded sum
        r = (s["x"].float() + s["residual"].float()).to(s["x"].dtype).double()
        rms = torch.sqrt((r ** 2).mean(-1, keepdim=True) + EPS)
    up = dy * w if gate is None else dy * w * gate
    K = r.shape[-1]
    dr = up / rms - r * (up * r).sum(-1, keepdim=True) / (K * rms ** 3)
    if gate is None:
        out["dx"] = dr + s["dr"].double()
        out["dweight"] = (dy * r / rms).sum(0)
    else:
        sig = torch.sigmoid(s["z"].double())
        out["dx"] = dr
        out["dz"] = dy * r / rms * w * (sig + gate * (1 - sig))
        out["dweight"] = (dy * r / rms * gate).sum((0, 1))
    return out
