"""The per-channel recurrence and the norms in 64 bits, token by token, with
bounds on what an fp32 evaluation may be off by.

``U`` is one unit in the last place of fp32 (2^-23 of the value).  A gate's
error is counted as
  log g: 8 U relative (exp, softplus, the products) and U |z| sigmoid(z) exp(A_log) for the sum z,
  g:     that, and 4 U for the exponential;   beta: 8 U,
so the state's error D (in units of U) obeys, with M the recurrence of |beta x|,
  D_t = g_t D_{t-1} + g_t M_{t-1} (8 |log g| + 4 + exp(A_log) |z| sigmoid(z)) + 8 M_t
whatever the order in which the products are taken, up to the factor 2 that the
tests leave for the re-association of a scan in pieces.
"""
import torch

U = 2.0 ** -23


def half(dtype) -> float:
    """Relative half step of a rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def scan(x, A_log, a, dt_bias, b, lens, state=None, dy=None, dns=None, first=0):
    """Values and error bounds of the packed recurrence and of its gradients."""
    x, a, b = x.double(), a.double(), b.double()
    T, C = x.shape
    N = len(lens)
    rate = A_log.double().exp()
    z = a + dt_bias.double()
    sp = torch.logaddexp(z, torch.zeros_like(z))
    l = -rate * sp
    g, beta, sig = l.exp(), torch.sigmoid(b), torch.sigmoid(z)
    u = beta * x
    gate_err = 8 * l.abs() + 4 + rate * z.abs() * sig
    h0 = torch.zeros(N, C, dtype=torch.float64, device=x.device) if state is None else state.double()
    y, y_err, prev, prev_abs, prev_err = (torch.zeros_like(x) for _ in range(5))
    ns, ns_err = h0.clone(), torch.zeros_like(h0)
    spans, t = [], first
    for n in lens:
        spans.append((t, t + n))
        t += n
    for n, (t0, t1) in enumerate(spans):
        h, M, D = h0[n].clone(), h0[n].abs(), torch.zeros_like(h0[n])
        for t in range(t0, t1):
            prev[t], prev_abs[t], prev_err[t] = h, M, D
            D = g[t] * D + g[t] * M * gate_err[t]
            h, M = g[t] * h + u[t], g[t] * M + u[t].abs()
            D = D + 8 * M
            y[t], y_err[t] = h, D
        ns[n], ns_err[n] = h, D
    out = {"y": (y, y_err * U * 2), "new_state": (ns, ns_err * U * 2)}
    if dy is None:
        return out
    dy = dy.double()
    G, Gabs, Gerr = (torch.zeros_like(x) for _ in range(3))
    dstate, dstate_err = torch.zeros_like(h0), torch.zeros_like(h0)
    for n, (t0, t1) in enumerate(spans):
        e = torch.zeros(C, dtype=torch.float64, device=x.device) if dns is None else dns[n].double()
        ea, ee = e.abs(), torch.zeros_like(e)
        for t in reversed(range(t0, t1)):
            G[t], Gabs[t] = dy[t] + e, dy[t].abs() + ea
            Gerr[t] = ee + Gabs[t]
            e, ea = g[t] * G[t], g[t] * Gabs[t]
            ee = g[t] * Gerr[t] + g[t] * Gabs[t] * (gate_err[t] + 1)
        dstate[n], dstate_err[n] = e, ee
    scale = g * rate * sig
    da = -G * prev * scale
    da_abs = Gabs * prev_abs * scale
    da_err = scale * (Gerr * prev_abs + Gabs * prev_err) + da_abs * (gate_err + 24)
    dA = G * g * prev * l
    dA_abs = Gabs * g * prev_abs * l.abs()
    dA_err = g * l.abs() * (Gerr * prev_abs + Gabs * prev_err) + dA_abs * (gate_err + 24 + rate * z.abs() * sig / l.abs().clamp(min=1e-300))
    db = G * x * beta * torch.sigmoid(-b)
    # 1 - beta cancels when beta is near one: 8 U of beta stay
    db_err = Gerr * (x * beta * torch.sigmoid(-b)).abs() + Gabs * x.abs() * beta * (8 * beta + 16 * torch.sigmoid(-b))
    out |= {"dx": (G * beta, (Gerr * beta + 8 * Gabs * beta) * U * 2), "da": (da, da_err * U * 2), "db": (db, db_err * U * 2),
            "dA_log": (dA.sum(0), (dA_err + T * dA_abs).sum(0) * U * 2), "d_dt_bias": (da.sum(0), (da_err + T * da_abs).sum(0) * U * 2),
            "d_state": (dstate, dstate_err * U * 2)}
    return out


def close(got, want, err, what=""):
    """``got`` (rounded to its type) is within half a step of its type and ``err`` of ``want``."""
    assert got.shape == want.shape, what
    g = got.double()
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # a subnormal's step
    tol = half(got.dtype) * (want.abs() + err) + err + tiny
    bad = ~((g - want).abs() <= tol)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((g - want).abs() / tol).nan_to_num(float('inf')).max()):.3g} of the bound")


def add_norm(x, residual, weight, eps, dy=None, dr=None, summed=None):
    """(r, y) or, with ``dy``, the gradients at the stored sum; each with its fp32 bound.
    A row's sums of at most 32768 terms are trees of depth 80 or less here: 80 U."""
    K = 100 * U
    if dy is None:
        r = x.double() + (0 if residual is None else residual.double())
        y = r / (r.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
        return (r, U * r.abs()), (y, K * y.abs())
    r, w, dy = summed.double(), weight.double(), dy.double()
    inv = 1 / (r.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    n, up = r * inv, dy * w
    dx = inv * (up - n * (up * n).mean(-1, keepdim=True))
    err = K * inv * (up.abs() + n.abs() * (up * n).abs().mean(-1, keepdim=True))
    if dr is not None:
        dx, err = dx + dr.double(), err + U * dr.double().abs()
    t = dy * n
    return (dx, err), (t.sum(0), (K + r.shape[0] * U) * t.abs().sum(0))


def gated_norm(x, z, weight, eps, dy=None):
    K = 100 * U
    x, z, w = x.double(), z.double(), weight.double()
    inv = 1 / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    n, sig = x * inv, torch.sigmoid(z)
    gate = z * sig
    # exp(-z) from a 2 U exponential of a rounded product: (2 + |z|) U
    K = K + U * z.abs() * 2
    if dy is None:
        y = n * w * gate
        return y, K * y.abs()
    dy = dy.double()
    up = dy * w * gate
    dx = inv * (up - n * (up * n).mean(-1, keepdim=True))
    dx_err = inv * (K * up.abs() + n.abs() * (K * (up * n).abs()).mean(-1, keepdim=True))
    dgate = sig + gate * (1 - sig)
    dz = dy * n * w * dgate
    dz_err = K * (dy * n * w).abs() * (sig + gate.abs() * (1 - sig) + gate.abs() * sig)
    t = dy * n * gate
    rows = t.numel() // t.shape[-1]
    dims = tuple(range(t.dim() - 1))
    return (dx, dx_err), (dz, dz_err), (t.sum(dims), ((K + rows * U) * t.abs()).sum(dims))


def codes_ok(codes, scale, y, err, group):
    """e4m3 codes and scales of ``y``: the scale within its bound, every code
    within half a step (2^-4 relative, 2^-10 among the subnormals) of y over
    that scale."""
    rows = y.reshape(*y.shape[:-1], -1, group)
    amax = rows.abs().amax(-1).clamp(min=1e-12)
    s = scale.double().reshape(amax.shape)
    rel = (err.reshape(rows.shape) / rows.abs().clamp(min=1e-300)).amax(-1)
    assert bool(((s - amax / 448).abs() <= (rel + 4 * U) * amax / 448).all()), "scale"
    want = rows / s[..., None]
    slack = err.reshape(rows.shape) / s[..., None] + 4 * U * want.abs()
    got = codes.double().reshape(rows.shape)
    tol = torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10)) + slack
    bad = ~((got - want.clamp(-448, 448)).abs() <= tol)
    assert not bool(bad.any()), f"codes: {int(bad.sum())} of {bad.numel()} off"
