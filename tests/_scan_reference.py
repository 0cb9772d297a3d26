"""The gated scan in float64 on the CPU, with a bound for what float32 arithmetic may add to it.

``scan_reference`` evaluates the definition position by position and its gradients from the
adjoint recurrence, written out here; ``test_reference_gradients_against_autograd`` (CPU) holds
them to automatic differentiation.

Tolerances. A hardware or library function is taken as off by at most 2 units in the last place
(4 half-steps of ``H = 2**-24``), an addition, product or fused product by one half-step:

  softplus 4, sigmoid: exp2 4 + its argument's rounding (|v| H <= 8 H for the test's |v| <= 8) + sum 1 + reciprocal 4 -> 17
  L = softplus * sigma: 4 + 17 + 1 = 22 half-steps, so a = exp(L) is off by (22 |L| + 6) H of itself
  (its series or exponential, one rounding), q = 1 - a by 30 H of itself, m = sqrt(q (1 + a)) by
  half of 38 plus 4 -> 23, u = m sigma(i) x by 23 + 17 + 2 = 42.
  Every composition of maps rounds its two products once more: 4 H a position covers the local pass,
  the fold over groups, segments and tiles (each fold spans many positions).

The error of h then obeys e_t = a e_{t-1} + H ((22 |L| + 10) Habs_{t-1} + 46 |u_t|) with
Habs_t = a Habs_{t-1} + |u_t|, and that of g the same with |dy| for |u|. Products of those add up.
Outputs in bfloat16 add half a step (2**-8 of the value) for their one rounding.
"""

import torch

H = 2.0**-24


def half_step(dtype):
    return {torch.float32: H, torch.bfloat16: 2.0**-8}[dtype]


def softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def live_mask(n, T, lengths):
    if lengths is None:
        return torch.ones(n, T, dtype=torch.bool)
    return torch.arange(T) < lengths.cpu().clamp(0, T)[:, None]


def scan_reference(gates, decay, state=None, lengths=None, reverse=False, grad_out=None, grad_last=None):
    """Dicts (values, tolerances) of float64 CPU tensors: out, last and, with ``grad_out``,
    grad_gates, grad_decay (per sample) and grad_state."""
    g64 = gates.detach().double().cpu()
    lam = decay.detach().double().cpu()
    n, T = g64.shape[:2]
    D = lam.shape[0]
    live = live_mask(n, T, lengths)[:, :, None]
    zero = torch.zeros((), dtype=torch.float64)
    x, r, i = (torch.where(live, v, zero) for v in g64.split(D, dim=2))
    sp, rho, s = softplus(lam), torch.sigmoid(r), torch.sigmoid(i)
    L = torch.where(live, -sp * rho, zero)
    a = L.exp()
    q = -torch.expm1(L)
    m = (q * (1 + a)).sqrt()
    u = m * s * x
    order = list(range(T - 1, -1, -1)) if reverse else list(range(T))
    h = torch.zeros(n, D, dtype=torch.float64) if state is None else state.detach().double().cpu()
    habs, e = h.abs(), torch.zeros_like(h)
    out, out_tol = torch.zeros(n, T, D, dtype=torch.float64), torch.zeros(n, T, D, dtype=torch.float64)
    prev, prev_abs, prev_e = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out)
    ca = 22 * L.abs() + 10
    for t in order:
        prev[:, t], prev_abs[:, t], prev_e[:, t] = h, habs, e
        on = live[:, t]
        e = torch.where(on, a[:, t] * e + H * (ca[:, t] * a[:, t] * habs + 46 * u[:, t].abs()), e)
        habs = torch.where(on, a[:, t] * habs + u[:, t].abs(), habs)
        h = torch.where(on, a[:, t] * h + u[:, t], h)
        out[:, t] = torch.where(on, h, zero)
        out_tol[:, t] = torch.where(on, e, zero)
    hs = half_step(gates.dtype)
    val = {"out": out, "last": h}
    tol = {"out": out_tol + hs * (out.abs() + out_tol), "last": e + H * habs}
    if grad_out is None:
        return val, tol
    dy = torch.where(live, grad_out.detach().double().cpu(), zero)
    R = torch.zeros(n, D, dtype=torch.float64) if grad_last is None else grad_last.detach().double().cpu()
    Rabs, Re = R.abs(), torch.zeros_like(R)
    gs, gabs, ge = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out)
    for t in reversed(order):
        gs[:, t] = dy[:, t] + R
        gabs[:, t] = dy[:, t].abs() + Rabs
        ge[:, t] = Re + 2 * H * gabs[:, t]
        R = a[:, t] * gs[:, t]
        Rabs = a[:, t] * gabs[:, t]
        Re = a[:, t] * ge[:, t] + H * ca[:, t] * Rabs
    kappa = torch.where(m > 0, -L / torch.where(m > 0, m, torch.ones_like(m)), zero)
    dx = gs * m * s
    di = dx * x * (1 - s)
    p1, p2 = L * a, s * x * a * a * kappa
    w = gs * (p1 * prev + p2)
    dr = w * (1 - rho)
    # dx: g's error, then 23 + 17 + 2; di: + x (1 - s), whose difference is off by 18 H of s
    dx_t = ge * (m * s) + 42 * H * dx.abs()
    di_t = dx_t * (x * (1 - s)).abs() + dx.abs() * x.abs() * 20 * H
    inner_abs = p1.abs() * prev_abs + p2.abs()
    w_t = ge * inner_abs + gabs * (p1.abs() * prev_e + H * ((22 * L.abs() + 40) * p1.abs() * prev_abs + (44 * L.abs() + 120) * p2.abs()))
    dr_t = w_t * (1 - rho) + w.abs() * 20 * H
    mask = live.expand_as(out)
    parts, part_tol = [], []
    for v, vt in ((dx, dx_t), (dr, dr_t), (di, di_t)):
        v, vt = torch.where(mask, v, zero), torch.where(mask, vt, zero)
        parts.append(v)
        part_tol.append(vt + hs * (v.abs() + vt))
    val["grad_gates"], tol["grad_gates"] = torch.cat(parts, 2), torch.cat(part_tol, 2)
    ratio = torch.sigmoid(lam) / sp
    w, w_t = torch.where(mask, w, zero), torch.where(mask, w_t, zero)
    val["grad_decay"] = w.sum(1) * ratio
    # the sum over positions: at most T roundings (a few dozen in a row where a row is a chain of tiles; T / 8 and
    # a few where one block walks it)
    tol["grad_decay"] = (w_t.sum(1) + H * (T + 30) * w.abs().sum(1)) * ratio
    val["grad_state"], tol["grad_state"] = R, Re + H * Rabs
    return val, tol


def assert_within(got, val, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == val.shape, f"{what}: {tuple(got.shape)} != {tuple(val.shape)}"
    if val.numel() == 0:
        return
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - val).abs() - tol - 1e-30
    worst = over.argmax()
    assert over.max() <= 0, (
        f"{what}: off by {(got - val).abs().reshape(-1)[worst]:.3e} where {tol.reshape(-1)[worst]:.3e} is allowed "
        f"(value {val.reshape(-1)[worst]:.3e}, index {int(worst)})"
    )
